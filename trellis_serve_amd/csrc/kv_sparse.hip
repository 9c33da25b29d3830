// Attention over the pages that each query's bounds make worth reading (gfx950).  Cache layout: kv_attention.hip.
//
// A page's bounds, per kv head and channel d: the largest and smallest key code hi_d, lo_d of its tokens, in the cache's own
// codes [pages][Hkv][2][128] (8 bits) or [..][64] (4 bits, packed like keys), so with its keys' scale ks they stay valid when
// kv_append rounds a page anew, as long as they are made anew with it.
//
// Worth of page p for a query row and kv head, over the head's G query heads g:
//   a_g = max |q_g| (finite values),  q8_gd = rint(127 q_gd / a_g)  (infinities +-127, NaN 0)
//   S_gp = sum_d q8_gd (q8_gd > 0 ? hi_pd : lo_pd) = sum_d q8+ hi + q8- lo      (exact, an integer below 2^22)
//   worth_p = max_g fp32(S_gp * (a_g ks_p))                                    (a_g ks_p is exact in fp32: one rounding)
// up to the rounding of q8 and a common factor an upper bound of every logit that the page holds for the group.  A row reads
// the pages of its first `first` and last `last` ones, and of the rest those of most worth, ties to the lower page.
// In integers the choice does not depend on any order of summation.
//
// page_bounds_kernel: a wave per (page, kv head).  Min and max in packed 16-bit integers that hold a code in their high bits.
// page_worth_kernel: a wave per 16 pages.  16 x 256 codes against the group's 16 columns (q8+ | q8-) are four MFMA 16x16x64
//   i8; the largest over the columns by DPP.  Worths are written as integers that order like them.
// page_select_kernel: a workgroup per (row, kv head) narrows the range of the T-th largest by histograms of 1024 equal parts
//   of it, then writes the pages in ascending order by prefix sums (no atomic decides an order).
// sparse_attention_kernel: (parts of the list, kv heads, rows) workgroups, waves take pages, one 16-token page is one MFMA
//   block; states are joined in LDS, parts by sparse_merge_kernel in order.
#include <math.h>

#include <algorithm>

#include "exl3_api.hpp"
#include "kv_device.hpp"

namespace exl3 {

typedef int kv_i32x4_t __attribute__((ext_vector_type(4)));
typedef int16_t kv_i16x2_t __attribute__((ext_vector_type(2)));

// ---- bounds ------------------------------------------------------------------------------------------------------------

struct PageBoundsArgs {
  const uint8_t* k_cache;
  int num_pages;
  const int* page_table;
  int max_pages;
  const int *seq_lens, *first;
  int max_new, Hkv, pages_each;
  long long items;
  uint8_t* bounds;
};

__device__ __forceinline__ uint32_t max_i16x2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(kv_i16x2_t, a),
                                                                __builtin_bit_cast(kv_i16x2_t, b)));
}
__device__ __forceinline__ uint32_t min_i16x2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(kv_i16x2_t, a),
                                                                __builtin_bit_cast(kv_i16x2_t, b)));
}
// over the lanes that differ in the bits from FROM up (a lane of 16: bits 2 and 3; 16 and 32)
template <int FROM>
__device__ __forceinline__ uint32_t max_rows(uint32_t v) {
  if constexpr (FROM <= 4) v = max_i16x2(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xF, 0xF, true));
  v = max_i16x2(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xF, 0xF, true));
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max_i16x2(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max_i16x2(b[0], b[1]);
}
template <int FROM>
__device__ __forceinline__ uint32_t min_rows(uint32_t v) {
  if constexpr (FROM <= 4) v = min_i16x2(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xF, 0xF, true));
  v = min_i16x2(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xF, 0xF, true));
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = min_i16x2(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return min_i16x2(b[0], b[1]);
}

template <int BITS>
__global__ __launch_bounds__(256) void page_bounds_kernel(const PageBoundsArgs a) {
  constexpr int ROW = BITS == 8 ? kHeadDim : kHeadDim / 2;
  constexpr int PER = ROW / 16;       // lanes of a token's row, 16 bytes each
  constexpr int LOADS = BITS == 8 ? 2 : 1;
  constexpr int PARTS = BITS == 8 ? 2 : 4;  // codes of a 16-bit half
  const int lane = threadIdx.x & 63;
  const long long item = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (item >= a.items) return;
  const long long at = item / a.Hkv;
  const int hk = (int)(item - at * a.Hkv);
  const int b = (int)(at / a.pages_each), pg = (int)(at - (long long)b * a.pages_each);
  const int len = min(a.seq_lens[b], a.max_pages * kPage);
  int from = a.first ? max(a.first[b], 0) : 0;
  if (len - from > a.max_new) from = len - a.max_new;
  const int lp = from / kPage + pg, first = lp * kPage;
  if (first >= len || from >= len) return;
  const int page = a.page_table[(size_t)b * a.max_pages + lp];
  if (page < 0 || page >= a.num_pages) return;
  const int live = min(len - first, kPage);
  const size_t block = (size_t)page * a.Hkv + hk;
  const uint8_t* src = a.k_cache + block * (kPage * ROW) + (lane % PER) * 16;
  uint32_t hi[4 * PARTS], lo[4 * PARTS];
#pragma unroll
  for (int j = 0; j < LOADS; j++) {
    const int token = min(lane / PER + j * (64 / PER), live - 1);  // the last live one for those that are not there
    const kv_u32x4_t raw = *reinterpret_cast<const kv_u32x4_t*>(src + token * ROW);
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int p = 0; p < PARTS; p++) {
        const uint32_t v = BITS == 8 ? (raw[i] << (8 - 8 * p)) & 0xFF00FF00u : (raw[i] << (12 - 4 * p)) & 0xF000F000u;
        uint32_t &h = hi[i * PARTS + p], &l = lo[i * PARTS + p];
        h = j ? max_i16x2(h, v) : v;
        l = j ? min_i16x2(l, v) : v;
      }
  }
#pragma unroll
  for (int i = 0; i < 4 * PARTS; i++) hi[i] = max_rows<PER>(hi[i]), lo[i] = min_rows<PER>(lo[i]);
  if (lane >= 2 * PER) return;
  kv_u32x4_t o;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    uint32_t w = 0;
#pragma unroll
    for (int p = 0; p < PARTS; p++) w |= (lane < PER ? hi : lo)[i * PARTS + p] >> (BITS == 8 ? 8 - 8 * p : 12 - 4 * p);
    o[i] = w;
  }
  *reinterpret_cast<kv_u32x4_t*>(a.bounds + block * (2 * ROW) + lane * 16) = o;
}

// ---- worth and choice of pages -----------------------------------------------------------------------------------------

struct SelectArgs {
  const uint16_t* q;
  long long ld_q;
  const uint16_t* k_scale;
  const uint8_t* bounds;
  int num_pages;
  const int* page_table;
  int batch, max_pages;
  const int *row_seq, *seq_lens;
  int Hq, Hkv, top, first, last;
  int stride;       // worths of a (row, kv head): max_pages rounded up to 16
  uint32_t* worth;
  int* pages_out;
};

// the sequence and the tokens of a row (0: none to see)
__device__ __forceinline__ int row_tokens(const int* row_seq, const int* seq_lens, int batch, int max_pages, int row, int& b) {
  b = row_seq ? row_seq[row] : row;
  return b < 0 || b >= batch ? 0 : min(max(seq_lens[row], 0), max_pages * kPage);
}

// rint(127 q / a) of |q| <= a: 127 q and the residual of the quotient are exact, so a half-way case comes out as itself, and
// any other is a part of 2^-19 away from half-way
__device__ __forceinline__ int whole(float q, float a, float r) {
  const float x = 127.f * q, y = x * r;
  return (int)__builtin_rintf(__builtin_fmaf(__builtin_fmaf(-y, a, x), r, y));
}

// integers that order like floats, NaN lowest, both zeros the same; never 0 or the largest
__device__ __forceinline__ uint32_t ordered(float f) {
  const uint32_t u = __builtin_bit_cast(uint32_t, f + 0.f);
  return f != f ? 1u : u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kWorthWaves = 4;

template <int BITS>
__global__ __launch_bounds__(64 * kWorthWaves) void page_worth_kernel(const SelectArgs a, int per_wave) {
  constexpr int ROW = BITS == 8 ? kHeadDim : kHeadDim / 2;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int hk = blockIdx.y, row = blockIdx.z;
  int b;
  const int len = row_tokens(a.row_seq, a.seq_lens, a.batch, a.max_pages, row, b);
  const int pages = (len + kPage - 1) / kPage;
  if (pages <= a.top) return;  // all of them are read
  const int wave = blockIdx.x * kWorthWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int p0 = wave * per_wave * 16, p1 = min(p0 + per_wave * 16, pages);
  if (p0 >= p1) return;
  const int G = a.Hq / a.Hkv;
  // the lane's channels of head min(n, G - 1), in the order that the bounds' fragments have: 8 bits, 16 g .. + 15 and
  // 64 + 16 g .. + 15; 4 bits, the even and the odd ones of 32 g .. + 31
  const uint16_t* qrow = a.q + row * a.ld_q + (size_t)(hk * G + min(n, G - 1)) * kHeadDim;
  kv_u32x4_t raw[4];
#pragma unroll
  for (int i = 0; i < 4; i++)
    raw[i] = *reinterpret_cast<const kv_u32x4_t*>(qrow + (BITS == 8 ? 64 * (i / 2) + 16 * g + 8 * (i & 1) : 32 * g + 8 * i));
  float x[32];
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const uint32_t u = raw[i / 4][i & 3];
    const half2_t h = __builtin_bit_cast(half2_t, u);
    x[2 * i] = (float)h[0], x[2 * i + 1] = (float)h[1];
  }
#pragma unroll
  for (int i = 0; i < 32; i++) {
    const float m = fabsf(x[i]);
    most = m < __builtin_inff() ? fmaxf(most, m) : most;
  }
  most = max_over_groups(most);
  const float inv = most > 0.f ? 1.f / most : 0.f;
  kv_i32x4_t plus[2], minus[2];
#pragma unroll
  for (int c = 0; c < 2; c++)
#pragma unroll
    for (int d = 0; d < 4; d++) {
      uint32_t p = 0, m = 0;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float v = BITS == 8 ? x[16 * c + 4 * d + e] : x[2 * (4 * d + e) + c];
        int w = whole(fminf(fmaxf(v, -most), most), most, inv);  // infinities as the largest
        w = v == v ? w : 0;
        p |= (uint32_t)max(w, 0) << (8 * e);
        m |= (uint32_t)(min(w, 0) & 0xFF) << (8 * e);
      }
      plus[c][d] = (int)p, minus[c][d] = (int)m;
    }
  const int* ptab = a.page_table + (size_t)b * a.max_pages;
  uint32_t* to = a.worth + ((size_t)row * a.Hkv + hk) * a.stride;
  for (int p = p0; p < p1; p += 16) {
    const int page = min(max(ptab[min(p + n, pages - 1)], 0), a.num_pages - 1);
    const size_t block = (size_t)page * a.Hkv + hk;
    const uint8_t* src = a.bounds + block * (2 * ROW) + 16 * g;
    const float ks = (float)__builtin_bit_cast(_Float16, a.k_scale[block]);
    kv_i32x4_t s = {0, 0, 0, 0};
    if constexpr (BITS == 8) {
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const kv_i32x4_t k = *reinterpret_cast<const kv_i32x4_t*>(src + 64 * c);
        s = __builtin_amdgcn_mfma_i32_16x16x64_i8(k, c < 2 ? plus[c & 1] : minus[c & 1], s, 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int c = 0; c < 2; c++) {
        const kv_i32x4_t k = *reinterpret_cast<const kv_i32x4_t*>(src + 64 * c);
        kv_i32x4_t even, odd;  // 16 times the codes
#pragma unroll
        for (int i = 0; i < 4; i++) even[i] = (int)(((uint32_t)k[i] << 4) & 0xF0F0F0F0u), odd[i] = (int)((uint32_t)k[i] & 0xF0F0F0F0u);
        s = __builtin_amdgcn_mfma_i32_16x16x64_i8(even, c ? minus[0] : plus[0], s, 0, 0, 0);
        s = __builtin_amdgcn_mfma_i32_16x16x64_i8(odd, c ? minus[1] : plus[1], s, 0, 0, 0);
      }
    }
    // lane: pages 4 g .. + 3 of head n
    uint32_t out[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float scale = most * __shfl(ks, 4 * g + i);  // exact
      const float total = (float)(BITS == 8 ? s[i] : s[i] / 16);
      uint32_t v = ordered(total * scale);
      v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xF, 0xF, true));
      v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xF, 0xF, true));
      v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xF, 0xF, true));
      v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xF, 0xF, true));
      out[i] = v;
    }
    if (n == 0) *reinterpret_cast<kv_u32x4_t*>(to + p + 4 * g) = kv_u32x4_t{out[0], out[1], out[2], out[3]};
  }
}

constexpr int kSelectThreads = 512;
constexpr int kSelectWaves = kSelectThreads / 64;
constexpr int kSelectBins = 1024;

// the sums over the workgroup of `v` before this thread's (exclusive) and in all; part: LDS, one int a wave
__device__ __forceinline__ int select_scan(int v, int& total, int* part) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int s = wave_scan(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) part[wave] = s;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSelectWaves; w++) {
    before += w < wave ? part[w] : 0;
    total += part[w];
  }
  return before + s - v;
}

__global__ __launch_bounds__(kSelectThreads) void page_select_kernel(const SelectArgs a) {
  __shared__ int hist[kSelectBins], part[kSelectWaves];
  __shared__ uint32_t range[2 * kSelectWaves];
  __shared__ int found[2];
  const int hk = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int b;
  const int len = row_tokens(a.row_seq, a.seq_lens, a.batch, a.max_pages, row, b);
  const int pages = (len + kPage - 1) / kPage;
  int* out = a.pages_out + ((size_t)row * a.Hkv + hk) * a.top;
  if (pages <= a.top) {
    for (int i = tid; i < a.top; i += kSelectThreads) out[i] = i < pages ? i : -1;
    return;
  }
  const uint32_t* worth = a.worth + ((size_t)row * a.Hkv + hk) * a.stride;
  const int p0 = a.first, p1 = pages - a.last;  // the pages that are chosen among
  int need = a.top - a.first - a.last;          // of them, 0 <= need < p1 - p0
  uint32_t lo = 0xFFFFFFFFu, hi = 0;
  for (int p = p0 + tid; p < p1; p += kSelectThreads) lo = min(lo, worth[p]), hi = max(hi, worth[p]);
  hi = wave_max_u32(hi), lo = ~wave_max_u32(~lo);
  if (lane == 0) range[wave] = lo, range[kSelectWaves + wave] = hi;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSelectWaves; w++) lo = min(lo, range[w]), hi = max(hi, range[kSelectWaves + w]);
  // the need-th largest is in [lo, hi], `need` counts from hi; it is found once the range is a single value
  while (need > 0 && lo < hi) {
    const uint32_t span = hi - lo;
    const int shift = max(0, 32 - __builtin_clz(span) - 10);  // span >> shift is below 1024
    for (int i = tid; i < kSelectBins; i += kSelectThreads) hist[i] = 0;
    __syncthreads();
    for (int p = p0 + tid; p < p1; p += kSelectThreads) {
      const uint32_t v = worth[p];
      if (v >= lo && v <= hi) atomicAdd(&hist[(hi - v) >> shift], 1);
    }
    __syncthreads();
    int here[2], total;
#pragma unroll
    for (int i = 0; i < 2; i++) here[i] = hist[2 * tid + i];
    int before = select_scan(here[0] + here[1], total, part);
#pragma unroll
    for (int i = 0; i < 2; i++) {
      if (before < need && before + here[i] >= need) found[0] = 2 * tid + i, found[1] = before;
      before += here[i];
    }
    __syncthreads();
    const uint32_t bin = found[0];
    need -= found[1];
    const uint32_t top = hi - (bin << shift), size = (1u << shift) - 1;
    hi = top;
    lo = top - lo > size ? top - size : lo;
    __syncthreads();
  }
  // above hi: chosen; at hi: the first `need`; none where nothing is needed
  const bool none = need == 0;
  int chosen = a.first, equal = 0;
  for (int i = tid; i < a.first; i += kSelectThreads) out[i] = i;
  for (int base = p0; base < p1; base += kSelectThreads) {
    const int p = base + tid;
    const uint32_t v = p < p1 ? worth[p] : 0;
    const int ties = !none && p < p1 && v == hi;
    int all_ties, taken;
    const int tie = equal + select_scan(ties, all_ties, part);
    const int take = !none && p < p1 && (v > hi || (ties && tie < need));
    const int at = chosen + select_scan(take, taken, part);
    if (take) out[at] = p;
    equal += all_ties, chosen += taken;
  }
  for (int i = tid; i < a.last; i += kSelectThreads) out[a.top - a.last + i] = p1 + i;
}

// ---- attention over the chosen pages -----------------------------------------------------------------------------------

struct SparseArgs {
  const _Float16* q;
  long long ld_q;
  const uint8_t *kc, *vc;
  const uint16_t *ksc, *vsc;
  int num_pages;
  const int* page_table;
  int batch, max_pages;
  const int *row_seq, *seq_lens, *pages;
  int Hq, Hkv, top;
  float qk_scale;
  int per, parts;  // list entries of a workgroup, workgroups of a (row, kv head)
  float *part_o, *part_ml;
  _Float16* out;
};

constexpr int kSparseWaves = 4;

// A wave's online softmax of the group's heads over pages.  P' = p * v_scale is rounded to fp16, so the reference m lies 11
// (base 2) below the largest p * v_scale so far, and moves when a page passes it by 15: probabilities keep fp16's normal
// range whatever the values' scale.  l sums p itself, at most 2^39 a key.
template <int BITS>
struct SparseState {
  float m = -INFINITY, l = 0.f;
  float4_t o[8];

  __device__ __forceinline__ void page(const KvRegs<BITS>& r, const half8_t qf[4], float qsum, int key0, int L,
                                       float qk_scale, int g) {
    constexpr float kBias = BITS == 8 ? 1152.0f : 1032.0f;
    float4_t st = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < 4; c++) st = __builtin_amdgcn_mfma_f32_16x16x32_f16(r.kfrag(c), qf[c], st, 0, 0, 0);
    const float sc = (float)r.kscale() * qk_scale, off = -kBias * qsum * sc;
    float sv[4];
#pragma unroll
    for (int i = 0; i < 4; i++) sv[i] = key0 + 4 * g + i < L ? __builtin_fmaf(st[i], sc, off) : -INFINITY;
    const float vs = (float)r.vscale();
    const float lv = __builtin_amdgcn_logf(fmaxf(fabsf(vs), 0x1p-24f));
    const float pm = max_over_groups(fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3]))) + lv;
    if (__builtin_amdgcn_ballot_w64(pm > m + 15.f)) {
      const float m_new = pm > m + 15.f ? pm - 11.f : m;
      const float alpha = m_new == m ? 1.f : __builtin_amdgcn_exp2f(m - m_new);  // 0 on the first page
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int db = 0; db < 8; db++) o[db] *= alpha;
    }
    float psum = 0.f;
    half4_t pf;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float p = __builtin_amdgcn_exp2f(sv[i] - m);
      psum += p;
      pf[i] = (_Float16)(p * vs);
    }
    l += sum_over_groups(psum);
    uint32_t vt[8];
    r.vtrans(vt);
#pragma unroll
    for (int db = 0; db < 8; db++)
      o[db] = __builtin_amdgcn_mfma_f32_16x16x16f16(codes_f16(vt[db], (_Float16)kBias), pf, o[db], 0, 0, 0);
  }
};

template <int BITS>
__global__ __launch_bounds__(64 * kSparseWaves) void sparse_attention_kernel(const SparseArgs a) {
  constexpr int ROW = KvRegs<BITS>::ROW, W = kSparseWaves;
  extern __shared__ float red[];  // [W][G][D + 1], then [W][G][2]
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63, n = l & 15, g = l >> 4;
  const int part = blockIdx.x, hk = blockIdx.y, row = blockIdx.z, G = a.Hq / a.Hkv;
  int b;
  const int L = row_tokens(a.row_seq, a.seq_lens, a.batch, a.max_pages, row, b);

  half8_t qf[4];
  float qpart = 0.f;
  {
    const _Float16* qrow = a.q + row * a.ld_q + (size_t)(hk * G + min(n, G - 1)) * kHeadDim + 32 * g;
    const bool live = n < G;
#pragma unroll
    for (int c = 0; c < 4; c++) {
      const half8_t raw = *reinterpret_cast<const half8_t*>(qrow + 8 * c);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        qf[c][e] = live ? raw[BITS == 8 ? e : (e >> 1) + 4 * (e & 1)] : (_Float16)0.0f;
        qpart += (float)qf[c][e];
      }
    }
  }
  const float qsum = sum_over_groups(qpart);
  SparseState<BITS> s;
#pragma unroll
  for (int db = 0; db < 8; db++) s.o[db] = float4_t{0.f, 0.f, 0.f, 0.f};

  const int* list = a.pages + ((size_t)row * a.Hkv + hk) * a.top;
  const int* ptab = a.page_table + (size_t)(L > 0 ? b : 0) * a.max_pages;
  const int end = min((part + 1) * a.per, a.top), table_pages = (L + kPage - 1) / kPage;
  for (int i = part * a.per + w; i < end; i += W) {
    const int lp = list[i];
    if (lp < 0 || lp >= table_pages) continue;  // not a page of the row's
    const size_t bi = (size_t)min(max(ptab[lp], 0), a.num_pages - 1) * a.Hkv + hk;
    KvRegs<BITS> r;
    r.load(a.kc + bi * (kPage * ROW), a.vc + bi * (kPage * ROW), a.ksc, a.vsc, bi, n, g);
    s.page(r, qf, qsum, lp * kPage, L, a.qk_scale, g);
  }

  // join the waves; lane (n, g) holds dims 32 g + 8 i + db of query n
  float* red_ml = red + W * G * (kHeadDim + 1);
  if (n < G) {
    float* dst = red + (w * G + n) * (kHeadDim + 1) + 32 * g;
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int db = 0; db < 8; db++) dst[8 * i + db] = s.o[db][i];
    if (g == 0) red_ml[(w * G + n) * 2] = s.m, red_ml[(w * G + n) * 2 + 1] = s.l;
  }
  __syncthreads();
  const int tq = threadIdx.x >> 4, td = (threadIdx.x & 15) * 8;
  if (tq >= G) return;
  float mx = -INFINITY;
#pragma unroll
  for (int ww = 0; ww < W; ww++) mx = fmaxf(mx, red_ml[(ww * G + tq) * 2]);
  float lsum = 0.f, acc[8] = {};
#pragma unroll
  for (int ww = 0; ww < W; ww++) {
    const float mw = red_ml[(ww * G + tq) * 2];
    if (mw == -INFINITY) continue;
    const float f = __builtin_amdgcn_exp2f(mw - mx);
    lsum += red_ml[(ww * G + tq) * 2 + 1] * f;
    const float* src = red + (ww * G + tq) * (kHeadDim + 1) + td;
#pragma unroll
    for (int e = 0; e < 8; e++) acc[e] += src[e] * f;
  }
  const size_t head = (size_t)row * a.Hq + hk * G + tq;
  if (a.parts == 1) {
    half8_t h;
#pragma unroll
    for (int e = 0; e < 8; e++) h[e] = (_Float16)(mx == -INFINITY ? 0.f : acc[e] / lsum);
    *reinterpret_cast<half8_t*>(a.out + head * kHeadDim + td) = h;
    return;
  }
  const size_t slot = head * a.parts + part;
  float4_t* po = reinterpret_cast<float4_t*>(a.part_o + slot * kHeadDim + td);
  po[0] = float4_t{acc[0], acc[1], acc[2], acc[3]};
  po[1] = float4_t{acc[4], acc[5], acc[6], acc[7]};
  if (td == 0) a.part_ml[slot * 2] = mx, a.part_ml[slot * 2 + 1] = lsum;
}

// One wave per (row, head): lane holds dims 2 l, 2 l + 1; parts in order
__global__ __launch_bounds__(256) void sparse_merge_kernel(const SparseArgs a, int heads) {
  const int head = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63;
  if (head >= heads) return;
  const float* ml = a.part_ml + (size_t)head * a.parts * 2;
  float mx = -INFINITY;
  for (int c = 0; c < a.parts; c++) mx = fmaxf(mx, ml[2 * c]);
  float lsum = 0.f, a0 = 0.f, a1 = 0.f;
  for (int c = 0; c < a.parts; c++) {
    if (ml[2 * c] == -INFINITY) continue;
    const float f = __builtin_amdgcn_exp2f(ml[2 * c] - mx);
    const float2 o = *reinterpret_cast<const float2*>(a.part_o + ((size_t)head * a.parts + c) * kHeadDim + 2 * l);
    lsum += ml[2 * c + 1] * f;
    a0 += o.x * f, a1 += o.y * f;
  }
  const bool empty = mx == -INFINITY;
  *reinterpret_cast<half2_t*>(a.out + (size_t)head * kHeadDim + 2 * l) =
      half2_t{(_Float16)(empty ? 0.f : a0 / lsum), (_Float16)(empty ? 0.f : a1 / lsum)};
}

struct SparsePlan {
  int per, parts;
};
// Enough workgroups for two a CU, each with a page a wave at least
static SparsePlan sparse_plan(int rows, int Hkv, int top) {
  const long long pairs = (long long)rows * Hkv;
  const int most = (top + kSparseWaves - 1) / kSparseWaves;
  const int parts = (int)std::max<long long>(1, std::min<long long>(most, (512 + pairs - 1) / pairs));
  const int per = ((top + parts - 1) / parts + kSparseWaves - 1) / kSparseWaves * kSparseWaves;
  return SparsePlan{per, (top + per - 1) / per};
}

static int check_rows(const char* what, int num_pages, int batch, int max_pages, int rows, const int* row_seq, int Hq, int Hkv,
                      int head_dim, int page_size, int bits, int top) {
  EXL3_CHECK_ARG(head_dim == kHeadDim && page_size == kPage, "%s: head_dim = %d, page_size = %d (supported: 128, 16)", what,
                 head_dim, page_size);
  EXL3_CHECK_ARG(bits == 4 || bits == 8, "%s: bits = %d (4 or 8)", what, bits);
  EXL3_CHECK_ARG(batch >= 0 && num_pages >= 1 && num_pages <= (1 << 26) && max_pages >= 1 && max_pages <= (1 << 26) &&
                     rows >= 0 && rows <= 65535 && top >= 1 && top <= (1 << 20),
                 "%s: batch = %d, pages = %d, max_pages = %d, rows = %d, top = %d", what, batch, num_pages, max_pages, rows,
                 top);
  EXL3_CHECK_ARG(Hkv >= 1 && Hkv <= 65535 && Hq >= 1 && Hq % Hkv == 0 && Hq / Hkv <= kMaxGroup,
                 "%s: heads %d / %d (group <= 16)", what, Hq, Hkv);
  EXL3_CHECK_ARG(row_seq || rows == batch, "%s: %d rows of %d sequences without row_seq", what, rows, batch);
  return EXL3_OK;
}

}  // namespace exl3

using namespace exl3;

extern "C" int exl3_kv_page_bounds(const void* k_cache, int num_pages, const int* page_table, int max_pages,
                                   const int* seq_lens, const int* first, int max_new, int batch, int num_kv_heads,
                                   int head_dim, int page_size, int bits, void* bounds, void* stream) {
  EXL3_CHECK_ARG(head_dim == kHeadDim && page_size == kPage,
                 "exl3_kv_page_bounds: head_dim = %d, page_size = %d (supported: 128, 16)", head_dim, page_size);
  EXL3_CHECK_ARG(bits == 4 || bits == 8, "exl3_kv_page_bounds: bits = %d (4 or 8)", bits);
  EXL3_CHECK_ARG(batch >= 0 && num_pages >= 1 && num_pages <= (1 << 26) && max_pages >= 1 && max_pages <= (1 << 26) &&
                     num_kv_heads >= 1 && num_kv_heads <= 65536 && max_new >= 0,
                 "exl3_kv_page_bounds: batch = %d, pages = %d, max_pages = %d, kv heads = %d, max_new = %d", batch, num_pages,
                 max_pages, num_kv_heads, max_new);
  EXL3_CHECK_ARG(k_cache && bounds && (((uintptr_t)k_cache | (uintptr_t)bounds) & 15) == 0,
                 "exl3_kv_page_bounds: the cache or the bounds are null or not 16-byte aligned");
  if (batch == 0 || max_new == 0) return EXL3_OK;
  EXL3_CHECK_ARG(page_table && seq_lens, "exl3_kv_page_bounds: null pointer");
  const size_t blocks = (size_t)num_pages * num_kv_heads, row = (size_t)head_dim * bits / 8;
  const Span all[] = {{bounds, blocks * 2 * row}, {k_cache, blocks * page_size * row},
                      {page_table, (size_t)batch * max_pages * sizeof(int)}, {seq_lens, batch * sizeof(int)},
                      {first, batch * sizeof(int)}};
  EXL3_CHECK_ARG(apart(all, 1), "exl3_kv_page_bounds: the bounds overlap another tensor of the call");
  const int pages_each = (int)std::min<long long>(max_pages, ((long long)max_new + 2 * (kPage - 1)) / kPage);
  const long long items = (long long)batch * pages_each * num_kv_heads;
  EXL3_CHECK_ARG(items < (1LL << 26), "exl3_kv_page_bounds: %d sequences of up to %d tokens", batch, max_new);
  const PageBoundsArgs a{static_cast<const uint8_t*>(k_cache), num_pages, page_table, max_pages, seq_lens, first, max_new,
                         num_kv_heads, pages_each, items, static_cast<uint8_t*>(bounds)};
  auto kern = bits == 8 ? page_bounds_kernel<8> : page_bounds_kernel<4>;
  kern<<<(unsigned)((items + 3) / 4), 256, 0, as_stream(stream)>>>(a);
  EXL3_CHECK_LAUNCH();
  return EXL3_OK;
}

static size_t select_stride(int max_pages) { return ((size_t)max_pages + 15) / 16 * 16; }

extern "C" size_t exl3_kv_select_workspace_bytes(int rows, int num_kv_heads, int max_pages) {
  if (rows <= 0 || num_kv_heads <= 0 || max_pages <= 0) return 0;
  return (size_t)rows * num_kv_heads * select_stride(max_pages) * sizeof(uint32_t);
}

extern "C" int exl3_kv_select_pages(const void* q, long long ld_q, const void* k_scale, const void* bounds, int num_pages,
                                    const int* page_table, int batch, int max_pages, const int* row_seq,
                                    const int* seq_lens, int rows, int num_q_heads, int num_kv_heads, int head_dim,
                                    int page_size, int bits, int top, int first, int last, int* pages_out, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  if (const int rc = check_rows("exl3_kv_select_pages", num_pages, batch, max_pages, rows, row_seq, num_q_heads,
                                num_kv_heads, head_dim, page_size, bits, top))
    return rc;
  EXL3_CHECK_ARG(first >= 0 && last >= 1 && first <= top && last <= top - first,
                 "exl3_kv_select_pages: first = %d and last = %d (1 at least) of top = %d pages", first, last, top);
  EXL3_CHECK_ARG(k_scale && bounds && ((uintptr_t)bounds & 15) == 0,
                 "exl3_kv_select_pages: the bounds or the scales are null, or the bounds not 16-byte aligned");
  if (rows == 0) return EXL3_OK;
  EXL3_CHECK_ARG(q && seq_lens && pages_out && (page_table || batch == 0), "exl3_kv_select_pages: null pointer");
  EXL3_CHECK_ARG(ld_q >= (long long)num_q_heads * head_dim && ld_q % 8 == 0 && ((uintptr_t)q & 15) == 0,
                 "exl3_kv_select_pages: row stride %lld (a multiple of 8, a row's heads at least; 16-byte aligned)", ld_q);
  const size_t need = exl3_kv_select_workspace_bytes(rows, num_kv_heads, max_pages);
  EXL3_CHECK_ARG(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0,
                 "exl3_kv_select_pages: workspace %zu bytes, need %zu (16-byte aligned)", workspace_bytes, need);
  const size_t blocks = (size_t)num_pages * num_kv_heads, ints = sizeof(int);
  const Span all[] = {{pages_out, (size_t)rows * num_kv_heads * top * ints}, {workspace, need},
                      {q, 2 * ((size_t)(rows - 1) * ld_q + (size_t)num_q_heads * head_dim)}, {k_scale, blocks * 2},
                      {bounds, blocks * 2 * head_dim * bits / 8}, {page_table, (size_t)batch * max_pages * ints},
                      {row_seq, rows * ints}, {seq_lens, rows * ints}};
  EXL3_CHECK_ARG(apart(all, 2), "exl3_kv_select_pages: an output or the workspace overlaps another tensor of the call");
  const SelectArgs a{static_cast<const uint16_t*>(q), ld_q, static_cast<const uint16_t*>(k_scale),
                     static_cast<const uint8_t*>(bounds), num_pages, page_table, batch, max_pages, row_seq, seq_lens,
                     num_q_heads, num_kv_heads, top, first, last, (int)select_stride(max_pages),
                     static_cast<uint32_t*>(workspace), pages_out};
  if (max_pages > top) {
    const int groups = (max_pages + 15) / 16;
    const long long pairs = (long long)rows * num_kv_heads;
    const int per_wave = (int)std::max<long long>(1, std::min<long long>(16, groups * pairs / 8192));
    const int waves = (groups + per_wave - 1) / per_wave;
    auto kern = bits == 8 ? page_worth_kernel<8> : page_worth_kernel<4>;
    kern<<<dim3((waves + kWorthWaves - 1) / kWorthWaves, num_kv_heads, rows), 64 * kWorthWaves, 0, as_stream(stream)>>>(
        a, per_wave);
    EXL3_CHECK_LAUNCH();
  }
  page_select_kernel<<<dim3(num_kv_heads, rows), kSelectThreads, 0, as_stream(stream)>>>(a);
  EXL3_CHECK_LAUNCH();
  return EXL3_OK;
}

extern "C" size_t exl3_kv_sparse_workspace_bytes(int rows, int num_q_heads, int num_kv_heads, int top) {
  if (rows <= 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads || top <= 0) return 0;
  const SparsePlan plan = sparse_plan(rows, num_kv_heads, top);
  return plan.parts == 1 ? 0 : (size_t)rows * num_q_heads * plan.parts * (kHeadDim + 2) * sizeof(float);
}

extern "C" int exl3_kv_sparse_attention(const void* q, long long ld_q, const void* k_cache, const void* v_cache,
                                        const void* k_scale, const void* v_scale, int num_pages, const int* page_table,
                                        int batch, int max_pages, const int* row_seq, const int* seq_lens, int rows,
                                        int num_q_heads, int num_kv_heads, int head_dim, int page_size, int bits,
                                        const int* pages, int top, float sm_scale, void* out, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  if (const int rc = check_rows("exl3_kv_sparse_attention", num_pages, batch, max_pages, rows, row_seq, num_q_heads,
                                num_kv_heads, head_dim, page_size, bits, top))
    return rc;
  EXL3_CHECK_ARG(k_cache && v_cache && k_scale && v_scale && (((uintptr_t)k_cache | (uintptr_t)v_cache) & 15) == 0,
                 "exl3_kv_sparse_attention: a cache is null or not 16-byte aligned");
  if (rows == 0) return EXL3_OK;
  EXL3_CHECK_ARG(q && seq_lens && pages && out && (page_table || batch == 0), "exl3_kv_sparse_attention: null pointer");
  EXL3_CHECK_ARG(ld_q >= (long long)num_q_heads * head_dim && ld_q % 8 == 0 && (((uintptr_t)q | (uintptr_t)out) & 15) == 0,
                 "exl3_kv_sparse_attention: row stride %lld (a multiple of 8, a row's heads at least; 16-byte aligned)", ld_q);
  const size_t need = exl3_kv_sparse_workspace_bytes(rows, num_q_heads, num_kv_heads, top);
  EXL3_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
                 "exl3_kv_sparse_attention: workspace %zu bytes, need %zu (16-byte aligned)", workspace_bytes, need);
  const size_t blocks = (size_t)num_pages * num_kv_heads, ints = sizeof(int), code_bytes = blocks * page_size * head_dim * bits / 8;
  const size_t heads = (size_t)num_q_heads * head_dim;
  const Span all[] = {{out, rows * heads * 2}, {need ? workspace : nullptr, need}, {q, 2 * ((size_t)(rows - 1) * ld_q + heads)},
                      {k_cache, code_bytes}, {v_cache, code_bytes}, {k_scale, blocks * 2}, {v_scale, blocks * 2},
                      {page_table, (size_t)batch * max_pages * ints}, {row_seq, rows * ints}, {seq_lens, rows * ints},
                      {pages, (size_t)rows * num_kv_heads * top * ints}};
  EXL3_CHECK_ARG(apart(all, 2), "exl3_kv_sparse_attention: the output or the workspace overlaps another tensor of the call");
  const SparsePlan plan = sparse_plan(rows, num_kv_heads, top);
  float* part_o = static_cast<float*>(workspace);
  const int G = num_q_heads / num_kv_heads, all_heads = rows * num_q_heads;
  const SparseArgs a{static_cast<const _Float16*>(q), ld_q, static_cast<const uint8_t*>(k_cache),
                     static_cast<const uint8_t*>(v_cache), static_cast<const uint16_t*>(k_scale),
                     static_cast<const uint16_t*>(v_scale), num_pages, page_table, batch, max_pages, row_seq, seq_lens, pages,
                     num_q_heads, num_kv_heads, top, sm_scale * 1.4426950408889634f, plan.per, plan.parts, part_o,
                     plan.parts == 1 ? nullptr : part_o + (size_t)all_heads * plan.parts * kHeadDim,
                     static_cast<_Float16*>(out)};
  const size_t lds = (size_t)kSparseWaves * G * (kHeadDim + 1 + 2) * sizeof(float);
  auto kern = bits == 8 ? sparse_attention_kernel<8> : sparse_attention_kernel<4>;
  kern<<<dim3(plan.parts, num_kv_heads, rows), 64 * kSparseWaves, lds, as_stream(stream)>>>(a);
  EXL3_CHECK_LAUNCH();
  if (plan.parts > 1) {
    sparse_merge_kernel<<<(all_heads + 3) / 4, 256, 0, as_stream(stream)>>>(a, all_heads);
    EXL3_CHECK_LAUNCH();
  }
  return EXL3_OK;
}
