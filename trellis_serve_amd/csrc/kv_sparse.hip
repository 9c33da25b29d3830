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
// page_bounds_kernel: lanes of a (page, kv head) go through its 16 tokens with packed 16-bit minima and maxima.  Bound by the
//   bytes: 7 sequences of up to 32k 4-bit tokens, 76 MB, in 16.7 us (4.5 TB/s).
// page_worth_kernel: waves take 16 pages at a time.  16 heads (q8+ | q8-) against 16 x 256 codes are four MFMA 16x16x64 i8; query
//   rows of one sequence share the codes.  Worths are written as integers that order like them.  Bound by latency, for one row
//   (4.5 us at 32k) and for more: 16 rows of up to 24k 8-bit tokens, 26 MB of bounds, take 14.6 us (1.8 TB/s), since a wave has
//   two groups of 16 pages behind its queries, their rounding and a barrier, one group ahead.
// page_select_kernel: a workgroup per (row, kv head) keeps the worths in registers, finds the T-th largest by a histogram of its
//   range and a ranked list of what is left, and writes the pages in ascending order by prefix sums (no atomic decides an
//   order).  Bound by its steps' latency: 5 us for up to 2048 pages, 10 us for 8192.
// sparse_attention_kernel: (parts of the list, kv heads, rows) workgroups, waves take pages, one 16-token page is one MFMA
//   block, the next page is loaded meanwhile; states are joined in LDS, parts by sparse_merge_kernel in order.  Bound by the
//   scattered pages' bytes: 16 rows x up to 128 pages of 8 bits, 66 MB, in 17.5 us (3.8 TB/s); 32 rows x 256 pages of 4 bits,
//   134 MB, in 33.7 us (VALU 72 % of the issue).
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
// Lanes of a token's row (16 bytes each) stay with one (page, kv head) and go through its 16 tokens, so that a wave has 16 of
// them (8 bits: 8) and nothing crosses lanes: 44 (40) instructions a page, where a wave a page with its reductions took ten
// times as many.
template <int BITS>
__global__ __launch_bounds__(64) void page_bounds_kernel(const PageBoundsArgs a) {
  constexpr int ROW = BITS == 8 ? kHeadDim : kHeadDim / 2;
  constexpr int PER = ROW / 16;             // lanes of a token's row
  constexpr int PARTS = BITS == 8 ? 2 : 4;  // codes of a 16-bit half
  const int lane = threadIdx.x;
  const unsigned item = blockIdx.x * (64u / PER) + lane / PER;
  if (item >= (unsigned)a.items) return;
  const unsigned at = item / (unsigned)a.Hkv;
  const int hk = (int)(item - at * (unsigned)a.Hkv);
  const int b = (int)(at / (unsigned)a.pages_each), pg = (int)(at - (unsigned)b * (unsigned)a.pages_each);
  const int len = min(a.seq_lens[b], a.max_pages * kPage);
  int from = a.first ? max(a.first[b], 0) : 0;
  if (from >= len) return;
  if (len - from > a.max_new) from = len - a.max_new;
  const int lp = from / kPage + pg, first = lp * kPage;
  if (first >= len) return;
  const int page = a.page_table[(size_t)b * a.max_pages + lp];
  if (page < 0 || page >= a.num_pages) return;
  const int live = min(len - first, kPage);
  const size_t block = (size_t)page * a.Hkv + hk;
  const uint8_t* src = a.k_cache + block * (kPage * ROW) + (lane % PER) * 16;
  kv_u32x4_t raw[kPage];
#pragma unroll
  for (int t = 0; t < kPage; t++)  // the last live token for those that are not there
    raw[t] = *reinterpret_cast<const kv_u32x4_t*>(src + min(t, live - 1) * ROW);
  kv_u32x4_t hi, lo;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    uint32_t out_hi = 0, out_lo = 0;
#pragma unroll
    for (int p = 0; p < PARTS; p++) {
      // code p of both halves moves to their tops; what is below it does not change the order of the tops
      constexpr uint32_t TOP = BITS == 8 ? 0xFF00FF00u : 0xF000F000u;
      const int up = BITS == 8 ? 8 - 8 * p : 12 - 4 * p;
      uint32_t h = raw[0][i] << up, l = h;
#pragma unroll
      for (int t = 1; t < kPage; t++) {
        const uint32_t v = raw[t][i] << up;
        h = max_i16x2(h, v), l = min_i16x2(l, v);
      }
      out_hi |= (h & TOP) >> up, out_lo |= (l & TOP) >> up;
    }
    hi[i] = out_hi, lo[i] = out_lo;
  }
  uint8_t* to = a.bounds + block * (2 * ROW) + (lane % PER) * 16;
  *reinterpret_cast<kv_u32x4_t*>(to) = hi;
  *reinterpret_cast<kv_u32x4_t*>(to + ROW) = lo;
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
constexpr int kWorthRows = 4;  // consecutive rows of a workgroup; those of one sequence share what it reads

// A page group's bounds (16 pages, the lane's is n) as MFMA operands, and its page's scale
template <int BITS>
struct WorthRegs {
  kv_i32x4_t k[BITS == 8 ? 4 : 2];
  uint32_t ks;
  __device__ __forceinline__ void load(const SelectArgs& a, int page, int hk, int g) {
    constexpr int ROW = BITS == 8 ? kHeadDim : kHeadDim / 2;
    const size_t block = (size_t)min(max(page, 0), a.num_pages - 1) * a.Hkv + hk;
    const uint8_t* src = a.bounds + block * (2 * ROW) + 16 * g;
    ks = a.k_scale[block];
#pragma unroll
    for (int c = 0; c < (BITS == 8 ? 4 : 2); c++) k[c] = *reinterpret_cast<const kv_i32x4_t*>(src + 64 * c);
  }
  // products with the rounded queries of 16 heads: lane (n, g) has those of heads 4 g .. + 3 with page n; 4 bits: 16 times that
  __device__ __forceinline__ kv_i32x4_t times(const kv_i32x4_t plus[2], const kv_i32x4_t minus[2]) const {
    kv_i32x4_t s = {0, 0, 0, 0};
    if constexpr (BITS == 8) {
#pragma unroll
      for (int c = 0; c < 4; c++)
        s = __builtin_amdgcn_mfma_i32_16x16x64_i8(c < 2 ? plus[c & 1] : minus[c & 1], k[c], s, 0, 0, 0);
    } else {
#pragma unroll
      for (int c = 0; c < 2; c++) {
        kv_i32x4_t even, odd;
#pragma unroll
        for (int i = 0; i < 4; i++)
          even[i] = (int)(((uint32_t)k[c][i] << 4) & 0xF0F0F0F0u), odd[i] = (int)((uint32_t)k[c][i] & 0xF0F0F0F0u);
        s = __builtin_amdgcn_mfma_i32_16x16x64_i8(c ? minus[0] : plus[0], even, s, 0, 0, 0);
        s = __builtin_amdgcn_mfma_i32_16x16x64_i8(c ? minus[1] : plus[1], odd, s, 0, 0, 0);
      }
    }
    return s;
  }
};

// A head, rounded: the lane's channels in the order that the bounds' operands have them: 8 bits, 16 g .. + 15 and
// 64 + 16 g .. + 15; 4 bits, the even and the odd ones of 32 g .. + 31.  Every wave of a workgroup needs the same, so each rounds
// a quarter and the others take it from LDS.
struct WorthShared {
  uint32_t plus[kWorthRows][8][64], minus[kWorthRows][8][64];
};
template <int BITS>
struct WorthQuery {
  kv_i32x4_t plus[2], minus[2];
  __device__ __forceinline__ static void load(const uint16_t* head, int g, kv_u32x4_t raw[4]) {
#pragma unroll
    for (int i = 0; i < 4; i++)
      raw[i] = *reinterpret_cast<const kv_u32x4_t*>(head + (BITS == 8 ? 64 * (i / 2) + 16 * g + 8 * (i & 1) : 32 * g + 8 * i));
  }
  // returns max |q| of the head
  __device__ __forceinline__ static float round(const kv_u32x4_t raw[4], int lane, int wave, uint32_t plus[8][64],
                                                uint32_t minus[8][64]) {
    uint32_t most_bits = 0;  // magnitudes of halves order as integers; infinities and NaN take no part
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const uint32_t u = raw[i / 4][i & 3];
      const uint32_t lo = u & 0x7FFFu, hi = u >> 16 & 0x7FFFu;
      most_bits = max(most_bits, max(lo < 0x7C00u ? lo : 0, hi < 0x7C00u ? hi : 0));
    }
    const float most = max_over_groups((float)__builtin_bit_cast(_Float16, (uint16_t)most_bits));
    const float inv = most > 0.f ? 1.f / most : 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if (i / 2 != wave) continue;
      const int c = i / 4, d = i & 3;  // dword d of operand c: channels 4 d .. + 3 of it
      uint32_t p = 0, m = 0;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int at = BITS == 8 ? 16 * c + 4 * d + e : 2 * (4 * d + e) + c;  // of the lane's 32 halves
        const uint32_t u = raw[at / 8][at / 2 & 3];
        const half2_t h = __builtin_bit_cast(half2_t, u);
        const float v = (float)h[at & 1];
        int w = whole(fminf(fmaxf(v, -most), most), most, inv);  // infinities as the largest
        w = v == v ? w : 0;
        p |= (uint32_t)max(w, 0) << (8 * e);
        m |= (uint32_t)(min(w, 0) & 0xFF) << (8 * e);
      }
      plus[i][lane] = p, minus[i][lane] = m;
    }
    return most;
  }
  __device__ __forceinline__ void take(int lane, const uint32_t p[8][64], const uint32_t m[8][64]) {
#pragma unroll
    for (int i = 0; i < 8; i++) plus[i / 4][i & 3] = (int)p[i][lane], minus[i / 4][i & 3] = (int)m[i][lane];
  }
};

// The MFMA's 16 head rows hold 4, 2 or 1 query rows of up to 4, 8 or 16 heads (the last one repeated), so that a query row's
// maximum is one over a lane's own four values and at most two exchanges between lanes of one page.
template <int BITS, int ROWS>
__global__ __launch_bounds__(64 * kWorthWaves) void page_worth_kernel(const SelectArgs a, int rows, int per_wave) {
  __shared__ WorthShared sh;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hk = blockIdx.x, row0 = blockIdx.z * ROWS;  // kv heads first: a page's bounds lie side by side
  const int G = a.Hq / a.Hkv, wide = G <= 4 ? 4 : G <= 8 ? 8 : 16, fit = 16 / wide;
  const int start = blockIdx.y * kWorthWaves * per_wave * 16, p0 = start + w * per_wave * 16;
  int seq[ROWS], pages[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; r++) {
    seq[r] = -1, pages[r] = 0;
    if (row0 + r < rows) {
      pages[r] = (row_tokens(a.row_seq, a.seq_lens, a.batch, a.max_pages, row0 + r, seq[r]) + kPage - 1) / kPage;
      if (pages[r] <= a.top) pages[r] = 0;  // all of them are read
    }
  }
  // runs of rows that share a sequence
  for (int first = 0, count; first < ROWS; first += count) {
    count = 1;
    int most = pages[0], b = seq[0];
#pragma unroll
    for (int r = 0; r < ROWS; r++)
      if (r == first) b = seq[r], most = pages[r];
#pragma unroll
    for (int r = 1; r < ROWS; r++)
      if (r == first + count && seq[r] == b) count++, most = max(most, pages[r]);
    // sets of `fit` rows of the run
    WorthQuery<BITS> q[ROWS];
    float a4[ROWS][4];  // max |q| of the lane's result heads
    const int sets = (count + fit - 1) / fit, head = hk * G + min(n % wide, G - 1);
    // (asked for before the rows' lengths are known: entries past a length are not used)
    const int* ptab = a.page_table + (size_t)min(max(b, 0), a.batch - 1) * a.max_pages;
    int page = ptab[min(p0 + n, a.max_pages - 1)], then = ptab[min(p0 + 16 + n, a.max_pages - 1)];
    kv_u32x4_t raw[4];
    auto ask = [&](int i) {
      WorthQuery<BITS>::load(a.q + min(row0 + first + min(i * fit + n / wide, count - 1), rows - 1) * a.ld_q +
                                 (size_t)head * kHeadDim, g, raw);
    };
    ask(0);
    if (start >= most) continue;  // (the whole workgroup)
    if (first > 0) __syncthreads();
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      if (i >= sets) continue;
      if (i > 0) ask(i);
      const float largest = WorthQuery<BITS>::round(raw, lane, w, sh.plus[i], sh.minus[i]);
#pragma unroll
      for (int j = 0; j < 4; j++) a4[i][j] = __shfl(largest, 4 * g + j);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ROWS; i++)
      if (i < sets) q[i].take(lane, sh.plus[i], sh.minus[i]);
    const int p1 = min(p0 + per_wave * 16, most);
    if (p0 >= p1) continue;
    WorthRegs<BITS> next;
    next.load(a, page, hk, g);
    for (int p = p0; p < p1; p += 16) {
      const WorthRegs<BITS> now = next;
      next.load(a, then, hk, g);
      then = ptab[min(p + 32 + n, most - 1)];
      const float ks = (float)__builtin_bit_cast(_Float16, (uint16_t)now.ks);
#pragma unroll
      for (int i = 0; i < ROWS; i++) {
        if (i >= sets) continue;
        const kv_i32x4_t s = now.times(q[i].plus, q[i].minus);
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = (float)(BITS == 8 ? s[j] : s[j] >> 4) * (a4[i][j] * ks);  // a4 ks is exact
        // (fmaxf passes a NaN by)
        float worth = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
        if (wide >= 8) {
          const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(worth), __float_as_uint(worth), false, false);
          worth = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
        }
        if (wide == 16) {
          const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(worth), __float_as_uint(worth), false, false);
          worth = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
        }
        const int r = i * fit + 4 * g / wide;
        if (4 * g % wide == 0 && r < count)
          a.worth[((size_t)(row0 + first + r) * a.Hkv + hk) * a.stride + p + n] = ordered(worth);
      }
    }
  }
}

constexpr int kSelectThreads = 512;
constexpr int kSelectWaves = kSelectThreads / 64;
constexpr int kSelectBins = 1024;
constexpr int kSelectList = 64;

struct SelectShared {
  int hist[kSelectBins], part[2][kSelectWaves], found[2][3], listed;
  uint32_t range[2][kSelectWaves];
  unsigned long long list[kSelectList];  // worth << 32 | ~page
};

// EACH consecutive pages a thread, in registers; longer sequences by tiles, loaded anew for each pass
template <int EACH>
__global__ __launch_bounds__(kSelectThreads) void page_select_kernel(const SelectArgs a) {
  constexpr int TILE = EACH * kSelectThreads;
  __shared__ SelectShared sh;
  const int hk = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t* worth = a.worth + ((size_t)row * a.Hkv + hk) * a.stride;
  kv_u32x4_t raw[EACH / 4];  // (asked for before the row's length is known)
  auto ask = [&](int tile) {
#pragma unroll
    for (int i = 0; i < EACH / 4; i++)
      raw[i] = *reinterpret_cast<const kv_u32x4_t*>(worth + min(tile * TILE + tid * EACH + 4 * i, a.stride - 4));
  };
  ask(0);
  int b;
  const int len = row_tokens(a.row_seq, a.seq_lens, a.batch, a.max_pages, row, b);
  const int pages = (len + kPage - 1) / kPage;
  int* out = a.pages_out + ((size_t)row * a.Hkv + hk) * a.top;
  if (pages <= a.top) {
    for (int i = tid; i < a.top; i += kSelectThreads) out[i] = i < pages ? i : -1;
    return;
  }
  const int p0 = a.first, p1 = pages - a.last;  // the pages that are chosen among; 0 for the others
  const int tiles = (pages + TILE - 1) / TILE;
  uint32_t v[EACH];
  auto keep = [&](int tile) {
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      const int p = tile * TILE + tid * EACH + i;
      v[i] = p >= p0 && p < p1 ? raw[i / 4][i & 3] : 0;
    }
  };
  auto load = [&](int tile) { ask(tile), keep(tile); };
  keep(0);
  int need = a.top - a.first - a.last;  // of them, 0 <= need < p1 - p0
  uint32_t lo = ~0u, hi = 0;
  for (int tile = 0; tile < tiles; tile++) {
    if (tiles > 1) load(tile);
#pragma unroll
    for (int i = 0; i < EACH; i++) lo = v[i] ? min(lo, v[i]) : lo, hi = max(hi, v[i]);
  }
  hi = wave_max_u32(hi), lo = wave_max_u32(~lo);
  if (lane == 0) sh.range[0][wave] = lo, sh.range[1][wave] = hi;
  if (tid == 0) sh.listed = 0;
  for (int i = tid; i < kSelectBins; i += kSelectThreads) sh.hist[i] = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSelectWaves; w++) lo = max(lo, sh.range[0][w]), hi = max(hi, sh.range[1][w]);
  lo = ~lo;
  // The need-th largest is in [lo, hi], `need` counts from hi.  The range narrows to one of 1024 parts of it until few are in it.
  int here = p1 - p0;
  for (int turn = 0; need > 0 && here > kSelectList && lo < hi; turn ^= 1) {
    const uint32_t span = hi - lo;
    const int shift = max(0, 32 - __builtin_clz(span) - 10);  // span >> shift is below 1024
    for (int tile = 0; tile < tiles; tile++) {
      if (tiles > 1) load(tile);
#pragma unroll
      for (int i = 0; i < EACH; i++)
        if (v[i] >= lo && v[i] <= hi) atomicAdd(&sh.hist[(hi - v[i]) >> shift], 1);
    }
    __syncthreads();
    const int h0 = sh.hist[2 * tid], h1 = sh.hist[2 * tid + 1];
    const int upto = wave_scan(h0 + h1);
    if (lane == 63) sh.part[turn][wave] = upto;
    __syncthreads();
    int before = upto - h0 - h1;
#pragma unroll
    for (int w = 0; w < kSelectWaves; w++) before += w < wave ? sh.part[turn][w] : 0;
    if (before < need && before + h0 >= need) sh.found[turn][0] = 2 * tid, sh.found[turn][1] = before, sh.found[turn][2] = h0;
    if (before + h0 < need && before + h0 + h1 >= need)
      sh.found[turn][0] = 2 * tid + 1, sh.found[turn][1] = before + h0, sh.found[turn][2] = h1;
    sh.hist[2 * tid] = sh.hist[2 * tid + 1] = 0;
    __syncthreads();
    need -= sh.found[turn][1], here = sh.found[turn][2];
    hi -= (uint32_t)sh.found[turn][0] << shift;
    const uint32_t size = (1u << shift) - 1;
    lo = hi - lo > size ? hi - size : lo;
  }
  // Above hi: chosen.  In [lo, hi]: the first `need` by worth and page, by their ranks in a list of them; a single worth held by
  // more pages than it takes: the first `need` by page.
  const bool ranked = need > 0 && here <= kSelectList;
  if (ranked) {
    for (int tile = 0; tile < tiles; tile++) {
      if (tiles > 1) load(tile);
#pragma unroll
      for (int i = 0; i < EACH; i++)
        if (v[i] && v[i] >= lo && v[i] <= hi)
          sh.list[atomicAdd(&sh.listed, 1)] = (unsigned long long)v[i] << 32 | (uint32_t)~(tile * TILE + tid * EACH + i);
    }
    __syncthreads();
  }
  const int listed = ranked ? sh.listed : 0;
  int chosen = a.first, ties = 0;
  for (int i = tid; i < a.first; i += kSelectThreads) out[i] = i;
  for (int tile = 0; tile < tiles; tile++) {
    if (tiles > 1) load(tile);
    unsigned take = 0, tie = 0;
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      if (need <= 0 || v[i] == 0) continue;
      bool in = v[i] > hi;
      if (v[i] >= lo && v[i] <= hi) {
        if (ranked) {
          const unsigned long long mine = (unsigned long long)v[i] << 32 | (uint32_t)~(tile * TILE + tid * EACH + i);
          int rank = 0;
          for (int j = 0; j < listed; j++) rank += sh.list[j] > mine;
          in = rank < need;
        } else {
          tie |= 1u << i;
        }
      }
      take |= (unsigned)in << i;
    }
    // counts of both, packed (at most 8192 of a tile)
    const int mine = __builtin_popcount(take) | __builtin_popcount(tie) << 16;
    const int upto = wave_scan(mine);
    __syncthreads();
    if (lane == 63) sh.part[0][wave] = upto;
    __syncthreads();
    int before = upto - mine, all = 0;
#pragma unroll
    for (int w = 0; w < kSelectWaves; w++) before += w < wave ? sh.part[0][w] : 0, all += sh.part[0][w];
    int to = chosen + (before & 0xFFFF) + min(need, ties + (before >> 16)) - min(need, ties), rank = ties + (before >> 16);
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      const bool is_tie = tie >> i & 1;
      if ((take >> i & 1) || (is_tie && rank < need)) out[to++] = tile * TILE + tid * EACH + i;
      rank += is_tie;
    }
    chosen += (all & 0xFFFF) + min(need, ties + (all >> 16)) - min(need, ties);
    ties += all >> 16;
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

// P' = p * v_scale enters the product as two halves, its first 11 bits and the next 11, so that it loses no more than 2^-21 of
// itself.  (By one half, rounded, outputs were 2.3e-4 of their norm off, of which fp16 outputs cannot but be 2.1e-4; by both they
// are 2.1e-4.)
constexpr uint32_t kFirstHalf = 0xFFFFE000u;  // of a float

// four values, each cut to 11 bits
__device__ __forceinline__ half4_t cut_to_halves(const float x[4]) {
  return __builtin_bit_cast(half4_t, kv_u32x2_t{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x[0], x[1])),
                                                __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x[2], x[3]))});
}
__device__ __forceinline__ float without(float x, uint32_t bits) {
  return x - __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & bits);
}

// A wave's online softmax of the group's heads over pages.  Groups of up to 8 heads have each head in columns n and n + 8 of the
// product, with the first halves in the one and the second in the other: one MFMA, as for the first alone (66 MB of 8 bits for
// groups of 4: 17.0 -> 17.5 us; 134 MB of 4 bits for groups of 5: 32.3 -> 33.7).  WIDE groups take two (the same lengths for
// groups of 16: 22.2 -> 22.5, 38.1 -> 41.0).  The reference m lies 11 (base 2) below the largest p * v_scale so far, and moves when
// a page passes it by 15: probabilities keep fp16's normal range whatever the values' scale.  l sums p itself, at most 2^39 a key.
template <int BITS, bool WIDE>
struct SparseState {
  float m = -INFINITY, l = 0.f;
  float4_t o[8];

  // left_out: not WIDE: kFirstHalf in columns 8 .. 15, 0 in the others
  __device__ __forceinline__ void page(const KvRegs<BITS>& r, const half8_t qf[4], float qsum, int key0, int L,
                                       float qk_scale, int g, uint32_t left_out) {
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
    float psum = 0.f, x[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float p = __builtin_amdgcn_exp2f(sv[i] - m);
      psum += p;
      x[i] = p * vs;
      if constexpr (!WIDE) x[i] = without(x[i], left_out);
    }
    const half4_t first = cut_to_halves(x);
    half4_t second;
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < 4; i++) x[i] = without(x[i], kFirstHalf);
      second = cut_to_halves(x);
    }
    l += sum_over_groups(psum);
    uint32_t vt[8];
    r.vtrans(vt);
#pragma unroll
    for (int db = 0; db < 8; db++) {
      const half4_t v = codes_f16(vt[db], (_Float16)kBias);
      o[db] = __builtin_amdgcn_mfma_f32_16x16x16f16(v, first, o[db], 0, 0, 0);
      if constexpr (WIDE) o[db] = __builtin_amdgcn_mfma_f32_16x16x16f16(v, second, o[db], 0, 0, 0);
    }
  }
};

template <int BITS, bool WIDE>
__global__ __launch_bounds__(64 * kSparseWaves) void sparse_attention_kernel(const SparseArgs a) {
  constexpr int ROW = KvRegs<BITS>::ROW, W = kSparseWaves;
  extern __shared__ float red[];  // [W][G][D + 1], then [W][G][2]
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63, n = l & 15, g = l >> 4;
  const int part = blockIdx.x, hk = blockIdx.y, row = blockIdx.z, G = a.Hq / a.Hkv;
  // (the list is asked for before the row's length is known)
  const int* list = a.pages + ((size_t)row * a.Hkv + hk) * a.top;
  const int end = min((part + 1) * a.per, a.top);
  auto entry = [&](int i) { return list[min(i, end - 1)]; };
  int i = part * a.per + w, lp = entry(i), after = entry(i + W);
  int b;
  const int L = row_tokens(a.row_seq, a.seq_lens, a.batch, a.max_pages, row, b);

  half8_t qf[4];
  float qpart = 0.f;
  {
    const int head = WIDE ? n : n & 7;
    const _Float16* qrow = a.q + row * a.ld_q + (size_t)(hk * G + min(head, G - 1)) * kHeadDim + 32 * g;
    const bool live = head < G;
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
  const uint32_t left_out = n & 8 ? kFirstHalf : 0;
  SparseState<BITS, WIDE> s;
#pragma unroll
  for (int db = 0; db < 8; db++) s.o[db] = float4_t{0.f, 0.f, 0.f, 0.f};

  const int* ptab = a.page_table + (size_t)(L > 0 ? b : 0) * a.max_pages;
  const int table_pages = (L + kPage - 1) / kPage;
  // One page's codes are in flight while the one before is worked on, and the list's entry after it.  Entries that are no page
  // of the row's load its first one and are left out.
  if (L > 0 && i < end) {
    KvRegs<BITS> r[2];
    auto load = [&](KvRegs<BITS>& to, int lp) {
      const size_t bi = (size_t)min(max(ptab[min(max(lp, 0), table_pages - 1)], 0), a.num_pages - 1) * a.Hkv + hk;
      to.load(a.kc + bi * (kPage * ROW), a.vc + bi * (kPage * ROW), a.ksc, a.vsc, bi, n, g);
    };
    load(r[0], lp);
    bool more = true;
    while (more) {
#pragma unroll
      for (int j = 0; j < 2; j++) {
        if (more) {
          load(r[j ^ 1], after);
          const int then = entry(i + 2 * W);
          issue_fence();
          if (lp >= 0 && lp < table_pages) s.page(r[j], qf, qsum, lp * kPage, L, a.qk_scale, g, left_out);
          lp = after, after = then;
          i += W;
          more = i < end;
        }
      }
    }
  }

  // (logits that are NaN move no reference: without this a query of them alone would count as one that sees nothing)
  if (s.m == -INFINITY && s.l != 0.f) s.m = 0.f;
  if constexpr (!WIDE) {
#pragma unroll
    for (int db = 0; db < 8; db++)
#pragma unroll
      for (int i = 0; i < 4; i++) s.o[db][i] += lane_xor<8>(s.o[db][i]);
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

// One wave per (row, head): lane c holds part c's maximum and sum (64 parts at most), then dims 2 l, 2 l + 1; parts in order
constexpr int kSparseParts = 64;

__global__ __launch_bounds__(256) void sparse_merge_kernel(const SparseArgs a, int heads) {
  const int head = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63;
  if (head >= heads) return;
  const float2 ml = reinterpret_cast<const float2*>(a.part_ml)[(size_t)head * a.parts + min(l, a.parts - 1)];
  const float m = l < a.parts ? ml.x : -INFINITY;
  float mx = fmaxf(m, lane_xor<1>(m));
  mx = fmaxf(mx, lane_xor<2>(mx));
  mx = fmaxf(mx, lane_xor<4>(mx));
  mx = fmaxf(mx, lane_xor<8>(mx));
  mx = max_over_groups(mx);
  const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mx);
  const float share = f == 0.f ? 0.f : ml.y * f;
  float lsum = 0.f, a0 = 0.f, a1 = 0.f;
  const float* from = a.part_o + (size_t)head * a.parts * kHeadDim + 2 * l;
  for (int c0 = 0; c0 < a.parts; c0 += 8) {
#pragma unroll
    for (int i = 0; i < 8; i++) {  // past the last part the weight is 0
      const int c = c0 + i;
      const float fc = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), c));
      lsum += __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, share), c));
      const float2 o = *reinterpret_cast<const float2*>(from + (size_t)min(c, a.parts - 1) * kHeadDim);
      a0 = __builtin_fmaf(o.x, fc, a0), a1 = __builtin_fmaf(o.y, fc, a1);
    }
  }
  const bool empty = mx == -INFINITY;
  *reinterpret_cast<half2_t*>(a.out + (size_t)head * kHeadDim + 2 * l) =
      half2_t{(_Float16)(empty ? 0.f : a0 / lsum), (_Float16)(empty ? 0.f : a1 / lsum)};
}

struct SparsePlan {
  int per, parts;
};
// Enough workgroups for four a CU, each with a page a wave at least (16 sequences of 128 pages, 8 bits, 8 kv heads: two a CU 19 us,
// four 17, eight 19; 32 rows of 256 pages, 4 bits: 43, 32, 34)
constexpr int kSparseGroups = 1024;
static int sparse_most_parts(int top) { return std::min(kSparseParts, (top + kSparseWaves - 1) / kSparseWaves); }
static SparsePlan sparse_plan(int rows, int Hkv, int top) {
  const long long pairs = (long long)rows * Hkv;
  const int parts = (int)std::max<long long>(1, std::min<long long>(sparse_most_parts(top), (kSparseGroups + pairs - 1) / pairs));
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
  EXL3_CHECK_ARG(items < (1LL << 28), "exl3_kv_page_bounds: %d sequences of up to %d tokens", batch, max_new);
  const PageBoundsArgs a{static_cast<const uint8_t*>(k_cache), num_pages, page_table, max_pages, seq_lens, first, max_new,
                         num_kv_heads, pages_each, items, static_cast<uint8_t*>(bounds)};
  auto kern = bits == 8 ? page_bounds_kernel<8> : page_bounds_kernel<4>;
  const int each = bits == 8 ? 8 : 16;
  kern<<<(unsigned)((items + each - 1) / each), 64, 0, as_stream(stream)>>>(a);
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
  EXL3_CHECK_ARG(batch >= 1, "exl3_kv_select_pages: %d rows of no sequence", rows);
  EXL3_CHECK_ARG(q && seq_lens && pages_out && page_table, "exl3_kv_select_pages: null pointer");
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
    // rows of one sequence share its bounds where row_seq says that there can be any (4 rows each of 8 sequences of up to 128k
    // tokens, 4 bits: 59 us apart, 20 together)
    const int each = row_seq ? kWorthRows : 1, blocks_z = (rows + each - 1) / each;
    const int groups = (max_pages + 15) / 16;
    const long long pairs = (long long)blocks_z * num_kv_heads;
    const int per_wave = (int)std::max<long long>(1, std::min<long long>(16, groups * pairs / 4096));
    const int waves = (groups + per_wave - 1) / per_wave;
    const dim3 grid(num_kv_heads, (waves + kWorthWaves - 1) / kWorthWaves, blocks_z);
    auto kern = bits == 8 ? (row_seq ? page_worth_kernel<8, kWorthRows> : page_worth_kernel<8, 1>)
                          : (row_seq ? page_worth_kernel<4, kWorthRows> : page_worth_kernel<4, 1>);
    kern<<<grid, 64 * kWorthWaves, 0, as_stream(stream)>>>(a, rows, per_wave);
    EXL3_CHECK_LAUNCH();
  }
  auto pick = max_pages <= 4 * kSelectThreads ? page_select_kernel<4> : page_select_kernel<16>;
  pick<<<dim3(num_kv_heads, rows), kSelectThreads, 0, as_stream(stream)>>>(a);
  EXL3_CHECK_LAUNCH();
  return EXL3_OK;
}

extern "C" size_t exl3_kv_sparse_workspace_bytes(int rows, int num_q_heads, int num_kv_heads, int top) {
  if (rows <= 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads || top <= 0) return 0;
  // rows times parts of any number of rows up to `rows`, or a little more: from kSparseGroups (row, kv head) pairs on there is one
  // part, below that r rows have at most (kSparseGroups - 1) / (r heads) + 1 parts
  const long long split = std::min(rows, (kSparseGroups - 1) / num_kv_heads);
  const int most = sparse_most_parts(top);
  if (split == 0 || most == 1) return 0;
  const long long parts = std::min(split * most, (kSparseGroups - 1) / num_kv_heads + split);
  return (size_t)parts * num_q_heads * (kHeadDim + 2) * sizeof(float);
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
  EXL3_CHECK_ARG(batch >= 1, "exl3_kv_sparse_attention: %d rows of no sequence", rows);
  EXL3_CHECK_ARG(q && seq_lens && pages && out && page_table, "exl3_kv_sparse_attention: null pointer");
  EXL3_CHECK_ARG(ld_q >= (long long)num_q_heads * head_dim && ld_q % 8 == 0 && (((uintptr_t)q | (uintptr_t)out) & 15) == 0,
                 "exl3_kv_sparse_attention: row stride %lld (a multiple of 8, a row's heads at least; 16-byte aligned)", ld_q);
  const SparsePlan plan = sparse_plan(rows, num_kv_heads, top);
  const size_t need = plan.parts == 1 ? 0 : exl3_kv_sparse_workspace_bytes(rows, num_q_heads, num_kv_heads, top);
  EXL3_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
                 "exl3_kv_sparse_attention: workspace %zu bytes, need %zu (16-byte aligned)", workspace_bytes, need);
  const size_t blocks = (size_t)num_pages * num_kv_heads, ints = sizeof(int), code_bytes = blocks * page_size * head_dim * bits / 8;
  const size_t heads = (size_t)num_q_heads * head_dim;
  const Span all[] = {{out, rows * heads * 2}, {need ? workspace : nullptr, need}, {q, 2 * ((size_t)(rows - 1) * ld_q + heads)},
                      {k_cache, code_bytes}, {v_cache, code_bytes}, {k_scale, blocks * 2}, {v_scale, blocks * 2},
                      {page_table, (size_t)batch * max_pages * ints}, {row_seq, rows * ints}, {seq_lens, rows * ints},
                      {pages, (size_t)rows * num_kv_heads * top * ints}};
  EXL3_CHECK_ARG(apart(all, 2), "exl3_kv_sparse_attention: the output or the workspace overlaps another tensor of the call");
  float* part_o = static_cast<float*>(workspace);
  const int G = num_q_heads / num_kv_heads, all_heads = rows * num_q_heads;
  const SparseArgs a{static_cast<const _Float16*>(q), ld_q, static_cast<const uint8_t*>(k_cache),
                     static_cast<const uint8_t*>(v_cache), static_cast<const uint16_t*>(k_scale),
                     static_cast<const uint16_t*>(v_scale), num_pages, page_table, batch, max_pages, row_seq, seq_lens, pages,
                     num_q_heads, num_kv_heads, top, sm_scale * 1.4426950408889634f, plan.per, plan.parts, part_o,
                     plan.parts == 1 ? nullptr : part_o + (size_t)all_heads * plan.parts * kHeadDim,
                     static_cast<_Float16*>(out)};
  const size_t lds = (size_t)kSparseWaves * G * (kHeadDim + 1 + 2) * sizeof(float);
  auto kern = bits == 8 ? (G > 8 ? sparse_attention_kernel<8, true> : sparse_attention_kernel<8, false>)
                        : (G > 8 ? sparse_attention_kernel<4, true> : sparse_attention_kernel<4, false>);
  kern<<<dim3(plan.parts, num_kv_heads, rows), 64 * kSparseWaves, lds, as_stream(stream)>>>(a);
  EXL3_CHECK_LAUNCH();
  if (plan.parts > 1) {
    sparse_merge_kernel<<<(all_heads + 3) / 4, 256, 0, as_stream(stream)>>>(a, all_heads);
    EXL3_CHECK_LAUNCH();
  }
  return EXL3_OK;
}
