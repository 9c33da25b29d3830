// Writing the paged quantized KV cache, and reading it back (gfx950).  Layout: kv_attention.hip.
//
// kv_append_kernel.  A page's keys (and its values) of one kv head share one fp16 scale, so new tokens and the page's
// older ones have to agree on it.  For the new tokens of a (page, kv head):
//   a = max |x| over their finite values;  c = the smallest fp16 >= a / qmax      (qmax = 127 or 7)
//   s = c when the page's first slot is among them, else max(the page's scale, c)
//   older codes, when s grew:  code' = rint(code * s_old / s)          (at most half a step of s per growth)
//   new codes:  min(max(rint(x / s), -qmax), qmax), NaN as 0            (at most half a step off: s * qmax >= a)
// x and s have 11 bits each, so a correctly rounded fp32 quotient falls on a half-way point only when the exact one does,
// and codes are those of exact arithmetic.
// One wave per (page, kv head, keys or values): 16 slots x 128 values are four 16-byte loads per lane, the maximum one
// wave reduction, and nobody else writes the page, so the launch needs no synchronisation.  2900 + 1933 + 967 tokens of 8
// heads (bf16 to 4 bits, 30 MB) take 10.6 us against 5.8 at a copy's rate: a chain of dependent loads (length, row range,
// rows) over barely more waves than the card holds at once (with IEEE divisions for the codes: 14.8).  A decode step of 16
// tokens is that chain: 3.7 us.
//
// kv_gather_kernel.  out = code * scale, rounded once, for rows of consecutive tokens.  A workgroup first finds its rows'
// pages (one thread a row), then copies 8 codes per lane and step: 128-byte (64) code rows in, 256-byte rows out.  Bound by
// memory: 7 prefixes up to 32k tokens (8 bits, 805 MB) take 163-177 us, 4.5-4.9 TB/s; a copy reaches 5.1.

#include <algorithm>

#include "exl3_api.hpp"
#include "kv_device.hpp"

namespace exl3 {

constexpr long long kMaxWaves = 1 << 26;  // of a launch: its threads are counted in 32 bits

struct KvAppendArgs {
  const uint16_t *k, *v;
  long long ld_k, ld_v;
  int rows;
  const int* row_start;
  int rows_per_seq;
  const int *select, *counts;
  int max_new;
  uint8_t *k_cache, *v_cache;
  uint16_t *k_scale, *v_scale;
  int num_pages;
  const int* page_table;
  int max_pages;
  const int* seq_lens;
  int batch, Hkv;
  int pages_each;  // the most pages that max_new tokens touch; 0: places go by rows (append_place)
  long long items;
};

template <bool BF16>
__device__ __forceinline__ float kv_half(uint32_t pair, int e) {  // half e (0, 1) of a pair
  if constexpr (BF16) {
    return __builtin_bit_cast(float, e ? pair & 0xFFFF0000u : pair << 16);
  } else {
    const half2_t h = __builtin_bit_cast(half2_t, pair);
    return (float)h[e];
  }
}

// the smallest fp16 >= a / qmax (a finite, >= 0), the largest finite fp16 past its range
__device__ __forceinline__ uint16_t page_scale(float a, float qmax) {
  const _Float16 h = (_Float16)(a / qmax);
  uint16_t bits = __builtin_bit_cast(uint16_t, h);
  if ((float)h * qmax < a) bits++;  // the product is exact (11 + 7 bits)
  return bits < 0x7C00 ? bits : (uint16_t)0x7BFF;
}

template <int BITS>
__device__ __forceinline__ int kv_code(float x, float s) {
  constexpr float Q = BITS == 8 ? 127.f : 7.f;
  const float r = __builtin_rintf(x / s);
  return r == r ? (int)fminf(fmaxf(r, -Q), Q) : 0;  // NaN: a NaN value, or 0 / 0 in an all-zero page
}

// x / s for finite |x| <= 127 s, r = 1 / s correctly rounded, as the low bits of a float: rint in two's complement.
// The residual of x r is exact, so a half-way quotient comes out as itself; any other is a part of 2^-19 away from
// half-way, more than the quotient's error.
__device__ __forceinline__ uint32_t kv_code_bits(float x, float s, float r) {
  const float y = x * r;
  const float q = __builtin_fmaf(__builtin_fmaf(-y, s, x), r, y);
  return __builtin_bit_cast(uint32_t, q + 12582912.f);  // 1.5 * 2^23: the unit is the last place
}

// By rows: n consecutive rows touch at most n / 16 + 2 pages wherever they begin, so sequence b has the places from
// row_start[b] / 16 + 2 b on.  The last sequence that begins at or before place `at` (-1: none), 64 at a time.
__device__ __forceinline__ int append_place(const int* row_start, int batch, long long at, int lane) {
  int lo = 0, n = batch;
  while (true) {
    const int step = (n + 63) / 64, i = lo + lane * step;
    const bool in = lane * step < n && row_start[min(i, batch)] / kPage + 2LL * i <= at;
    const int before = __builtin_popcountll(__builtin_amdgcn_ballot_w64(in));
    if (before == 0) return -1;
    lo += (before - 1) * step;
    if (step == 1) return lo;
    n = min(step, n - (before - 1) * step);
  }
}

template <int BITS, bool XB>
__global__ __launch_bounds__(256) void kv_append_kernel(const KvAppendArgs a) {
  constexpr float Q = BITS == 8 ? 127.f : 7.f;
  constexpr int ROW = BITS == 8 ? kHeadDim : kHeadDim / 2;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const long long item = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (item >= a.items) return;
  const bool is_v = item & 1;
  const long long pair = item >> 1;  // (sequence, page, kv head)
  const long long at = pair / a.Hkv;
  const int hk = (int)(pair - at * a.Hkv);
  int b, pg;
  if (a.pages_each > 0) {
    b = (int)(at / a.pages_each), pg = (int)(at - (long long)b * a.pages_each);
  } else {
    b = append_place(a.row_start, a.batch, at, lane);
    if (b < 0) return;
    pg = (int)(at - a.row_start[b] / kPage) - 2 * b;
  }
  const int len = max(a.seq_lens[b], 0);
  long long r0 = (long long)b * a.rows_per_seq;
  int avail = a.rows_per_seq;  // rows of the sequence
  if (a.row_start) {
    r0 = a.row_start[b];
    avail = a.row_start[b + 1] - (int)r0;
  }
  int count = a.select ? a.max_new : min(avail, a.max_new);
  if (a.counts) count = min(count, a.counts[b]);
  count = min(count, a.max_pages * kPage - len);  // nothing past the table
  if (count <= 0 || pg < 0 || pg > count / kPage + 1) return;  // (below 0: row starts that do not ascend)
  const int lp = len / kPage + pg, first = lp * kPage;  // logical page, its first token
  if (first >= len + count) return;
  const int page = a.page_table[(size_t)b * a.max_pages + lp];

  const uint16_t* x = is_v ? a.v : a.k;
  const long long ld = is_v ? a.ld_v : a.ld_k;
  constexpr uint32_t INF = XB ? 0x7F80 : 0x7C00;
  kv_u32x4_t raw[4];
  bool live[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int token = first + 4 * i + g - len;  // of the new ones
    live[i] = token >= 0 && token < count;
    long long src = r0;
    if (live[i]) {
      const int node = a.select ? a.select[(size_t)b * a.max_new + token] : token;
      src = r0 + node;
      live[i] = node >= 0 && node < avail && src >= 0 && src < a.rows;
    }
    raw[i] = kv_u32x4_t{0, 0, 0, 0};
    if (live[i]) raw[i] = *reinterpret_cast<const kv_u32x4_t*>(x + src * ld + hk * kHeadDim + 8 * n);
  }
  if (page < 0 || page >= a.num_pages) return;
  if (!__builtin_amdgcn_ballot_w64(live[0] || live[1] || live[2] || live[3])) return;
  // magnitudes of halves order as integers
  uint32_t pairs = 0;
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int e = 0; e < 4; e++) pairs = max_u16x2(pairs, raw[i][e] & 0x7FFF7FFFu);
  const uint32_t largest = wave_max_u32(max(pairs & 0xFFFFu, pairs >> 16));
  float most = kv_half<XB>(largest, 0);
  if (largest >= INF) {  // infinities and NaN take no part
    uint32_t finite = 0;
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const uint32_t lo = raw[i][e] & 0x7FFFu, hi = raw[i][e] >> 16 & 0x7FFFu;
        finite = max(finite, max(lo < INF ? lo : 0, hi < INF ? hi : 0));
      }
    most = kv_half<XB>(wave_max_u32(finite), 0);
  }

  const size_t block = (size_t)page * a.Hkv + hk;
  uint16_t* scale = (is_v ? a.v_scale : a.k_scale) + block;
  uint8_t* codes = (is_v ? a.v_cache : a.k_cache) + block * (kPage * ROW) + n * (ROW / 16);
  uint16_t bits = page_scale(most, Q);
  const int kept = max(len - first, 0);  // older tokens in the page
  const float grown = (float)__builtin_bit_cast(_Float16, bits);
  if (kept > 0) {
    const uint16_t old_bits = *scale;
    const float old = (float)__builtin_bit_cast(_Float16, old_bits);
    if (old >= grown) {
      bits = old_bits;
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (4 * i + g >= kept) continue;
        uint32_t* p = reinterpret_cast<uint32_t*>(codes + (4 * i + g) * ROW);
        if constexpr (BITS == 8) {
#pragma unroll
          for (int d = 0; d < 2; d++) {
            const uint32_t u = p[d];
            uint32_t r = 0;
#pragma unroll
            for (int e = 0; e < 4; e++)
              r |= (uint32_t)(kv_code<8>((float)(int8_t)(u >> (8 * e)) * old, grown) & 0xFF) << (8 * e);
            p[d] = r;
          }
        } else {
          const uint32_t u = p[0];
          uint32_t r = 0;
#pragma unroll
          for (int e = 0; e < 8; e++)
            r |= (uint32_t)(kv_code<4>((float)((int)(u << (28 - 4 * e)) >> 28) * old, grown) & 0xF) << (4 * e);
          p[0] = r;
        }
      }
    }
  }
  const float s = (float)__builtin_bit_cast(_Float16, bits);
  if (lane == 0) *scale = bits;
  // infinities, NaN, a scale that stopped at fp16's largest (or was infinite), 0 / 0: with their limits, else without
  const bool plain = __builtin_amdgcn_readfirstlane(largest < INF && most <= s * Q && s > 0.f && s < __builtin_inff());
  const float r = 1.f / s;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if (!live[i]) continue;
    uint32_t code[8];
    if (plain) {
#pragma unroll
      for (int e = 0; e < 8; e++) code[e] = kv_code_bits(kv_half<XB>(raw[i][e / 2], e & 1), s, r);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) code[e] = (uint32_t)kv_code<BITS>(kv_half<XB>(raw[i][e / 2], e & 1), s);
    }
    uint32_t* p = reinterpret_cast<uint32_t*>(codes + (4 * i + g) * ROW);
    if constexpr (BITS == 8) {
      kv_u32x2_t o;
#pragma unroll
      for (int d = 0; d < 2; d++) {  // the low bytes of four
        const uint32_t lo = __builtin_amdgcn_perm(code[4 * d + 1], code[4 * d], 0x0C0C0400u);
        const uint32_t hi = __builtin_amdgcn_perm(code[4 * d + 3], code[4 * d + 2], 0x04000C0Cu);
        o[d] = lo | hi;
      }
      *reinterpret_cast<kv_u32x2_t*>(p) = o;
    } else {
      uint32_t o = 0;
#pragma unroll
      for (int e = 0; e < 8; e++) o |= (code[e] & 0xF) << (4 * e);
      *p = o;
    }
  }
}

struct KvGatherArgs {
  const uint8_t *k_cache, *v_cache;
  const uint16_t *k_scale, *v_scale;
  int num_pages;
  const int* page_table;
  int max_pages;
  const int *seq_lens, *starts, *row_start;
  int batch, rows, Hkv;
  uint16_t *k_out, *v_out;
};

constexpr int kGatherRows = 16;  // most rows per workgroup (from 8192 rows on; 4 below, for more workgroups)

template <int BITS, bool OB>
__global__ __launch_bounds__(256) void kv_gather_kernel(const KvGatherArgs a, int rows_each) {
  constexpr int ROW = BITS == 8 ? kHeadDim : kHeadDim / 2;
  __shared__ int slot_of[kGatherRows];  // page * 16 + slot (the page in [0, num_pages)), -1: not written
  const int row0 = blockIdx.x * rows_each;
  if ((int)threadIdx.x < rows_each) {
    const int r = row0 + threadIdx.x;
    int slot = -1;
    if (r < a.rows && r >= a.row_start[0] && r < a.row_start[a.batch]) {
      int lo = 0, hi = a.batch;  // row_start[lo] <= r < row_start[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.row_start[mid] <= r)
          lo = mid;
        else
          hi = mid;
      }
      const long long t = (long long)(a.starts ? a.starts[lo] : 0) + r - a.row_start[lo];
      if (t >= 0 && t < min(a.seq_lens[lo], a.max_pages * kPage)) {
        const int page = a.page_table[(size_t)lo * a.max_pages + t / kPage];
        slot = min(max(page, 0), a.num_pages - 1) * kPage + (int)(t % kPage);
      }
    }
    slot_of[threadIdx.x] = slot;
  }
  __syncthreads();
  const int per_row = a.Hkv * 16, items = rows_each * per_row;
#pragma unroll 4
  for (int i = threadIdx.x; i < items; i += 256) {
    const int row = i / per_row, rest = i - row * per_row, hk = rest >> 4, n = rest & 15;
    const int slot = slot_of[row];
    if (slot < 0) continue;
    const size_t block = (size_t)(slot / kPage) * a.Hkv + hk;
    const size_t code_at = block * (kPage * ROW) + (slot % kPage) * ROW + n * (ROW / 16);
    const size_t out_at = ((size_t)(row0 + row) * a.Hkv + hk) * kHeadDim + 8 * n;
#pragma unroll
    for (int kv = 0; kv < 2; kv++) {
      const float s = (float)__builtin_bit_cast(_Float16, (kv ? a.v_scale : a.k_scale)[block]);
      const uint8_t* p = (kv ? a.v_cache : a.k_cache) + code_at;
      float v[8];
      if constexpr (BITS == 8) {
        const kv_u32x2_t u = *reinterpret_cast<const kv_u32x2_t*>(p);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = (float)(int8_t)(u[e / 4] >> (8 * (e & 3))) * s;
      } else {
        const uint32_t u = *reinterpret_cast<const uint32_t*>(p);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = (float)((int)(u << (28 - 4 * e)) >> 28) * s;
      }
      kv_u32x4_t o;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        if constexpr (OB)
          o[e] = (uint32_t)f32_to_bf16(v[2 * e]) | ((uint32_t)f32_to_bf16(v[2 * e + 1]) << 16);
        else
          o[e] = __builtin_bit_cast(uint32_t, half2_t{(_Float16)v[2 * e], (_Float16)v[2 * e + 1]});
      }
      *reinterpret_cast<kv_u32x4_t*>((kv ? a.v_out : a.k_out) + out_at) = o;
    }
  }
}

static int check_cache(const char* what, const void* k_cache, const void* v_cache, const void* k_scale,
                       const void* v_scale, int num_pages, int max_pages, int batch, int num_kv_heads, int head_dim,
                       int page_size, int bits) {
  EXL3_CHECK_ARG(k_cache && v_cache && k_scale && v_scale, "%s: null pointer", what);
  EXL3_CHECK_ARG(head_dim == kHeadDim && page_size == kPage, "%s: head_dim = %d, page_size = %d (supported: 128, 16)",
                 what, head_dim, page_size);
  EXL3_CHECK_ARG(bits == 4 || bits == 8, "%s: bits = %d (4 or 8)", what, bits);
  EXL3_CHECK_ARG(batch >= 0 && num_pages >= 1 && num_pages <= (1 << 26) && max_pages >= 1 && max_pages <= (1 << 26) &&
                     num_kv_heads >= 1 && num_kv_heads <= 65536,
                 "%s: batch = %d, pages = %d, max_pages = %d, kv heads = %d", what, batch, num_pages, max_pages,
                 num_kv_heads);
  EXL3_CHECK_ARG((((uintptr_t)k_cache | (uintptr_t)v_cache) & 15) == 0, "%s: a cache is not 16-byte aligned", what);
  return EXL3_OK;
}

struct Span {
  const void* at;
  size_t bytes;
  bool meets(const Span& o) const {
    const uintptr_t a = (uintptr_t)at, b = (uintptr_t)o.at;
    return at && o.at && a < b + o.bytes && b < a + bytes;
  }
};

}  // namespace exl3

using namespace exl3;

extern "C" int exl3_kv_append(const void* k, const void* v, int x_bf16, long long ld_k, long long ld_v, int rows,
                              const int* row_start, int rows_per_seq, const int* select, const int* counts,
                              int max_new, void* k_cache, void* v_cache, void* k_scale, void* v_scale, int num_pages,
                              const int* page_table, int max_pages, const int* seq_lens, int batch, int num_kv_heads,
                              int head_dim, int page_size, int bits, void* stream) {
  if (const int rc = check_cache("exl3_kv_append", k_cache, v_cache, k_scale, v_scale, num_pages, max_pages, batch,
                                 num_kv_heads, head_dim, page_size, bits))
    return rc;
  EXL3_CHECK_ARG(rows >= 0 && max_new >= 0 && max_new <= (1 << 30),
                 "exl3_kv_append: rows = %d, max_new = %d", rows, max_new);
  if (batch == 0 || rows == 0 || max_new == 0) return EXL3_OK;
  EXL3_CHECK_ARG(k && v && page_table && seq_lens, "exl3_kv_append: null pointer");
  EXL3_CHECK_ARG(row_start || (rows_per_seq >= 1 && (long long)rows_per_seq * batch == rows),
                 "exl3_kv_append: %d rows are not %d sequences of %d", rows, batch, rows_per_seq);
  EXL3_CHECK_ARG(ld_k >= (long long)num_kv_heads * head_dim && ld_v >= (long long)num_kv_heads * head_dim &&
                     ld_k % 8 == 0 && ld_v % 8 == 0 && (((uintptr_t)k | (uintptr_t)v) & 15) == 0,
                 "exl3_kv_append: token strides %lld / %lld (multiples of 8, a token's heads at least; 16-byte aligned)",
                 ld_k, ld_v);
  // a place per page that max_new tokens of each sequence can touch, or, where that is far fewer, that `rows` of them all can
  // (finding a place's sequence takes half a microsecond: 3 sequences, 368 places by rows, 549 else: 10.8 and 10.2 us)
  int pages_each = (int)std::min<long long>(max_pages, ((long long)max_new + 2 * (kPage - 1)) / kPage);
  long long places = (long long)batch * pages_each;
  const long long by_rows = rows / kPage + 2LL * batch;
  if (row_start && !select && 2 * by_rows < places) pages_each = 0, places = by_rows;
  const long long items = 2 * places * num_kv_heads;
  EXL3_CHECK_ARG(items < kMaxWaves, "exl3_kv_append: %d sequences of up to %d new tokens", batch, max_new);
  // what one wave writes, no other may read or write: caches and scales apart from each other and from every input
  const size_t blocks = (size_t)num_pages * num_kv_heads, heads = (size_t)num_kv_heads * head_dim, ints = sizeof(int);
  const size_t code_bytes = blocks * page_size * head_dim * bits / 8;
  const Span all[] = {{k_cache, code_bytes}, {v_cache, code_bytes}, {k_scale, blocks * 2}, {v_scale, blocks * 2},
                      {k, 2 * ((size_t)(rows - 1) * ld_k + heads)}, {v, 2 * ((size_t)(rows - 1) * ld_v + heads)},
                      {page_table, (size_t)batch * max_pages * ints}, {seq_lens, batch * ints},
                      {row_start, (batch + (size_t)1) * ints}, {select, (size_t)batch * max_new * ints},
                      {counts, batch * ints}};
  for (int i = 0; i < 4; i++)
    for (int j = i + 1; j < (int)(sizeof(all) / sizeof(all[0])); j++)
      EXL3_CHECK_ARG(!all[i].meets(all[j]), "exl3_kv_append: a cache or its scales overlap another tensor of the call");
  const KvAppendArgs a{static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), ld_k, ld_v, rows, row_start,
                       rows_per_seq, select, counts, max_new, static_cast<uint8_t*>(k_cache),
                       static_cast<uint8_t*>(v_cache), static_cast<uint16_t*>(k_scale),
                       static_cast<uint16_t*>(v_scale), num_pages, page_table, max_pages, seq_lens, batch,
                       num_kv_heads, pages_each, items};
  auto kern = bits == 8 ? (x_bf16 ? kv_append_kernel<8, true> : kv_append_kernel<8, false>)
                        : (x_bf16 ? kv_append_kernel<4, true> : kv_append_kernel<4, false>);
  kern<<<(unsigned)((items + 3) / 4), 256, 0, as_stream(stream)>>>(a);
  EXL3_CHECK_LAUNCH();
  return EXL3_OK;
}

extern "C" int exl3_kv_gather(const void* k_cache, const void* v_cache, const void* k_scale, const void* v_scale,
                              int num_pages, const int* page_table, int max_pages, const int* seq_lens,
                              const int* starts, const int* row_start, int batch, int rows, int num_kv_heads,
                              int head_dim, int page_size, int bits, void* k_out, void* v_out, int out_bf16,
                              void* stream) {
  if (const int rc = check_cache("exl3_kv_gather", k_cache, v_cache, k_scale, v_scale, num_pages, max_pages, batch,
                                 num_kv_heads, head_dim, page_size, bits))
    return rc;
  EXL3_CHECK_ARG(rows >= 0 && rows < (1 << 28), "exl3_kv_gather: rows = %d", rows);
  if (batch == 0 || rows == 0) return EXL3_OK;
  EXL3_CHECK_ARG(page_table && seq_lens && row_start && k_out && v_out, "exl3_kv_gather: null pointer");
  EXL3_CHECK_ARG((((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0, "exl3_kv_gather: an output is not 16-byte aligned");
  const KvGatherArgs a{static_cast<const uint8_t*>(k_cache), static_cast<const uint8_t*>(v_cache),
                       static_cast<const uint16_t*>(k_scale), static_cast<const uint16_t*>(v_scale), num_pages,
                       page_table, max_pages, seq_lens, starts, row_start, batch, rows, num_kv_heads,
                       static_cast<uint16_t*>(k_out), static_cast<uint16_t*>(v_out)};
  const int rows_each = rows >= 8192 ? kGatherRows : 4;
  auto kern = bits == 8 ? (out_bf16 ? kv_gather_kernel<8, true> : kv_gather_kernel<8, false>)
                        : (out_bf16 ? kv_gather_kernel<4, true> : kv_gather_kernel<4, false>);
  kern<<<(unsigned)((rows + (long long)rows_each - 1) / rows_each), 256, 0, as_stream(stream)>>>(a, rows_each);
  EXL3_CHECK_LAUNCH();
  return EXL3_OK;
}
