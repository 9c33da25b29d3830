// Tokens from logits by temperature, top-k, top-p and min-p, from given random numbers, and the distribution that they are
// drawn from (gfx950).
//
// A row's logits l (NaN counts as -inf) of largest M, temperature t:  w = exp((l - M) / t).  In the order of falling logits,
// ties by rising index, three rules each keep a beginning of the row, and the shortest stands:
//   top-k  the first k;
//   top-p  the elements whose predecessors have less than p of the first k's sum of w;
//   min-p  those with w >= m;
// and always the first element.  So what is kept is known from its last element, the cut (its logit, its index).
// The token is the smallest v whose running sum of w over the kept passes u times their sum; its row of probabilities is w over
// that sum, 0 elsewhere.  t = 0 (or no number) keeps the first element alone.
//
// Weights are 64-bit.  Where atomics sum them (in LDS) they are integers, so that no result depends on an order, in units of
// 2^-50 of a chunk's largest weight or 2^-42 to 2^-52 of the row's: another summation decides differently only where a
// threshold lies within some 10^-12 of the total of an edge.
//
// sample_chunk_kernel: (chunks of 8192 elements, rows) workgroups.  A chunk's largest logit m, its sum of exp((l - m) / t), and
//   counts and sums in 256 bins an eighth of an octave of w wide.  An element's bin is a monotone function of its logit alone,
//   so the chunks' bins match, and an element of a lower bin comes before every one of a higher.
// sample_row_kernel: a workgroup per row adds the bins up and so knows the bins that each rule's last element is in.  Only
//   their elements (some hundreds) are looked at one by one, in LDS: the cut comes from histograms of ever smaller ranges.
//   Then the chunk, and in it the element, where the running sum passes the threshold.  Rows so flat that those bins hold more
//   than the list takes go through the same search over the whole row instead.
// sample_probs_kernel: (chunks, rows) workgroups write the probabilities.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "exl3_api.hpp"
#include "exl3_device.hpp"
#include "kv_device.hpp"

namespace exl3 {

typedef unsigned long long u64_t;
typedef uint32_t sample_u32x4_t __attribute__((ext_vector_type(4), aligned(2)));  // rows start at any element

constexpr int kMaxVocab = 1 << 20;
constexpr int kChunk = 8192;                     // elements of a chunk
constexpr int kMaxChunks = kMaxVocab / kChunk;
constexpr int kChunkThreads = 1024;
constexpr int kEach = kChunk / kChunkThreads;    // 8 elements a thread
constexpr int kBins = 256;
constexpr int kRowThreads = 1024;
constexpr int kRowWaves = kRowThreads / 64;
constexpr int kCrossBins = 1024;
constexpr int kList = 4096;
constexpr double kBinUnit = 0x1p-50;             // a bin's sum is in 2^-50 of the chunk's largest weight
constexpr double kBinBase = 0x1p52 * kBinUnit;

struct SampleChunk {
  double sum;    // of exp((l - m) / t)
  float m, top;  // the largest logit, its place on the bins' scale
};
struct SampleCut {
  uint32_t key;  // of the last kept element
  int at;        // its index
  double min_w;  // what a kept weight is not below
  double inv;    // 1 / the sum of the kept weights; 0: no logit above -inf
  float m;       // the row's largest logit
};

struct SampleArgs {
  const void* logits;
  long long ld;
  int rows, vocab, shift;                              // the row's weights are summed in units of 2^-shift
  const float *uniform, *temperature, *top_p, *min_p;  // NULL: the value for every row
  const int* top_k;
  double all_temperature, all_top_p, all_min_p;
  int all_top_k;
  int* tokens;
  float* probs;
  int chunks;
  SampleChunk* chunk;  // [rows][chunks]
  u64_t* bin_mass;     // [rows][chunks][kBins]
  int* bin_count;      // [rows][chunks][kBins]
  SampleCut* cuts;     // [rows]
};

// A row's rules, and the scales of its weights (2^(scale (l - M))) and bins
struct SampleRules {
  double scale, p, m;
  float bin_scale;
  int k;
};

__device__ __forceinline__ SampleRules sample_rules(const SampleArgs& a, int row) {
  SampleRules r;
  double t = a.temperature ? (double)a.temperature[row] : a.all_temperature;
  r.p = a.top_p ? (double)a.top_p[row] : a.all_top_p;
  r.m = a.min_p ? (double)a.min_p[row] : a.all_min_p;
  r.k = a.top_k ? a.top_k[row] : a.all_top_k;
  if (!(t > 0.0)) t = 1.0, r.k = 1;
  if (r.k <= 0 || r.k > a.vocab) r.k = a.vocab;
  r.p = r.p < 1.0 ? fmax(r.p, 0.0) : 1.0;  // NaN: all
  r.m = r.m > 0.0 ? fmin(r.m, 1.0) : 0.0;
  r.scale = 1.4426950408889634074 / t;
  // any positive number makes the bins a monotone function of the logit
  r.bin_scale = (float)fmin(fmax(8.0 * r.scale, 0x1p-126), 0x1p60);
  return r;
}

// An element's place on the bins' scale, an integer; bin = the largest element's place - its own, 255 at most
__device__ __forceinline__ float sample_place(float l, float bin_scale) {
  return __builtin_floorf(__builtin_amdgcn_fmed3f(l * bin_scale, -0x1p126f, 0x1p126f));
}
__device__ __forceinline__ int sample_bin(float l, float bin_scale, float top) {
  return (int)fminf(top - sample_place(l, bin_scale), (float)(kBins - 1));
}

// ln(2)^i / i!, a constant (a constexpr function called in device code is computed there)
template <int I>
struct Exp2Term {
  static constexpr double value = Exp2Term<I - 1>::value * 0.69314718055994530942 / I;
};
template <>
struct Exp2Term<0> {
  static constexpr double value = 1.0;
};

// 2^t for t <= 0: 2^k exp(r ln 2) with |r| <= 1/2 by the series (the first term left out is below 2 * 10^-16); below 2^-1000 the
// same (far below every unit that weights are summed in)
__device__ __forceinline__ double exp2_f64(double t) {
  t = fmax(t, -1000.0);  // NaN (-inf at a scale of 0) too
  const double k = __builtin_rint(t), r = t - k;
  double p = Exp2Term<12>::value;
#define EXL3_TERM(i) p = __builtin_fma(p, r, Exp2Term<i>::value);
  EXL3_TERM(11) EXL3_TERM(10) EXL3_TERM(9) EXL3_TERM(8) EXL3_TERM(7) EXL3_TERM(6) EXL3_TERM(5) EXL3_TERM(4) EXL3_TERM(3)
  EXL3_TERM(2) EXL3_TERM(1) EXL3_TERM(0)
#undef EXL3_TERM
  return __builtin_amdgcn_ldexp(p, (int)k);
}

// the weight of l where the largest logit is m (> -inf)
__device__ __forceinline__ double sample_weight(float l, float m, double scale) {
  return exp2_f64(l == m ? 0.0 : ((double)l - (double)m) * scale);
}

// rint(w / unit) for 0 <= w <= 1: added to base = 2^52 unit (1 at least), w's last place is the unit
__device__ __forceinline__ u64_t sample_units(double w, double base) {
  return __builtin_bit_cast(u64_t, w + base) - __builtin_bit_cast(u64_t, base);
}

__device__ __forceinline__ uint32_t sample_key(float f) {  // orders like the logits, both zeros the same
  const uint32_t u = __builtin_bit_cast(uint32_t, f + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float sample_logit(uint32_t key) {
  return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

template <int TYPE>
__device__ __forceinline__ float sample_value(uint32_t bits) {
  float f;
  if constexpr (TYPE == EXL3_F32)
    f = __builtin_bit_cast(float, bits);
  else if constexpr (TYPE == EXL3_BF16)
    f = __builtin_bit_cast(float, bits << 16);
  else
    f = (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
  return f == f ? f : -INFINITY;
}

template <int TYPE>
struct SampleRow {
  using Raw = std::conditional_t<TYPE == EXL3_F32, uint32_t, uint16_t>;
  static constexpr int VEC = 16 / sizeof(Raw);  // elements of a 16-byte load
  const Raw* row;
  int vocab;

  __device__ __forceinline__ float at(int i) const { return sample_value<TYPE>(row[i]); }
  // elements i .. i + VEC - 1, -inf past the row; `whole` (uniform): none is
  __device__ __forceinline__ void get(int i, bool whole, float v[VEC]) const {
    if (whole || i + VEC <= vocab) {
      const sample_u32x4_t r = *reinterpret_cast<const sample_u32x4_t*>(row + i);
#pragma unroll
      for (int e = 0; e < VEC; e++)
        v[e] = sample_value<TYPE>(TYPE == EXL3_F32 ? r[e % 4] : (r[e / 2 % 4] >> (16 * (e & 1))) & 0xFFFFu);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; e++) v[e] = i + e < vocab ? at(i + e) : -INFINITY;
    }
  }
};

template <int TYPE>
__device__ __forceinline__ SampleRow<TYPE> sample_row(const SampleArgs& a, int row) {
  using Row = SampleRow<TYPE>;
  return Row{static_cast<const typename Row::Raw*>(a.logits) + (size_t)row * a.ld, a.vocab};
}

template <int TYPE>
__global__ __launch_bounds__(kChunkThreads) void sample_chunk_kernel(const SampleArgs a) {
  constexpr int VEC = SampleRow<TYPE>::VEC, WAVES = kChunkThreads / 64;
  __shared__ u64_t mass[kBins];
  __shared__ int count[kBins];
  __shared__ float part[WAVES];
  __shared__ double sums[WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = blockIdx.x, row = blockIdx.y;
  const SampleRow<TYPE> x = sample_row<TYPE>(a, row);
  const SampleRules rules = sample_rules(a, row);
  const bool bins = rules.k < a.vocab || rules.p < 1.0 || rules.m > 0.0;
  const int first = c * kChunk;
  float l[kEach];
  const bool whole = first + kChunk <= a.vocab;
  if (whole) {
#pragma unroll
    for (int j = 0; j < kEach / VEC; j++) x.get(first + (j * kChunkThreads + tid) * VEC, true, l + j * VEC);
  } else {
#pragma unroll
    for (int j = 0; j < kEach / VEC; j++) x.get(first + (j * kChunkThreads + tid) * VEC, false, l + j * VEC);
  }
  if (bins && tid < kBins) mass[tid] = 0, count[tid] = 0;
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < kEach; i++) m = fmaxf(m, l[i]);
#pragma unroll
  for (int d = 1; d < 64; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
  if (lane == 0) part[wave] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; w++) m = fmaxf(m, part[w]);
  const size_t at = (size_t)row * a.chunks + c;
  const float top = sample_place(m, rules.bin_scale);
  double sum = 0.0;
  if (m > -INFINITY) {
#pragma unroll
    for (int i = 0; i < kEach; i++) {
      if (i % 4 == 0) __builtin_amdgcn_sched_barrier(0);  // four chains at a time: all sixteen do not fit the registers
      const double w = sample_weight(l[i], m, rules.scale);
      const bool in = whole || first + (i / VEC * kChunkThreads + tid) * VEC + i % VEC < a.vocab;
      sum += in ? w : 0.0;
      if (bins && in) {
        const int bin = sample_bin(l[i], rules.bin_scale, top);
        atomicAdd(&count[bin], 1);
        atomicAdd(&mass[bin], sample_units(w, kBinBase));
      }
    }
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
  if (lane == 0) sums[wave] = sum;
  __syncthreads();
  if (tid == 0) {
    sum = 0.0;
    for (int w = 0; w < WAVES; w++) sum += sums[w];
    a.chunk[at] = SampleChunk{sum, m, top};
  }
  if (bins && tid < kBins) {
    a.bin_mass[at * kBins + tid] = mass[tid];
    a.bin_count[at * kBins + tid] = count[tid];
  }
}

struct SampleShared {
  u64_t list[kList];  // key << 32 | ~index
  u64_t hist[kCrossBins], part[kRowWaves], chunk_mass[kMaxChunks];
  double cum_mass[kBins + 1], factor[kMaxChunks], red[4][kBins], sum;
  int cum_count[kBins + 1], red_count[4][kBins];
  float shift[kMaxChunks];
  uint32_t key[kRowWaves];
  u64_t before;
  int bin, listed, k_bin, p_first, p_last, token, last;
};

__device__ __forceinline__ u64_t shfl_up_u64(u64_t v, int d) {
  const uint32_t lo = __shfl_up((int)(uint32_t)v, d), hi = __shfl_up((int)(uint32_t)(v >> 32), d);
  return (u64_t)hi << 32 | lo;
}

// sum before this thread, and of all
__device__ __forceinline__ u64_t row_scan(u64_t v, u64_t& total, SampleShared& sh) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  u64_t s = v;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const u64_t o = shfl_up_u64(s, d);
    s += lane >= d ? o : 0;
  }
  __syncthreads();
  if (lane == 63) sh.part[wave] = s;
  __syncthreads();
  u64_t before = 0;
  total = 0;
  for (int w = 0; w < kRowWaves; w++) {
    before += w < wave ? sh.part[w] : 0;
    total += sh.part[w];
  }
  return before + s - v;
}

// Of the elements i < n with a value get(i, value, mass) in [lo, hi]: the value at which their masses, summed from hi down, reach
// `target` (at least 1, at most their sum); target becomes what is left of it for that value.  Every pass leaves a range of
// 1/1024 of the one before.
template <class Get>
__device__ uint32_t row_cross(int n, uint32_t lo, uint32_t hi, u64_t& target, SampleShared& sh, Get get) {
  while (lo < hi) {
    const uint32_t span = hi - lo;
    const int shift = max(0, 32 - __builtin_clz(span) - 10);
    __syncthreads();
    for (int i = threadIdx.x; i < kCrossBins; i += kRowThreads) sh.hist[i] = 0;
    if (threadIdx.x == 0) sh.bin = 0, sh.before = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kRowThreads) {
      uint32_t v;
      u64_t m;
      if (get(i, lo, hi, v, m)) atomicAdd(&sh.hist[(hi - v) >> shift], m);
    }
    __syncthreads();
    u64_t total;
    const u64_t here = sh.hist[threadIdx.x], before = row_scan(here, total, sh);
    if (before < target && before + here >= target) sh.bin = threadIdx.x, sh.before = before;
    __syncthreads();
    target -= sh.before;
    hi -= min((uint32_t)sh.bin, span >> shift) << shift;
    const uint32_t size = (1u << shift) - 1;
    lo = hi - lo > size ? hi - size : lo;
  }
  __syncthreads();
  return hi;
}

template <int TYPE>
__global__ __launch_bounds__(kRowThreads) void sample_row_kernel(const SampleArgs a) {
  constexpr int VEC = SampleRow<TYPE>::VEC;
  __shared__ SampleShared sh;
  const int row = blockIdx.x, tid = threadIdx.x, V = a.vocab, C = a.chunks;
  const SampleRow<TYPE> x = sample_row<TYPE>(a, row);
  const SampleRules rules = sample_rules(a, row);
  const bool by_k = rules.k < V, by_p = rules.p < 1.0, by_m = rules.m > 0.0;
  const SampleChunk* chunk = a.chunk + (size_t)row * C;

  float M = -INFINITY, top = -INFINITY;
  for (int c = tid; c < C; c += kRowThreads) M = fmaxf(M, chunk[c].m), top = fmaxf(top, chunk[c].top);
  // (C <= 128: the first two waves hold them; a key orders like its float)
  auto most = [&](float f) {
    const uint32_t v = wave_max_u32(sample_key(f));
    __syncthreads();
    if ((tid & 63) == 0) sh.key[tid >> 6] = v;
    __syncthreads();
    return sample_logit(max(sh.key[0], sh.key[1]));
  };
  M = most(M);
  if (!(M > -INFINITY)) {  // nothing to draw from
    if (tid == 0) {
      if (a.tokens) a.tokens[row] = -1;
      if (a.cuts) a.cuts[row] = SampleCut{0, 0, 0.0, 0.0, M};
    }
    return;
  }
  top = most(top);
  const double one = (double)(1ull << a.shift);
  auto weight = [&](float l) { return sample_weight(l, M, rules.scale); };
  const double base = (double)(1ull << (52 - a.shift));
  auto mass = [&](float l) { return sample_units(weight(l), base); };
  auto bin_of = [&](float l) { return sample_bin(l, rules.bin_scale, top); };
  for (int c = tid; c < C; c += kRowThreads) {
    sh.factor[c] = chunk[c].m > -INFINITY ? weight(chunk[c].m) : 0.0;
    sh.shift[c] = fminf(top - chunk[c].top, (float)kBins);
  }
  if (tid == 0) sh.listed = 0;
  __syncthreads();
  if (tid < 64) {  // in a fixed order
    double s = 0.0;
    for (int c = tid; c < C; c += 64) s += sh.factor[c] * chunk[c].sum;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) s += __shfl_xor(s, d);
    if (tid == 0) sh.sum = s;
  }
  __syncthreads();
  const double sum_all = sh.sum;

  // the cut: the last kept element's key and index, and a bound on kept weights
  uint32_t cut = 0;
  int cut_at = V - 1;
  auto before_cut = [&](uint32_t key, int i) { return key > cut || (key == cut && i <= cut_at); };
  auto kept = [&](float l, int i) {
    return before_cut(sample_key(l), i) && (!by_m || weight(l) >= rules.m);
  };
  // the first `count` elements of key `at` by index, among the elements get(i, key, index) for i < n
  auto cut_ties = [&](int n, uint32_t at, u64_t count, auto get) {
    const uint32_t last = ~0u - (uint32_t)(V - 1);
    const uint32_t v = row_cross(n, last, ~0u, count, sh, [&](int i, uint32_t lo, uint32_t hi, uint32_t& v, u64_t& m) {
      uint32_t key;
      int index;
      get(i, key, index);
      v = ~(uint32_t)index, m = 1;
      return key == at && v >= lo && v <= hi;
    });
    cut = at, cut_at = (int)~v;
  };
  // of the sum of get's masses
  auto sum_of = [&](int n, auto get) {
    u64_t sum = 0, total;
    for (int i = tid; i < n; i += kRowThreads) sum += get(i);
    row_scan(sum, total, sh);
    return total;
  };

  // ---- from the bins: where each rule's last element is
  int g_first = kBins, g_last = kBins - 1, k_bin = -1, p_first = 0, p_last = kBins - 1;
  int listed = 0;
  if (by_k || by_p || by_m) {
    const int bin = tid & (kBins - 1), quarter = tid / kBins;
    double s = 0.0;
    int n = 0;
    if (bin < kBins - 1)
      for (int c = quarter; c < C; c += 4) {
        const int local = bin - (int)sh.shift[c];
        if (local < 0) continue;
        const size_t at = ((size_t)row * C + c) * kBins + local;
        s += sh.factor[c] * (double)a.bin_mass[at];
        n += a.bin_count[at];
      }
    sh.red[quarter][bin] = s, sh.red_count[quarter][bin] = n;
    __syncthreads();
    u64_t all;
    n = 0, s = 0.0;
    if (tid < kBins) {
#pragma unroll
      for (int i = 0; i < 4; i++) s += sh.red[i][tid], n += sh.red_count[i][tid];
      s *= kBinUnit;
    }
    const int before = (int)row_scan((u64_t)n, all, sh);
    // sums of the bins before, in a fixed order: inside each wave, then the waves'
    double run = s;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const double o = __shfl_up(run, d);
      run += (tid & 63) >= d ? o : 0.0;
    }
    if ((tid & 63) == 63 && tid < kBins) sh.red[0][tid >> 6] = run;
    __syncthreads();
    if (tid < kBins) {
      double base = 0.0;
      for (int w = 0; w < tid >> 6; w++) base += sh.red[0][w];
      sh.cum_mass[tid + 1] = base + run;
      sh.cum_count[tid + 1] = before + n;
    }
    if (tid == 0) sh.cum_mass[0] = 0.0, sh.cum_count[0] = 0, sh.k_bin = kBins - 1, sh.p_first = kBins - 1, sh.p_last = 0;
    __syncthreads();
    if (tid == 0) sh.cum_mass[kBins] = fmax(sum_all, sh.cum_mass[kBins]), sh.cum_count[kBins] = V;  // the last bin: the rest
    __syncthreads();
    if (by_k && tid < kBins && sh.cum_count[tid] < rules.k && sh.cum_count[tid + 1] >= rules.k) sh.k_bin = tid;
    __syncthreads();
    if (by_k) k_bin = sh.k_bin;
    if (by_p) {
      // a bin's sum is off by half a unit an element, the threshold by the part of the first k in their last bin
      const double slack = (double)V * kBinUnit + 1e-13 * sum_all;
      const double lo = rules.p * (by_k ? sh.cum_mass[k_bin] : sum_all) - slack;
      const double hi = rules.p * (by_k ? sh.cum_mass[k_bin + 1] : sum_all) + slack;
      if (tid < kBins) {
        if (sh.cum_mass[tid + 1] >= lo) atomicMin(&sh.p_first, tid);
        if (sh.cum_mass[tid] < hi) atomicMax(&sh.p_last, tid);
      }
      __syncthreads();
      p_first = sh.p_first, p_last = max(sh.p_first, sh.p_last);
      g_first = min(g_first, p_first), g_last = min(g_last, p_last);
    }
    if (by_m) {
      // w >= m from the logit M + log2(m) / scale on; places are off by a few 2^-24 of themselves
      const double y = (double)M * rules.bin_scale + log2(rules.m) * (rules.bin_scale / rules.scale);
      const double e = 0.01 + fabs(y) * 1e-6 + fabs((double)M * rules.bin_scale) * 1e-6;
      const double lo = (double)top - floor(y + e), hi = (double)top - floor(y - e);
      const bool far = !(e < 64.0);  // (infinite M too)
      g_first = min(g_first, far ? 0 : (int)fmin(fmax(lo, 0.0), kBins - 1.0));
      g_last = min(g_last, far ? kBins - 1 : (int)fmin(fmax(hi, 0.0), kBins - 1.0));
    }
    if (by_k) {
      if (!by_p && k_bin > g_last) k_bin = -1;  // min-p stops before
      else g_first = min(g_first, k_bin), g_last = min(g_last, k_bin);
    }
    listed = sh.cum_count[g_last + 1] - sh.cum_count[g_first];
    const bool apart = k_bin > g_last;  // its elements are listed too
    if (apart) listed += sh.cum_count[k_bin + 1] - sh.cum_count[k_bin];
    if (listed <= kList) {
      for (int i = tid * VEC; i < V; i += kRowThreads * VEC) {
        float l[VEC];
        x.get(i, false, l);
#pragma unroll
        for (int e = 0; e < VEC; e++) {
          const int b = bin_of(l[e]);
          if (((b >= g_first && b <= g_last) || b == k_bin) && i + e < V)
            sh.list[atomicAdd(&sh.listed, 1)] = (u64_t)sample_key(l[e]) << 32 | (uint32_t)~(i + e);
        }
      }
      __syncthreads();
    }
  }
  const bool fast = listed <= kList;

  // ---- the cut
  const uint32_t largest = sample_key(M);
  auto element = [&](int i, uint32_t& key, int& index) {
    if (fast) {
      const u64_t v = sh.list[i];
      key = (uint32_t)(v >> 32), index = (int)~(uint32_t)v;
    } else {
      key = sample_key(x.at(i)), index = i;
    }
  };
  const int n = fast ? listed : V;
  if (by_k && (!fast || k_bin >= 0)) {
    u64_t target = fast ? rules.k - sh.cum_count[k_bin] : rules.k;
    const uint32_t at = row_cross(n, 0, largest, target, sh, [&](int i, uint32_t lo, uint32_t hi, uint32_t& v, u64_t& m) {
      int index;
      element(i, v, index);
      m = 1;
      return v >= lo && v <= hi && (!fast || bin_of(sample_logit(v)) == k_bin);
    });
    cut_ties(n, at, target, element);
  }
  if (by_p) {
    u64_t target = 0, most = 0;
    if (fast) {
      double total = sum_all;
      if (by_k)
        total = sh.cum_mass[k_bin] + (double)sum_of(n, [&](int i) -> u64_t {
                  uint32_t key;
                  int index;
                  element(i, key, index);
                  const float l = sample_logit(key);
                  return bin_of(l) == k_bin && before_cut(key, index) ? mass(l) : 0;
                }) / one;
      most = sum_of(n, [&](int i) -> u64_t {
        uint32_t key;
        int index;
        element(i, key, index);
        const float l = sample_logit(key);
        const int b = bin_of(l);
        return b >= p_first && b <= p_last && before_cut(key, index) ? mass(l) : 0;
      });
      const double bar = __builtin_ceil((rules.p * total - sh.cum_mass[p_first]) * one);
      target = bar >= 1.0 ? min((u64_t)bar, most) : 1;
    } else {
      most = sum_of(V, [&](int i) -> u64_t {
        const float l = x.at(i);
        return before_cut(sample_key(l), i) ? mass(l) : 0;
      });
      const double bar = __builtin_ceil(rules.p * (double)most);
      target = bar >= 1.0 ? min((u64_t)bar, most) : 1;
    }
    if (most > 0) {
      const uint32_t at = row_cross(n, cut, largest, target, sh, [&](int i, uint32_t lo, uint32_t hi, uint32_t& v, u64_t& m) {
        int index;
        element(i, v, index);
        if (v < lo || v > hi || !before_cut(v, index)) return false;
        const float l = sample_logit(v);
        if (fast) {
          const int b = bin_of(l);
          if (b < p_first || b > p_last) return false;
        }
        m = mass(l);
        return true;
      });
      const u64_t each = mass(sample_logit(at));
      if (each > 0) cut_ties(n, at, (target + each - 1) / each, element);
    }
  }

  // ---- the token
  u64_t total = 0;
  const float u = a.uniform ? a.uniform[row] : 0.f;
  auto threshold = [&]() {  // the smallest whole number above u times the sum
    const double bar = (u > 0.f ? (double)u : 0.0) * (double)total;
    return bar < (double)total ? min((u64_t)bar + 1, total) : total;
  };
  if (!fast) {
    total = sum_of(V, [&](int i) -> u64_t {
      const float l = x.at(i);
      return kept(l, i) ? mass(l) : 0;
    });
    if (a.tokens) {
      u64_t target = threshold();
      const uint32_t last = ~0u - (uint32_t)(V - 1);
      const uint32_t v = row_cross(V, last, ~0u, target, sh, [&](int i, uint32_t lo, uint32_t hi, uint32_t& v, u64_t& m) {
        v = ~(uint32_t)i;
        if (v < lo || v > hi) return false;
        const float l = x.at(i);
        if (!kept(l, i)) return false;
        m = mass(l);
        return true;
      });
      if (tid == 0) a.tokens[row] = (int)~v;
    }
  } else {
    // each chunk's kept sum: its bins before g_first, and its listed elements
    for (int c = tid >> 6; c < C; c += kRowWaves) {
      double s = 0.0;
      if (g_first == kBins) {
        s = chunk[c].sum;
      } else {
        const int end = g_first - (int)sh.shift[c];
        for (int b = tid & 63; b < end; b += 64) s += (double)a.bin_mass[((size_t)row * C + c) * kBins + b];
#pragma unroll
        for (int d = 1; d < 64; d *= 2) s += __shfl_xor(s, d);
        s *= kBinUnit;
      }
      if ((tid & 63) == 0) sh.chunk_mass[c] = (u64_t)__builtin_rint(s * sh.factor[c] * one);
    }
    __syncthreads();
    for (int i = tid; i < n; i += kRowThreads) {
      uint32_t key;
      int index;
      element(i, key, index);
      const float l = sample_logit(key);
      if (bin_of(l) <= g_last && kept(l, index)) atomicAdd(&sh.chunk_mass[index / kChunk], mass(l));
    }
    __syncthreads();
    const u64_t here = tid < C ? sh.chunk_mass[tid] : 0;
    const u64_t before = row_scan(here, total, sh);
    if (a.tokens) {
      const u64_t target = threshold();
      if (tid == 0) sh.bin = 0, sh.before = 0, sh.token = V, sh.last = -1;
      __syncthreads();
      if (here > 0 && before < target && before + here >= target) sh.bin = tid, sh.before = before;
      __syncthreads();
      const u64_t left = target - sh.before;
      const int i0 = sh.bin * kChunk + tid * (kChunk / kRowThreads);
      u64_t w[kChunk / kRowThreads], sum = 0, all;
#pragma unroll
      for (int j = 0; j < kChunk / kRowThreads / VEC; j++) {
        float l[VEC];
        x.get(i0 + j * VEC, false, l);
#pragma unroll
        for (int e = 0; e < VEC; e++) {
          const int i = i0 + j * VEC + e;
          w[j * VEC + e] = i < V && kept(l[e], i) ? mass(l[e]) : 0;
          sum += w[j * VEC + e];
        }
      }
      u64_t run = row_scan(sum, all, sh);
      int found = V, last = -1;
#pragma unroll
      for (int j = 0; j < kChunk / kRowThreads; j++) {
        run += w[j];
        if (w[j] > 0) {
          last = i0 + j;
          if (run >= left) found = min(found, i0 + j);
        }
      }
      if (found < V) atomicMin(&sh.token, found);
      if (last >= 0) atomicMax(&sh.last, last);  // rounding may leave the threshold to nobody
      __syncthreads();
      if (tid == 0) a.tokens[row] = sh.token < V ? sh.token : sh.last;
    }
  }
  if (a.cuts && tid == 0) a.cuts[row] = SampleCut{cut, cut_at, by_m ? rules.m : 0.0, one / (double)total, M};
}

template <int TYPE>
__global__ __launch_bounds__(kChunkThreads) void sample_probs_kernel(const SampleArgs a) {
  constexpr int VEC = SampleRow<TYPE>::VEC;
  typedef float f4_t __attribute__((ext_vector_type(4), aligned(4)));
  const int row = blockIdx.y;
  const SampleRow<TYPE> x = sample_row<TYPE>(a, row);
  const SampleCut cut = a.cuts[row];
  const double scale = sample_rules(a, row).scale;
  float* out = a.probs + (size_t)row * a.vocab;
#pragma unroll
  for (int j = 0; j < kEach / VEC; j++) {
    const int i = blockIdx.x * kChunk + (j * kChunkThreads + (int)threadIdx.x) * VEC;
    float l[VEC], p[VEC];
    x.get(i, false, l);
#pragma unroll
    for (int e = 0; e < VEC; e++) {
      const uint32_t key = sample_key(l[e]);
      p[e] = 0.f;
      if (cut.inv > 0.0 && (key > cut.key || (key == cut.key && i + e <= cut.at))) {
        const double w = sample_weight(l[e], cut.m, scale);
        p[e] = w >= cut.min_w ? (float)(w * cut.inv) : 0.f;
      }
    }
    if (i + VEC <= a.vocab) {
#pragma unroll
      for (int e = 0; e < VEC; e += 4) *reinterpret_cast<f4_t*>(out + i + e) = f4_t{p[e], p[e + 1], p[e + 2], p[e + 3]};
    } else {
#pragma unroll
      for (int e = 0; e < VEC; e++)
        if (i + e < a.vocab) out[i + e] = p[e];
    }
  }
}

static size_t sample_chunk_bytes(int rows, int vocab) {
  const size_t chunks = (vocab + kChunk - 1) / kChunk;
  return rows * chunks * (sizeof(SampleChunk) + kBins * (sizeof(u64_t) + sizeof(int)));
}

}  // namespace exl3

using namespace exl3;

extern "C" size_t exl3_sample_workspace_bytes(int rows, int vocab) {
  if (rows <= 0 || vocab <= 0 || vocab > kMaxVocab) return 0;
  return sample_chunk_bytes(rows, vocab) + rows * sizeof(SampleCut);
}

extern "C" int exl3_sample(const void* logits, int type, long long ld, int rows, int vocab, const float* uniform,
                           const float* temperature, double all_temperature, const int* top_k, int all_top_k,
                           const float* top_p, double all_top_p, const float* min_p, double all_min_p, int* tokens, float* probs,
                           void* workspace, size_t workspace_bytes, void* stream) {
  EXL3_CHECK_ARG(rows >= 0 && rows <= 65535 && vocab >= 1 && vocab <= kMaxVocab,
                 "exl3_sample: rows = %d (up to 65535), vocab = %d (1 to %d)", rows, vocab, kMaxVocab);
  EXL3_CHECK_ARG(type >= EXL3_F16 && type <= EXL3_F32, "exl3_sample: logits type %d", type);
  if (rows == 0) return EXL3_OK;
  EXL3_CHECK_ARG(tokens || probs, "exl3_sample: neither tokens nor probabilities");
  EXL3_CHECK_ARG(!tokens || uniform, "exl3_sample: tokens need random numbers");
  const size_t bytes = type == EXL3_F32 ? 4 : 2;
  EXL3_CHECK_ARG(logits && ld >= vocab && (uintptr_t)logits % bytes == 0,
                 "exl3_sample: logits are null, not aligned to their type, or their rows overlap (stride %lld)", ld);
  const size_t n = rows, need = exl3_sample_workspace_bytes(rows, vocab);
  EXL3_CHECK_ARG(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0,
                 "exl3_sample: workspace %zu bytes, need %zu (16-byte aligned)", workspace_bytes, need);
  const Span all[] = {{tokens, n * 4}, {probs, n * vocab * 4}, {workspace, need}, {logits, ((n - 1) * ld + vocab) * bytes},
                      {uniform, n * 4}, {temperature, n * 4}, {top_k, n * 4}, {top_p, n * 4}, {min_p, n * 4}};
  EXL3_CHECK_ARG(apart(all, 3), "exl3_sample: an output or the workspace overlaps another tensor of the call");
  int shift = 52;
  while ((1ll << (62 - shift)) < vocab) shift--;
  const int chunks = (vocab + kChunk - 1) / kChunk;
  SampleChunk* chunk = static_cast<SampleChunk*>(workspace);
  u64_t* bin_mass = reinterpret_cast<u64_t*>(chunk + n * chunks);
  int* bin_count = reinterpret_cast<int*>(bin_mass + n * chunks * kBins);
  SampleCut* cuts = reinterpret_cast<SampleCut*>(static_cast<char*>(workspace) + sample_chunk_bytes(rows, vocab));
  const SampleArgs a{logits, ld, rows, vocab, shift, uniform, temperature, top_p, min_p, top_k, all_temperature, all_top_p,
                     all_min_p, all_top_k, tokens, probs, chunks, chunk, bin_mass, bin_count, probs ? cuts : nullptr};
  hipStream_t st = as_stream(stream);
  const dim3 grid(chunks, rows);
#define EXL3_BY_TYPE(kern) (type == EXL3_F32 ? kern<EXL3_F32> : type == EXL3_BF16 ? kern<EXL3_BF16> : kern<EXL3_F16>)
  EXL3_BY_TYPE(sample_chunk_kernel)<<<grid, kChunkThreads, 0, st>>>(a);
  EXL3_CHECK_LAUNCH();
  EXL3_BY_TYPE(sample_row_kernel)<<<rows, kRowThreads, 0, st>>>(a);
  EXL3_CHECK_LAUNCH();
  if (probs) {
    EXL3_BY_TYPE(sample_probs_kernel)<<<grid, kChunkThreads, 0, st>>>(a);
    EXL3_CHECK_LAUNCH();
  }
#undef EXL3_BY_TYPE
  return EXL3_OK;
}
