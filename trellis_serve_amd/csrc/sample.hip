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
// Weights are 64-bit; they are summed as integers, rint(w 2^s) with s = 62 - ceil(log2 vocab), so no sum depends on an order
// (LDS atomics included).  A weight is off by 2^-(s+1) of the largest one at most: another summation decides differently only
// within some 10^-11 of the total of an edge.
#include <math.h>

#include <algorithm>

#include "exl3_api.hpp"
#include "exl3_device.hpp"
#include "kv_device.hpp"

namespace exl3 {

struct SampleArgs {
  const void* logits;
  int type;
  long long ld;
  int rows, vocab, shift;  // shift: s above
  const float *uniform, *temperature, *top_p, *min_p;  // NULL: the value for every row
  const int* top_k;
  double all_temperature, all_top_p, all_min_p;
  int all_top_k;
  int* tokens;
  float* probs;
};

typedef unsigned long long u64_t;

// exp(z) for z <= 0: 2^k exp(r), |r| <= ln(2) / 2, by its series (the first term left out is below 10^-17); 0 below -700
__device__ __forceinline__ double exp_f64(double z) {
  const double k = __builtin_rint(z * 1.4426950408889634074);
  double r = __builtin_fma(k, -0.693147180369123816490, z);  // ln 2 in two parts, the first of 33 bits
  r = __builtin_fma(k, -1.90821492927058770002e-10, r);
  double p = 1.0 / 6227020800.0;
  constexpr double kInv[] = {1.0 / 479001600.0, 1.0 / 39916800.0, 1.0 / 3628800.0, 1.0 / 362880.0, 1.0 / 40320.0, 1.0 / 5040.0,
                             1.0 / 720.0,       1.0 / 120.0,      1.0 / 24.0,      1.0 / 6.0,      0.5,           1.0,
                             1.0};
#pragma unroll
  for (int i = 0; i < 13; i++) p = __builtin_fma(p, r, kInv[i]);
  const u64_t u = __builtin_bit_cast(u64_t, p) + ((u64_t)(long long)k << 52);
  return z > -700.0 ? __builtin_bit_cast(double, u) : 0.0;
}

__device__ __forceinline__ uint32_t sample_key(float f) {  // orders like the logits, both zeros the same
  const uint32_t u = __builtin_bit_cast(uint32_t, f + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float sample_logit(uint32_t key) {
  return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}
constexpr uint32_t kKeyOfMinusInf = 0x007FFFFFu;

__device__ __forceinline__ float sample_load(const SampleArgs& a, const void* row, int i) {
  float f;
  if (a.type == EXL3_F32) {
    f = static_cast<const float*>(row)[i];
  } else {
    const uint16_t u = static_cast<const uint16_t*>(row)[i];
    f = a.type == EXL3_BF16 ? __builtin_bit_cast(float, (uint32_t)u << 16) : (float)__builtin_bit_cast(_Float16, u);
  }
  return f == f ? f : -INFINITY;
}

constexpr int kSampleThreads = 1024;
constexpr int kSampleBins = 1024;

struct SampleShared {
  u64_t hist[kSampleBins], part[16];
  uint32_t key[16];
  u64_t before;
  int bin;
};

__device__ __forceinline__ u64_t shfl_up_u64(u64_t v, int d) {
  const uint32_t lo = __shfl_up((int)(uint32_t)v, d), hi = __shfl_up((int)(uint32_t)(v >> 32), d);
  return (u64_t)hi << 32 | lo;
}

// sum before this thread, and of all
__device__ __forceinline__ u64_t sample_scan(u64_t v, u64_t& total, SampleShared& sh) {
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
  for (int w = 0; w < 16; w++) {
    before += w < wave ? sh.part[w] : 0;
    total += sh.part[w];
  }
  return before + s - v;
}

__device__ __forceinline__ uint32_t sample_max(uint32_t v, SampleShared& sh) {
  v = wave_max_u32(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.key[threadIdx.x >> 6] = v;
  __syncthreads();
  for (int w = 0; w < 16; w++) v = max(v, sh.key[w]);
  return v;
}

// Of the elements i < n with a value get(i, value, mass) in [lo, hi]: the value at which their masses, summed from hi down, reach
// `target` (at least 1, at most their sum); target becomes what is left of it for that value
template <class Get>
__device__ uint32_t sample_cross(int n, uint32_t lo, uint32_t hi, u64_t& target, SampleShared& sh, Get get) {
  while (lo < hi) {
    const uint32_t span = hi - lo;
    const int shift = max(0, 32 - __builtin_clz(span) - 10);
    __syncthreads();
    for (int i = threadIdx.x; i < kSampleBins; i += kSampleThreads) sh.hist[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kSampleThreads) {
      uint32_t v;
      u64_t m;
      if (get(i, lo, hi, v, m)) atomicAdd(&sh.hist[(hi - v) >> shift], m);
    }
    __syncthreads();
    u64_t total;
    const u64_t here = sh.hist[threadIdx.x], before = sample_scan(here, total, sh);
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

__global__ __launch_bounds__(kSampleThreads) void sample_row_kernel(const SampleArgs a) {
  __shared__ SampleShared sh;
  const int row = blockIdx.x, tid = threadIdx.x, V = a.vocab;
  const void* logits = static_cast<const char*>(a.logits) + (size_t)row * a.ld * (a.type == EXL3_F32 ? 4 : 2);
  const double t = a.temperature ? (double)a.temperature[row] : a.all_temperature;
  const double top_p = a.top_p ? (double)a.top_p[row] : a.all_top_p, min_p = a.min_p ? (double)a.min_p[row] : a.all_min_p;
  int k = a.top_k ? a.top_k[row] : a.all_top_k;
  const bool greedy = !(t > 0.0);
  if (greedy) k = 1;
  if (k <= 0 || k > V) k = V;
  const double inv_t = greedy ? 1.0 : 1.0 / t;

  uint32_t most = 0;
  for (int i = tid; i < V; i += kSampleThreads) most = max(most, sample_key(sample_load(a, logits, i)));
  most = sample_max(most, sh);
  float* probs = a.probs ? a.probs + (size_t)row * V : nullptr;
  if (most <= kKeyOfMinusInf) {  // nothing to draw from
    if (tid == 0 && a.tokens) a.tokens[row] = -1;
    if (probs)
      for (int i = tid; i < V; i += kSampleThreads) probs[i] = 0.f;
    return;
  }
  const float M = sample_logit(most);
  const double one = (double)(1ull << a.shift);
  auto weight = [&](float l) { return l == M ? 1.0 : exp_f64(((double)l - (double)M) * inv_t); };
  auto mass = [&](float l) { return (u64_t)__builtin_rint(weight(l) * one); };

  uint32_t cut = 0;  // the last kept element: its key, its index
  int cut_at = V - 1;
  auto kept = [&](uint32_t key, int i) { return key > cut || (key == cut && i <= cut_at); };
  // the first `count` elements of key `at`, by index
  auto cut_ties = [&](uint32_t at, u64_t count) {
    const uint32_t last = ~0u - (uint32_t)(V - 1);
    const uint32_t v = sample_cross(V, last, ~0u, count, sh, [&](int i, uint32_t lo, uint32_t hi, uint32_t& v, u64_t& m) {
      v = ~(uint32_t)i, m = 1;
      return v >= lo && v <= hi && sample_key(sample_load(a, logits, i)) == at;
    });
    cut = at, cut_at = (int)~v;
  };
  auto total_kept = [&]() {
    u64_t sum = 0, total;
    for (int i = tid; i < V; i += kSampleThreads) {
      const float l = sample_load(a, logits, i);
      if (kept(sample_key(l), i)) sum += mass(l);
    }
    sample_scan(sum, total, sh);
    return total;
  };
  if (k < V) {
    u64_t target = k;
    const uint32_t at = sample_cross(V, 0, most, target, sh, [&](int i, uint32_t lo, uint32_t hi, uint32_t& v, u64_t& m) {
      v = sample_key(sample_load(a, logits, i)), m = 1;
      return v >= lo && v <= hi;
    });
    cut_ties(at, target);
  }
  if (top_p < 1.0) {
    const u64_t sum = total_kept();
    const double bar = __builtin_ceil((top_p > 0.0 ? top_p : 0.0) * (double)sum);
    u64_t target = max((u64_t)1, min((u64_t)bar, sum));
    const uint32_t at = sample_cross(V, cut, most, target, sh, [&](int i, uint32_t lo, uint32_t hi, uint32_t& v, u64_t& m) {
      const float l = sample_load(a, logits, i);
      v = sample_key(l);
      if (v < lo || v > hi || !kept(v, i)) return false;
      m = mass(l);
      return true;
    });
    const u64_t each = mass(sample_logit(at));
    cut_ties(at, (target + each - 1) / each);
  }
  if (min_p > 0.0) {
    const double m = fmin(min_p, 1.0);
    uint32_t least = 0;
    for (int i = tid; i < V; i += kSampleThreads) {
      const float l = sample_load(a, logits, i);
      if (weight(l) >= m) least = max(least, ~sample_key(l));
    }
    least = ~sample_max(least, sh);
    if (least > cut) cut = least, cut_at = V - 1;
  }
  const u64_t sum = total_kept();
  if (a.tokens) {
    const float u = a.uniform[row];
    const double bar = (u > 0.f ? (double)u : 0.0) * (double)sum;
    u64_t target = bar < (double)sum ? min((u64_t)bar + 1, sum) : sum;
    const uint32_t last = ~0u - (uint32_t)(V - 1);
    const uint32_t v = sample_cross(V, last, ~0u, target, sh, [&](int i, uint32_t lo, uint32_t hi, uint32_t& v, u64_t& m) {
      v = ~(uint32_t)i;
      if (v < lo || v > hi) return false;
      const float l = sample_load(a, logits, i);
      if (!kept(sample_key(l), i)) return false;
      m = mass(l);
      return true;
    });
    if (tid == 0) a.tokens[row] = (int)~v;
  }
  if (probs) {
    const double scale = one / (double)sum;
    for (int i = tid; i < V; i += kSampleThreads) {
      const float l = sample_load(a, logits, i);
      probs[i] = kept(sample_key(l), i) ? (float)(weight(l) * scale) : 0.f;
    }
  }
}

constexpr int kMaxVocab = 1 << 24;

}  // namespace exl3

using namespace exl3;

extern "C" size_t exl3_sample_workspace_bytes(int rows, int vocab) { return 0; }

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
  const size_t n = rows;
  const Span all[] = {{tokens, n * 4}, {probs, n * vocab * 4}, {logits, ((n - 1) * ld + vocab) * bytes}, {uniform, n * 4},
                      {temperature, n * 4}, {top_k, n * 4}, {top_p, n * 4}, {min_p, n * 4}};
  EXL3_CHECK_ARG(apart(all, 2), "exl3_sample: an output overlaps another tensor of the call");
  int shift = 62;
  while ((1ll << (62 - shift)) < vocab) shift--;
  shift = std::min(shift, 52);
  const SampleArgs a{logits, type, ld, rows, vocab, shift, uniform, temperature, top_p, min_p, top_k, all_temperature,
                     all_top_p, all_min_p, all_top_k, tokens, probs};
  sample_row_kernel<<<rows, kSampleThreads, 0, as_stream(stream)>>>(a);
  EXL3_CHECK_LAUNCH();
  return EXL3_OK;
}
