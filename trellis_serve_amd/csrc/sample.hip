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
// threshold lies within some 10^-12 of the total (131072 elements) of an edge.
//
// sample_chunk_kernel: (chunks, rows) workgroups.  A chunk's largest logit m, its sum of exp((l - m) / t), and counts and sums
//   in 256 bins an eighth of an octave of w wide (less where the row is flat).  An element's bin is a monotone function of its
//   logit alone (and of the row's scale), so the chunks' bins match, and an element of a lower bin comes before every one of a
//   higher.  Elements that the chunk alone shows to be cut (behind its k-th; by up to an octave too few, so that finer bins hardly
//   leave any of these out: less than (1 - p) / vocab of its sum, below m of its largest) stay out of the bins.
// sample_border_kernel: a workgroup per row adds the bins up and so knows the bins that each rule's last element is in.
// sample_list_kernel: (chunks, rows) workgroups list those bins' elements (some hundreds a row) and sum what lies before them.
// sample_row_kernel: a workgroup per row finds the cut in the list, by histograms of ever smaller ranges; then the chunk, and in
//   it the element, where the running sum passes the threshold.  Rows of which the border bins hold more than the list takes (most
//   of the row equal; a top-k of half of 131072 with a top-p; normal logits of 262144 whose deviation is 0.3 to 1 of t, top-p 0.9;
//   a top-p with a top-k whose last element is some 2^-32 of the largest or less, past the bins, as a low t makes it) go through the
//   same search over the whole row, in one workgroup (131072 equal logits, top-p 0.9: 970 us; such a top-k of 40: 280 us).
// sample_probs_kernel: (chunks, rows) workgroups write the probabilities.
//
// Latency bounds it: each kernel waits for the whole of the one before, and a row's search is a chain of barriers.  In us, chunks,
// border, list, row, probabilities:  one row of 32003 fp32  5.5 + 3.9 + 5.1 + 8.2;  48 of 100352 fp16  14.4 + 5.5 + 7.7 + 13.5
// + 10.5;  64 of 131072 bf16  16.7 + 6.6 + 8.3 + 16.3.  (48 x 100352 half-precision logits read once are 1.9 us.)
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
constexpr int kChunkThreads = 512;
constexpr int kLargeChunk = 16 * kChunkThreads;
constexpr int kSmallChunk = 8 * kChunkThreads;
constexpr int kMaxChunks = kMaxVocab / kSmallChunk;
constexpr int kBins = 256;
constexpr int kBorderThreads = 256;               // a bin each, and a chunk each
constexpr int kRowThreads = 512;
constexpr int kRowWaves = kRowThreads / 64;
constexpr int kCrossBins = 1024;
constexpr int kList = 8192;                       // (two workgroups' fit a CU's LDS; sample_row_kernel reads 1024 ahead)
constexpr int kSliceRows = 512;                   // rows of a workspace
constexpr double kBinUnit = 0x1p-50;              // a bin's sum is in 2^-50 of the chunk's largest weight
constexpr double kBinBase = 0x1p52 * kBinUnit;
static_assert(kMaxChunks <= kBorderThreads && kBins == kBorderThreads);

struct SampleChunk {
  double sum;    // of exp((l - m) / t); with a top-k of at least those of the first k
  float m, top;  // the largest logit, its place on the bins' scale
  float bin_scale, unused;  // of the row
};

// What a row's kernels know of it
struct SampleBorder {
  double sum;                 // of all weights; with a top-k of at least the first k's
  double before_k, before_p;  // of those in the bins before k_bin, p_first
  double inv;                 // 1 / the sum of the kept weights (sample_row_kernel); 0: no logit above -inf
  double scale, min_w;        // of SampleRules: scale, m
  float m, top, bin_scale;    // the largest logit, its place; of SampleRules
  int first, last;            // the bins with elements that may be kept or not; before them all are, behind them none; first
                              // kBins: no rule
  int k_bin, k_left;          // the bin of the k-th element (-1: it does not matter), its rank there
  int p_first, p_last;        // the bins that top-p's last element may be in
  int listed;
  int cut_at;                 // the last kept element's index
  uint32_t cut;               // its key
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
  SampleBorder* border;  // [rows]
  SampleChunk* chunk;    // [rows][chunks]
  double* factor;        // [rows][chunks]: the weight of the chunk's largest logit
  u64_t* chunk_mass;     // [rows][chunks]: what lies before the border bins, in the row's units
  u64_t* bin_mass;       // [rows][chunks][kBins]
  int* bin_count;        // [rows][chunks][kBins], where there is a top-k
  u64_t* list;           // [rows][kList]: key << 32 | ~index
};

// A row's rules, and the scales of its weights (2^(scale (l - M))) and bins
struct SampleRules {
  double scale, p, m;
  float bin_scale;
  int k;
  bool by_k, by_p, by_m;
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
  r.by_k = r.k < a.vocab, r.by_p = r.p < 1.0, r.by_m = r.m > 0.0;
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
  // (in scalar registers: as literals the compiler moves each into the accumulator, two instructions a term)
  auto term = [](double c) {
    asm("" : "+s"(c));
    return c;
  };
  double p = term(Exp2Term<12>::value);
#define EXL3_TERM(i) p = __builtin_fma(p, r, term(Exp2Term<i>::value));
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

template <int TYPE>
struct SampleRow {
  using Raw = std::conditional_t<TYPE == EXL3_F32, uint32_t, uint16_t>;
  static constexpr int VEC = 16 / sizeof(Raw);  // elements of a 16-byte load
  static constexpr int LOW = TYPE == EXL3_F32 ? 0 : TYPE == EXL3_BF16 ? 16 : 13;  // bits that the type leaves 0 in a float
  const Raw* row;
  int vocab;

  __device__ __forceinline__ static float value(uint32_t bits) {
    float f;
    if constexpr (TYPE == EXL3_F32)
      f = __builtin_bit_cast(float, bits);
    else if constexpr (TYPE == EXL3_BF16)
      f = __builtin_bit_cast(float, bits << 16);
    else
      f = (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
    return fmaxf(f, -INFINITY);  // NaN: -inf
  }
  __device__ __forceinline__ float at(int i) const { return value(row[i]); }
  // elements i .. i + VEC - 1, -inf past the row; `whole` (uniform): none is
  __device__ __forceinline__ void get(int i, bool whole, float v[VEC]) const {
    if (whole || i + VEC <= vocab) {
      const sample_u32x4_t r = *reinterpret_cast<const sample_u32x4_t*>(row + i);
#pragma unroll
      for (int e = 0; e < VEC; e++)
        v[e] = value(TYPE == EXL3_F32 ? r[e % 4] : (r[e / 2 % 4] >> (16 * (e & 1))) & 0xFFFFu);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; e++) v[e] = i + e < vocab ? at(i + e) : -INFINITY;
    }
  }
  // a thread's EACH elements of a chunk: VEC j 's at first + j * step
  template <int EACH>
  __device__ __forceinline__ void get_each(int first, int step, bool whole, float v[EACH]) const {
    if (whole) {
#pragma unroll
      for (int j = 0; j < EACH / VEC; j++) get(first + j * step, true, v + j * VEC);
    } else {
#pragma unroll
      for (int j = 0; j < EACH / VEC; j++) get(first + j * step, false, v + j * VEC);
    }
  }
  // whole numbers that order like the logits, both zeros the same
  __device__ __forceinline__ static uint32_t key(float f) {
    const uint32_t u = __builtin_bit_cast(uint32_t, f + 0.f);
    return (u & 0x80000000u ? ~u : u | 0x80000000u) >> LOW;
  }
  __device__ __forceinline__ static float logit(uint32_t key) {
    const uint32_t u = key << LOW;
    return __builtin_bit_cast(float, u & 0x80000000u ? u & 0x7FFFFFFFu : ~u & (0xFFFFFFFFu << LOW));
  }
};

template <int TYPE>
__device__ __forceinline__ SampleRow<TYPE> sample_row(const SampleArgs& a, int row) {
  using Row = SampleRow<TYPE>;
  return Row{static_cast<const typename Row::Raw*>(a.logits) + (size_t)row * a.ld, a.vocab};
}

// ---- sums and maxima over a wave ---------------------------------------------------------------------------------------

template <int CTRL, int ROWS>
__device__ __forceinline__ u64_t dpp_u64(u64_t v) {  // 0 where no lane feeds
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, ROWS == 0xF);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xF, ROWS == 0xF);
  return (u64_t)hi << 32 | lo;
}
__device__ __forceinline__ u64_t wave_scan_u64(u64_t v) {  // inclusive
  v += dpp_u64<0x111, 0xF>(v);
  v += dpp_u64<0x112, 0xF>(v);
  v += dpp_u64<0x114, 0xF>(v);
  v += dpp_u64<0x118, 0xF>(v);
  v += dpp_u64<0x142, 0xA>(v);
  v += dpp_u64<0x143, 0xC>(v);
  return v;
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double v) {
  return v + __builtin_bit_cast(double, dpp_u64<CTRL, ROWS>(__builtin_bit_cast(u64_t, v)));
}
__device__ __forceinline__ double wave_scan_double(double v) {  // inclusive, in a fixed order
  v = dpp_add<0x111, 0xF>(v);
  v = dpp_add<0x112, 0xF>(v);
  v = dpp_add<0x114, 0xF>(v);
  v = dpp_add<0x118, 0xF>(v);
  v = dpp_add<0x142, 0xA>(v);
  return dpp_add<0x143, 0xC>(v);
}
__device__ __forceinline__ float wave_max_f32(float v) {  // of values that are no NaN
  v = fmaxf(v, lane_xor<1>(v));
  v = fmaxf(v, lane_xor<2>(v));
  v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x124, 0xF, 0xF, false)));
  v = fmaxf(v, lane_xor<8>(v));
  return max_over_groups(v);
}

// ---- the chunks --------------------------------------------------------------------------------------------------------

template <int TYPE, int EACH>
__global__ __launch_bounds__(kChunkThreads) void sample_chunk_kernel(const SampleArgs a) {
  constexpr int VEC = SampleRow<TYPE>::VEC, THREADS = kChunkThreads, WAVES = THREADS / 64, CHUNK = THREADS * EACH;
  __shared__ u64_t mass[kBins];
  __shared__ int count[kBins], firsts[kBins];
  __shared__ float part[WAVES], ends[2], coarse[WAVES];
  __shared__ double sums[WAVES];
  __shared__ int deepest;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = blockIdx.x, row = blockIdx.y;
  const SampleRow<TYPE> x = sample_row<TYPE>(a, row);
  const int first = c * CHUNK;
  const bool whole = first + CHUNK <= a.vocab;
  float l[EACH];
  x.template get_each<EACH>(first + tid * VEC, THREADS * VEC, whole, l);
  // Each chunk looks at the same 64 elements of the row: one that is flat there has finer bins (by a power of two, so that they still
  // reach over four times the range of these), or its border bins would hold more than the list takes (131072 logits whose
  // deviation is a tenth of t, top-p 0.9: 38 us for 463; the kernel takes 0.3 us more).  The 256 bins and the list know no vocabulary:
  // that serves 131072 of every deviation tried from 0.01 t on, 262144 of some, 2^20 of none up to 1.6 t (top-p 0.9: 3.3 ms)
  constexpr int SIDE = 16;  // elements side by side
  const bool probed = a.vocab > kList && wave == 0;
  const float probe = probed ? x.at(lane / SIDE * (a.vocab / (64 / SIDE)) + lane % SIDE) : 0.f;
  SampleRules rules = sample_rules(a, row);
  const bool bins = rules.by_k || rules.by_p || rules.by_m;
  // behind a chunk's k-th largest element, for k up to half its threads: bins of its threads' largest elements tell (others are more)
  const bool by_firsts = rules.by_k && rules.k <= THREADS / 2;
  static_assert(THREADS >= kBins);
  if (bins && tid < kBins) mass[tid] = 0, count[tid] = 0, firsts[tid] = 0;
  float mine = l[0];
#pragma unroll
  for (int i = 1; i < EACH; i++) mine = fmaxf(mine, l[i]);
  float m = wave_max_f32(mine);
  if (lane == 0) part[wave] = m;
  if (wave == 0) {
    const float high = wave_max_f32(probe), low = wave_max_f32(probe > -INFINITY ? -probe : -INFINITY);
    if (lane == 0) ends[0] = high, ends[1] = low;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; w++) m = fmaxf(m, part[w]);
  int finer = 0;
  const float range = (ends[0] + ends[1]) * (float)rules.scale;  // (0 where none were looked at)
  if (range > 0.f && range < 8.f) finer = min(max(5 - __builtin_amdgcn_frexp_expf(4.f * range), 0), 10);
  rules.bin_scale = __builtin_amdgcn_ldexpf(rules.bin_scale, finer);
  const size_t at = (size_t)row * a.chunks + c;
  const float top = sample_place(m, rules.bin_scale);
  const bool any = m > -INFINITY;
  // Elements of bins past `deep` take no part in any rule.  By weight that holds with bins to spare while places are exact to a
  // small part of one; exponents stand for logarithms, so `deep` is less than an octave, 8 << finer bins, more than needed (with
  // finer bins that and what is needed pass the 256 soon, and nothing is left out by weight), and for top-p a sum in 32 bits is
  // good enough.
  int deep = bins ? kBins - 2 : -1;
  const bool near = any && fabsf(top) < 0x1p16f;
  auto bins_to = [=](double w) { return (8 - 8 * __builtin_amdgcn_frexp_exp(w)) * (1 << finer) + 3; };
  if (near && rules.by_m && !(rules.by_k && rules.by_p)) deep = min(deep, bins_to(rules.m));
  const bool by_sum = near && rules.by_p && !rules.by_k;
  if (by_sum) {
    const float scale = (float)rules.scale;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < EACH; i++) s += __builtin_amdgcn_exp2f((l[i] - m) * scale);  // (0 for those past the row)
    s += lane_xor<1>(s);
    s += lane_xor<2>(s);
    s += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, s), 0x124, 0xF, 0xF, false));
    s += lane_xor<8>(s);
    s = sum_over_groups(s);
    if (lane == 0) coarse[wave] = s;
  }
  if (any && by_firsts) {
    const int bin = sample_bin(mine, rules.bin_scale, top);
    if (bin < kBins - 1) atomicAdd(&firsts[bin], 1);
  }
  if (by_sum || by_firsts) __syncthreads();
  if (by_sum) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < WAVES; i++) s += coarse[i];
    if (s > 0.5f) deep = min(deep, bins_to((1.0 - rules.p) * (double)s / (double)a.vocab));  // (NaN: -inf at a scale of 0)
  }
  if (any && by_firsts) {
    if (wave == 0) {
      int n[4], all = 0;
#pragma unroll
      for (int i = 0; i < 4; i++) n[i] = firsts[4 * lane + i], all += n[i];
      int run = wave_scan(all) - all, d = kBins;
#pragma unroll
      for (int i = 3; i >= 0; i--) {
        int upto = run;
#pragma unroll
        for (int j = 0; j <= i; j++) upto += n[j];
        if (upto >= rules.k) d = 4 * lane + i;
      }
      const unsigned long long hit = __builtin_amdgcn_ballot_w64(d < kBins);
      const int found = hit ? __builtin_amdgcn_readlane(d, __builtin_ctzll(hit)) : kBins;
      if (lane == 0) deepest = found;
    }
    __syncthreads();
    deep = min(deep, deepest);
  }
  double sum = 0.0;
  auto add = [&](float l, bool in, double w) {
    sum += in ? w : 0.0;
    const int bin = sample_bin(l, rules.bin_scale, top);
    if (in && bin <= deep) {
      atomicAdd(&mass[bin], sample_units(w, kBinBase));
      if (rules.by_k) atomicAdd(&count[bin], 1);
    }
  };
  if (any && by_firsts && deepest < kBins) {
    // the first k's weights are all that is asked for: the few that may be theirs, each lane's in turn
    unsigned take = 0;
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      const bool in = whole || first + (i / VEC * THREADS + tid) * VEC + i % VEC < a.vocab;
      take |= (unsigned)(in && sample_bin(l[i], rules.bin_scale, top) <= deep) << i;
    }
    while (take) {
      const int i = __builtin_ctz(take);
      take &= take - 1;
      const float one = x.at(first + (i / VEC * THREADS + tid) * VEC + i % VEC);
      add(one, true, sample_weight(one, m, rules.scale));
    }
  } else if (any && m < INFINITY && whole) {
    const double m64 = (double)m;
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      if (i % 4 == 0) __builtin_amdgcn_sched_barrier(0);  // a few chains at a time: all of them do not fit the registers
      add(l[i], true, exp2_f64(((double)l[i] - m64) * rules.scale));
    }
  } else if (any) {
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      if (i % 4 == 0) __builtin_amdgcn_sched_barrier(0);
      const bool in = whole || first + (i / VEC * THREADS + tid) * VEC + i % VEC < a.vocab;
      add(l[i], in, sample_weight(l[i], m, rules.scale));
    }
  }
  sum = wave_scan_double(sum);
  if (lane == 63) sums[wave] = sum;
  __syncthreads();
  if (tid == 0) {
    sum = 0.0;
    for (int w = 0; w < WAVES; w++) sum += sums[w];
    a.chunk[at] = SampleChunk{sum, m, top, rules.bin_scale, 0.f};
  }
  if (bins && tid < kBins) {
    a.bin_mass[at * kBins + tid] = mass[tid];
    if (rules.by_k) a.bin_count[at * kBins + tid] = count[tid];
  }
}

// ---- the border bins ---------------------------------------------------------------------------------------------------

__global__ __launch_bounds__(kBorderThreads) void sample_border_kernel(const SampleArgs a) {
  constexpr int WAVES = kBorderThreads / 64;
  __shared__ double factor[kMaxChunks], sums[WAVES], masses[WAVES], at_k[2], at_p;
  __shared__ float part[2][WAVES];
  __shared__ int shift[kMaxChunks], counts[WAVES], k_at[2], below[2][WAVES];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, C = a.chunks;
  SampleRules rules = sample_rules(a, row);
  rules.bin_scale = a.chunk[(size_t)row * C].bin_scale;
  SampleChunk chunk{0.0, -INFINITY, -INFINITY, 0.f, 0.f};
  if (tid < C) chunk = a.chunk[(size_t)row * C + tid];
  const float m = wave_max_f32(chunk.m), t = wave_max_f32(chunk.top);
  if (lane == 0) part[0][wave] = m, part[1][wave] = t;
  if (tid == 0) k_at[0] = kBins - 1;
  __syncthreads();
  float M = part[0][0], top = part[1][0];
#pragma unroll
  for (int w = 1; w < WAVES; w++) M = fmaxf(M, part[0][w]), top = fmaxf(top, part[1][w]);
  SampleBorder b{};
  b.m = M, b.top = top, b.scale = rules.scale, b.min_w = rules.m, b.bin_scale = rules.bin_scale;
  b.first = kBins, b.last = kBins - 1, b.k_bin = -1, b.p_last = -1, b.cut_at = a.vocab - 1;
  if (!(M > -INFINITY)) {  // nothing to draw from
    if (tid == 0) a.border[row] = b;
    return;
  }
  const double f = chunk.m > -INFINITY ? sample_weight(chunk.m, M, rules.scale) : 0.0;
  if (tid < C) a.factor[(size_t)row * C + tid] = f, factor[tid] = f * kBinUnit, shift[tid] = (int)fminf(top - chunk.top, (float)kBins);
  const double s = wave_scan_double(f * chunk.sum);
  if (lane == 63) sums[wave] = s;
  __syncthreads();
  b.sum = 0.0;
#pragma unroll
  for (int w = 0; w < WAVES; w++) b.sum += sums[w];
  if (rules.by_k || rules.by_p || rules.by_m) {
    // the bins of all chunks; the last one is what is not in the others
    double mass = 0.0;
    int count = 0;
    const u64_t* masses_of = a.bin_mass + (size_t)row * C * kBins;
    const int* counts_of = a.bin_count + (size_t)row * C * kBins;
    for (int c0 = 0; c0 < C; c0 += 8) {
      u64_t m8[8];
      int n8[8];
#pragma unroll
      for (int i = 0; i < 8; i++) {  // all loads first
        const int c = min(c0 + i, C - 1), at = c * kBins + max(tid - shift[c], 0);
        m8[i] = masses_of[at];
        n8[i] = rules.by_k ? counts_of[at] : 0;
      }
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const bool in = c0 + i < C && tid < kBins - 1 && tid >= shift[min(c0 + i, C - 1)];
        mass += in ? factor[min(c0 + i, C - 1)] * (double)m8[i] : 0.0;
        count += in ? n8[i] : 0;
      }
    }
    double mass_to = wave_scan_double(mass);
    int count_to = wave_scan(count);
    if (lane == 63) masses[wave] = mass_to, counts[wave] = count_to;
    __syncthreads();
    for (int w = 0; w < wave; w++) mass_to += masses[w], count_to += counts[w];
    const double mass_from = mass_to - mass;  // (a rounding apart from the bin before's mass_to)
    const int count_from = count_to - count;
    double bar_lo = b.sum, bar_hi = b.sum;
    if (rules.by_k) {
      if (tid < kBins - 1 && count_from < rules.k && count_to >= rules.k) k_at[0] = tid;
      __syncthreads();
      b.k_bin = k_at[0];
      if (tid == b.k_bin) k_at[1] = rules.k - count_from, at_k[0] = mass_from, at_k[1] = tid < kBins - 1 ? mass_to : b.sum;
      __syncthreads();
      b.k_left = k_at[1], b.before_k = bar_lo = at_k[0], bar_hi = fmax(at_k[1], bar_lo);
    }
    if (rules.by_p) {
      // a bin's sum is off by half a unit an element, the threshold by the part of the first k in their last bin
      const double slack = (double)a.vocab * kBinUnit + 1e-13 * b.sum;
      const double lo = rules.p * bar_lo - slack, hi = rules.p * bar_hi + slack;
      const int short_of = __builtin_popcountll(__builtin_amdgcn_ballot_w64(tid < kBins - 1 && mass_to < lo));
      const int from = __builtin_popcountll(__builtin_amdgcn_ballot_w64(mass_from < hi));
      if (lane == 0) below[0][wave] = short_of, below[1][wave] = from;
      __syncthreads();
      int p_last = -1;
#pragma unroll
      for (int w = 0; w < WAVES; w++) b.p_first += below[0][w], p_last += below[1][w];
      b.p_last = max(b.p_first, p_last);
      if (tid == b.p_first) at_p = mass_from;
      __syncthreads();
      b.before_p = at_p;
      b.first = min(b.first, b.p_first), b.last = min(b.last, b.p_last);
    }
    if (rules.by_m) {
      // w >= m from the logit M + log2(m) / scale on; places are off by a few 2^-24 of themselves
      const double y0 = (double)M * rules.bin_scale, y = y0 + log2(rules.m) * (rules.bin_scale / rules.scale);
      const double e = 0.01 + (fabs(y) + fabs(y0)) * 1e-6;
      const bool far = !(e < 64.0);  // (infinite M too)
      const double lo = (double)top - floor(y + e), hi = (double)top - floor(y - e);
      b.first = min(b.first, far ? 0 : (int)fmin(fmax(lo, 0.0), kBins - 1.0));
      b.last = min(b.last, far ? kBins - 1 : (int)fmin(fmax(hi, 0.0), kBins - 1.0));
    }
    if (rules.by_k) {
      if (!rules.by_p && b.k_bin > b.last)
        b.k_bin = -1;  // min-p stops before
      else
        b.first = min(b.first, b.k_bin), b.last = min(b.last, b.k_bin);
    }
    b.first = min(b.first, b.last);
  }
  if (tid == 0) a.border[row] = b;
}

// ---- their elements ----------------------------------------------------------------------------------------------------

template <int TYPE, int EACH>
__global__ __launch_bounds__(kChunkThreads) void sample_list_kernel(const SampleArgs a) {
  using Row = SampleRow<TYPE>;
  constexpr int VEC = Row::VEC, THREADS = kChunkThreads, WAVES = THREADS / 64, CHUNK = THREADS * EACH;
  __shared__ int part[WAVES], base;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = blockIdx.x, row = blockIdx.y;
  SampleBorder* border = a.border + row;
  const int g_first = border->first, g_last = border->last, k_bin = border->k_bin;
  if (g_first == kBins) return;  // no rule, or nothing to draw from
  const float top = border->top, bin_scale = border->bin_scale;
  const size_t at = (size_t)row * a.chunks + c;
  const float ahead = top - a.chunk[at].top;  // bins
  if (wave == 0) {  // its weights in the bins before the border
    const int end = g_first - (int)fminf(ahead, (float)kBins);
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < kBins / 64; i++) {
      const double m = (double)a.bin_mass[at * kBins + 64 * i + lane];
      s += 64 * i + lane < end ? m : 0.0;
    }
    s = wave_scan_double(s) * kBinUnit;
    if (lane == 63) a.chunk_mass[at] = (u64_t)__builtin_rint(s * a.factor[at] * (double)(1ull << a.shift));
  }
  if (ahead > (float)max(g_last, k_bin)) return;  // none listed
  const int first = c * CHUNK;
  const bool whole = first + CHUNK <= a.vocab;
  float l[EACH];
  sample_row<TYPE>(a, row).template get_each<EACH>(first + tid * VEC, THREADS * VEC, whole, l);
  unsigned take = 0;
#pragma unroll
  for (int i = 0; i < EACH; i++) {
    const int b = sample_bin(l[i], bin_scale, top);
    const bool in = whole || first + (i / VEC * THREADS + tid) * VEC + i % VEC < a.vocab;
    take |= (unsigned)(in && ((b >= g_first && b <= g_last) || b == k_bin)) << i;
  }
  const int mine = __builtin_popcount(take), upto = wave_scan(mine);
  if (lane == 63) part[wave] = upto;
  __syncthreads();
  int before = upto - mine, all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; w++) before += w < wave ? part[w] : 0, all += part[w];
  if (all == 0) return;
  if (tid == 0) base = atomicAdd(&border->listed, all);
  __syncthreads();
  int to = base + before;
  u64_t* list = a.list + (size_t)row * kList;
#pragma unroll
  for (int i = 0; i < EACH; i++)
    if (take >> i & 1) {
      if (to < kList) list[to] = (u64_t)Row::key(l[i]) << 32 | (uint32_t)~(first + (i / VEC * THREADS + tid) * VEC + i % VEC);
      to++;
    }
}

// ---- the cut and the token ---------------------------------------------------------------------------------------------

constexpr u64_t kNobody = ~(u64_t)0;  // (no key is that large)

struct SampleFound {
  u64_t before;
  int bin;
};
struct SampleShared {
  union {
    u64_t list[kList];
    int kept[kLargeChunk];
  };
  u64_t hist[kCrossBins], part[2][kRowWaves], chunk_mass[kMaxChunks];
  u64_t few[64], few_mass[64], result;
  SampleFound found[2];
  uint32_t ends[2][kRowWaves];
  int few_n;
};

template <int XOR>
__device__ __forceinline__ u64_t add_lane_xor(u64_t v) {
  const float lo = lane_xor<XOR>(__builtin_bit_cast(float, (uint32_t)v));
  const float hi = lane_xor<XOR>(__builtin_bit_cast(float, (uint32_t)(v >> 32)));
  return v + ((u64_t)__builtin_bit_cast(uint32_t, hi) << 32 | __builtin_bit_cast(uint32_t, lo));
}

// A workgroup's steps in LDS; `turn` alternates between two places, so that one barrier a step is enough
struct SampleGroup {
  SampleShared& sh;
  int turn = 0;

  // sum before this thread, and of all
  __device__ __forceinline__ u64_t scan(u64_t v, u64_t& total) {
    const int wave = threadIdx.x >> 6;
    const u64_t s = wave_scan_u64(v);
    turn ^= 1;
    if ((threadIdx.x & 63) == 63) sh.part[turn][wave] = s;
    __syncthreads();
    u64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kRowWaves; w++) {
      const u64_t one = sh.part[turn][w];
      before += w < wave ? one : 0;
      total += one;
    }
    return before + s - v;
  }

  // Elements that each(f) calls f(key, index, mass()) for (a thread has its own; n of all threads at most), keys in [lo, hi],
  // indices below vocab, in order of falling keys and rising indices: the one (key << 32 | ~index) at which their running mass
  // reaches `target` (at least 1, at most their sum).  An element's place in that order is one number, (hi - key, index);
  // histograms narrow its range to 1/1024 a pass, the last 64 are ranked.  (Few keys leave bits of the first histogram to the
  // indices, so that equal logits do not all add to one place of it.)
  template <class Each>
  __device__ __forceinline__ u64_t cross(int n, uint32_t lo, uint32_t hi, int vocab, u64_t target, Each each) {
    const int low = vocab > 1 ? 32 - __builtin_clz(vocab - 1) : 0;
    int bits = low + (hi > lo ? 32 - __builtin_clz(hi - lo) : 0);
    u64_t from = 0;
    auto offset = [&](uint32_t key, int index) { return ((u64_t)(hi - key) << low | (uint32_t)index) - from; };
    bool narrow = n > 64;
    while (true) {
      __syncthreads();
      if (threadIdx.x == 0) sh.few_n = 0, sh.result = kNobody;
      if (narrow) {
        const int shift = max(0, bits - 10);
        for (int i = threadIdx.x; i < kCrossBins; i += kRowThreads) sh.hist[i] = 0;
        turn ^= 1;
        SampleFound& found = sh.found[turn];
        if (threadIdx.x == 0) found = SampleFound{0, 0};
        __syncthreads();
        each([&](uint32_t key, int index, auto mass) {
          const u64_t v = offset(key, index);
          if (v >> bits == 0) atomicAdd(&sh.hist[v >> shift], mass());
        });
        __syncthreads();
        constexpr int PER = kCrossBins / kRowThreads;
        u64_t bin[PER], all = 0, total;
#pragma unroll
        for (int i = 0; i < PER; i++) bin[i] = sh.hist[threadIdx.x * PER + i], all += bin[i];
        turn ^= 1;  // (scan turns again: it does not touch what `found` refers to)
        u64_t before = scan(all, total);
#pragma unroll
        for (int i = 0; i < PER; i++) {
          if (before < target && before + bin[i] >= target) found = SampleFound{before, (int)threadIdx.x * PER + i};
          before += bin[i];
        }
        __syncthreads();
        target -= found.before;
        from += (u64_t)found.bin << shift;
        bits = shift;
      } else {
        __syncthreads();
      }
      each([&](uint32_t key, int index, auto mass) {
        const u64_t v = offset(key, index);
        if (v >> bits == 0) {
          const int at = atomicAdd(&sh.few_n, 1);
          if (at < 64) sh.few[at] = v, sh.few_mass[at] = mass();
        }
      });
      __syncthreads();
      const int few = sh.few_n;
      if (few <= 64) {
        // 8 lanes an element, each sums what an eighth of the others puts before it
        constexpr int LANES = kRowThreads / 64;
        const int e = threadIdx.x / LANES, part = threadIdx.x % LANES;
        const u64_t mine = sh.few[e], m = sh.few_mass[e];
        u64_t before = 0;
#pragma unroll
        for (int j = 0; j < 64; j += LANES) {
          const u64_t other = sh.few[j + part], mass = sh.few_mass[j + part];
          before += j + part < few && other < mine ? mass : 0;
        }
        before = add_lane_xor<1>(before), before = add_lane_xor<2>(before), before = add_lane_xor<4>(before);
        if (e < few && part == 0 && before < target && before + m >= target) {
          const u64_t v = mine + from;
          sh.result = (u64_t)(hi - (uint32_t)(v >> low)) << 32 | ~((uint32_t)v & ((1u << low) - 1));
        }
        __syncthreads();
        return sh.result;
      }
      narrow = true;
    }
  }
};

template <int TYPE, int CHUNK>
__global__ __launch_bounds__(kRowThreads) void sample_row_kernel(const SampleArgs a) {
  using Row = SampleRow<TYPE>;
  constexpr int VEC = Row::VEC, EACH = CHUNK / kRowThreads;
  __shared__ SampleShared sh;
  SampleGroup group{sh};
  const int row = blockIdx.x, tid = threadIdx.x, V = a.vocab, C = a.chunks;
  SampleBorder* border = a.border + row;
  const u64_t* list = a.list + (size_t)row * kList;
  // (before their number is known: what the list does not hold is not looked at)
  constexpr int AHEAD = 2;
  u64_t ahead[AHEAD];
#pragma unroll
  for (int j = 0; j < AHEAD; j++) ahead[j] = list[tid + j * kRowThreads];
  const SampleBorder b = *border;
  if (!(b.m > -INFINITY)) {
    if (tid == 0 && a.tokens) a.tokens[row] = -1;
    return;
  }
  const Row x = sample_row<TYPE>(a, row);
  const SampleRules rules = sample_rules(a, row);
  const double one = (double)(1ull << a.shift), base = (double)(1ull << (52 - a.shift));
  auto weight = [&](float l) { return sample_weight(l, b.m, b.scale); };
  auto mass = [&](float l) { return sample_units(weight(l), base); };
  auto bin_of = [&](uint32_t key) { return sample_bin(Row::logit(key), b.bin_scale, b.top); };
  const bool ruled = b.first < kBins, fast = b.listed <= kList;
  const int n = fast ? b.listed : V;
  uint32_t lo = ~0u, hi = 0;  // of the list's keys
  if (fast) {
    auto take = [&](int i, u64_t v) {
      const uint32_t key = (uint32_t)(v >> 32);
      sh.list[i] = v;
      lo = min(lo, key), hi = max(hi, key);
    };
#pragma unroll
    for (int j = 0; j < AHEAD; j++)
      if (tid + j * kRowThreads < n) take(tid + j * kRowThreads, ahead[j]);
    for (int i = tid + AHEAD * kRowThreads; i < n; i += kRowThreads) take(i, list[i]);
  }
  lo = wave_max_u32(~lo), hi = wave_max_u32(hi);
  if ((tid & 63) == 0) sh.ends[0][tid >> 6] = lo, sh.ends[1][tid >> 6] = hi;
  for (int c = tid; c < C; c += kRowThreads) {
    const size_t at = (size_t)row * C + c;
    sh.chunk_mass[c] = ruled && !fast ? 0
                       : ruled        ? a.chunk_mass[at]
                                      : (u64_t)__builtin_rint(a.factor[at] * a.chunk[at].sum * one);
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kRowWaves; w++) lo = max(lo, sh.ends[0][w]), hi = max(hi, sh.ends[1][w]);
  lo = fast ? ~lo : 0, hi = fast ? hi : Row::key(b.m);
  // f(key, index, mass()) of the list's elements, or of the row's
  auto each = [&](auto f) {
    if (fast) {
      for (int i = tid; i < n; i += kRowThreads) {
        const u64_t v = sh.list[i];
        f((uint32_t)(v >> 32), (int)~(uint32_t)v, [&] { return mass(Row::logit((uint32_t)(v >> 32))); });
      }
    } else {
      for (int i = tid * VEC; i < V; i += kRowThreads * VEC) {
        float l[VEC];
        x.get(i, false, l);
#pragma unroll
        for (int e = 0; e < VEC; e++)
          if (i + e < V) f(Row::key(l[e]), i + e, [&] { return mass(l[e]); });
      }
    }
  };

  // the last kept element
  uint32_t cut = 0;
  int cut_at = V - 1;
  auto before_cut = [&](uint32_t key, int i) { return key > cut || (key == cut && i <= cut_at); };
  if (rules.by_k && (!fast || b.k_bin >= 0)) {
    const u64_t at = group.cross(n, lo, hi, V, fast ? b.k_left : rules.k, [&](auto f) {
      each([&](uint32_t key, int index, auto) {
        if (!fast || bin_of(key) == b.k_bin) f(key, index, [] { return (u64_t)1; });
      });
    });
    if (at != kNobody) cut = (uint32_t)(at >> 32), cut_at = (int)~(uint32_t)at;
  }
  if (rules.by_p) {
    auto in_p = [&](uint32_t key, int index) {
      if (!before_cut(key, index)) return false;
      const int g = fast ? bin_of(key) : b.p_first;
      return g >= b.p_first && g <= b.p_last;
    };
    // the sums of the bins that its last element may be in, and of what top-k keeps of its last one
    u64_t most = 0, at_k = 0, before;
    each([&](uint32_t key, int index, auto mass_of) {
      if (!before_cut(key, index)) return;
      const u64_t m = mass_of();
      most += in_p(key, index) ? m : 0;
      at_k += fast && bin_of(key) == b.k_bin ? m : 0;
    });
    group.scan(most, before), most = before;
    double total = fast ? b.sum : (double)most / one;
    if (fast && rules.by_k) {
      group.scan(at_k, before);
      total = b.before_k + (double)before / one;
    }
    const double bar = __builtin_ceil((rules.p * total - (fast ? b.before_p : 0.0)) * one);
    if (most > 0) {
      const u64_t target = bar >= 1.0 ? min((u64_t)bar, most) : 1;
      const u64_t at = group.cross(n, lo, hi, V, target, [&](auto f) {
        each([&](uint32_t key, int index, auto mass_of) {
          if (in_p(key, index)) f(key, index, mass_of);
        });
      });
      if (at != kNobody) cut = (uint32_t)(at >> 32), cut_at = (int)~(uint32_t)at;
    }
  }

  // the kept sum of every chunk, and the token
  if (ruled)
    each([&](uint32_t key, int index, auto mass_of) {
      if ((fast && bin_of(key) > b.last) || !before_cut(key, index)) return;
      if (rules.by_m && !(weight(Row::logit(key)) >= rules.m)) return;
      atomicAdd(&sh.chunk_mass[index / CHUNK], mass_of());
    });
  __syncthreads();
  const u64_t here = tid < C ? sh.chunk_mass[tid] : 0;
  u64_t total;
  const u64_t before = group.scan(here, total);
  if (tid == 0) border->cut = cut, border->cut_at = cut_at, border->inv = one / (double)total;
  if (!a.tokens) return;
  const float u = a.uniform[row];
  const double bar = (u > 0.f ? (double)u : 0.0) * (double)total;  // the smallest whole number above it
  const u64_t target = bar < (double)total ? min((u64_t)bar + 1, total) : total;
  if (here > 0 && before < target && before + here >= target) sh.found[0] = SampleFound{before, tid};
  __syncthreads();
  u64_t left = target - sh.found[0].before;
  const int c = sh.found[0].bin;
  // the chunk's kept elements, by index
  const int i0 = c * CHUNK + tid * EACH;
  float l[EACH];
  x.template get_each<EACH>(i0, VEC, (c + 1) * CHUNK <= V, l);
  unsigned flags = 0;
#pragma unroll
  for (int j = 0; j < EACH; j++)
    flags |= (unsigned)(i0 + j < V && before_cut(Row::key(l[j]), i0 + j) && sample_bin(l[j], b.bin_scale, b.top) <= b.last) << j;
  u64_t kept;
  int to = (int)group.scan(__builtin_popcount(flags), kept);
#pragma unroll
  for (int j = 0; j < EACH; j++)
    if (flags >> j & 1) sh.kept[to++] = i0 + j;
  __syncthreads();
  const int per = ((int)kept + kRowThreads - 1) / kRowThreads, first = tid * per;
  u64_t w[EACH], sum = 0, all;
#pragma unroll
  for (int j = 0; j < EACH; j++) {
    w[j] = 0;
    if (j >= per) continue;  // (uniform)
    if (first + j < (int)kept) {
      const float l = x.at(sh.kept[first + j]);
      const double v = weight(l);
      w[j] = v >= b.min_w ? sample_units(v, base) : 0;
    }
    sum += w[j];
  }
  u64_t run = group.scan(sum, all);
  left = min(left, all);  // (the chunk's sum from its bins may be a rounding apart)
  if (all == 0 && tid == 0) a.tokens[row] = kept > 0 ? sh.kept[0] : -1;
  if (run < left && run + sum >= left) {
    int at = 0;
#pragma unroll
    for (int j = 0; j < EACH; j++) {
      if (w[j] > 0 && run < left) at = first + j;
      run += w[j];
    }
    a.tokens[row] = sh.kept[at];
  }
}

template <int TYPE, int EACH>
__global__ __launch_bounds__(kChunkThreads) void sample_probs_kernel(const SampleArgs a) {
  using Row = SampleRow<TYPE>;
  constexpr int VEC = Row::VEC, THREADS = kChunkThreads;
  typedef float f4_t __attribute__((ext_vector_type(4), aligned(4)));
  const int row = blockIdx.y, first = blockIdx.x * (THREADS * EACH);
  const bool whole = first + THREADS * EACH <= a.vocab;
  const Row x = sample_row<TYPE>(a, row);
  float l[EACH];
  x.template get_each<EACH>(first + (int)threadIdx.x * VEC, THREADS * VEC, whole, l);
  const SampleBorder* border = a.border + row;
  const double inv = border->inv, scale = border->scale, min_w = border->min_w;
  const float m = border->m;
  const uint32_t cut = border->cut;
  const int cut_at = border->cut_at;
  float* out = a.probs + (size_t)row * a.vocab;
  auto index = [&](int i) { return first + (i / VEC * THREADS + (int)threadIdx.x) * VEC + i % VEC; };
  unsigned kept = 0;
#pragma unroll
  for (int i = 0; i < EACH; i++) {
    const uint32_t key = Row::key(l[i]);
    kept |= (unsigned)((whole || index(i) < a.vocab) && (key > cut || (key == cut && index(i) <= cut_at))) << i;
  }
  if (!(inv > 0.0)) kept = 0;
  // zeros everywhere, then the few kept ones, each lane's in turn: a wave computes as many as its fullest lane has
#pragma unroll
  for (int j = 0; j < EACH / VEC; j++) {
    const int at = index(j * VEC);
    if (whole || at + VEC <= a.vocab) {
#pragma unroll
      for (int e = 0; e < VEC; e += 4) *reinterpret_cast<f4_t*>(out + at + e) = f4_t{0.f, 0.f, 0.f, 0.f};
    } else {
#pragma unroll
      for (int e = 0; e < VEC; e++)
        if (at + e < a.vocab) out[at + e] = 0.f;
    }
  }
  while (kept) {
    const int at = index(__builtin_ctz(kept));
    kept &= kept - 1;
    const double w = sample_weight(x.at(at), m, scale);
    if (w >= min_w) out[at] = (float)(w * inv);
  }
}

// Chunks of 8192 elements, or 4096 for more workgroups where there are few elements in all (one row of 32003 fp32: the chunks'
// kernel takes 7.0 us with 4 chunks, 5.0 with 8)
constexpr int kFewElements = 1 << 19;
static int sample_chunk(int rows, int vocab) { return (long long)rows * vocab <= kFewElements ? kSmallChunk : kLargeChunk; }
static size_t sample_bytes(int rows, int chunks) {
  return rows * (sizeof(SampleBorder) + kList * sizeof(u64_t) +
                 chunks * (sizeof(SampleChunk) + sizeof(double) + sizeof(u64_t) + kBins * (sizeof(u64_t) + sizeof(int))));
}

template <int TYPE, int EACH>
static hipError_t sample_launch(const SampleArgs& a, bool ruled, hipStream_t st) {
  const dim3 grid(a.chunks, a.rows);
  sample_chunk_kernel<TYPE, EACH><<<grid, kChunkThreads, 0, st>>>(a);
  sample_border_kernel<<<a.rows, kBorderThreads, 0, st>>>(a);
  if (ruled) sample_list_kernel<TYPE, EACH><<<grid, kChunkThreads, 0, st>>>(a);
  sample_row_kernel<TYPE, kChunkThreads * EACH><<<a.rows, kRowThreads, 0, st>>>(a);
  if (a.probs) sample_probs_kernel<TYPE, EACH><<<grid, kChunkThreads, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace exl3

using namespace exl3;

extern "C" size_t exl3_sample_workspace_bytes(int rows, int vocab) {
  if (rows <= 0 || vocab <= 0 || vocab > kMaxVocab) return 0;
  // the most that up to `rows` rows need, of which a slice is there at a time: fewer may take smaller chunks
  const int slice = std::min(rows, kSliceRows), chunk = sample_chunk(rows, vocab);
  const int few = std::min(slice, kFewElements / vocab);
  return std::max(sample_bytes(slice, (vocab + chunk - 1) / chunk), sample_bytes(few, (vocab + kSmallChunk - 1) / kSmallChunk));
}

extern "C" int exl3_sample(const void* logits, int type, long long ld, int rows, int vocab, const float* uniform,
                           const float* temperature, double all_temperature, const int* top_k, int all_top_k,
                           const float* top_p, double all_top_p, const float* min_p, double all_min_p, int* tokens, float* probs,
                           void* workspace, size_t workspace_bytes, void* stream) {
  EXL3_CHECK_ARG(rows >= 0 && rows < (1 << 26) && vocab >= 1 && vocab <= kMaxVocab,
                 "exl3_sample: rows = %d, vocab = %d (1 to %d)", rows, vocab, kMaxVocab);
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
  const int chunk = sample_chunk(rows, vocab), chunks = (vocab + chunk - 1) / chunk;
  const bool ruled = temperature || top_k || top_p || min_p || !(all_temperature > 0.0) || (all_top_k > 0 && all_top_k < vocab) ||
                     all_top_p < 1.0 || all_min_p > 0.0;
  for (int first = 0; first < rows; first += kSliceRows) {
    const int slice = std::min(rows - first, kSliceRows);
    auto from = [&](auto* p, long long step) { return p ? p + first * step : p; };
    SampleArgs a{static_cast<const char*>(logits) + (size_t)first * ld * bytes, ld, slice, vocab, shift, from(uniform, 1),
                 from(temperature, 1), from(top_p, 1), from(min_p, 1), from(top_k, 1), all_temperature, all_top_p, all_min_p,
                 all_top_k, from(tokens, 1), from(probs, vocab), chunks};
    a.border = static_cast<SampleBorder*>(workspace);
    a.list = reinterpret_cast<u64_t*>(a.border + slice);
    a.bin_mass = a.list + (size_t)slice * kList;
    a.chunk_mass = a.bin_mass + (size_t)slice * chunks * kBins;
    a.factor = reinterpret_cast<double*>(a.chunk_mass + (size_t)slice * chunks);
    a.chunk = reinterpret_cast<SampleChunk*>(a.factor + (size_t)slice * chunks);
    a.bin_count = reinterpret_cast<int*>(a.chunk + (size_t)slice * chunks);
    const bool large = chunk == kLargeChunk;
    hipStream_t st = as_stream(stream);
    EXL3_CHECK_HIP(type == EXL3_F32    ? (large ? sample_launch<EXL3_F32, 16>(a, ruled, st) : sample_launch<EXL3_F32, 8>(a, ruled, st))
                   : type == EXL3_BF16 ? (large ? sample_launch<EXL3_BF16, 16>(a, ruled, st) : sample_launch<EXL3_BF16, 8>(a, ruled, st))
                                       : (large ? sample_launch<EXL3_F16, 16>(a, ruled, st) : sample_launch<EXL3_F16, 8>(a, ruled, st)));
  }
  return EXL3_OK;
}
