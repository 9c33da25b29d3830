// The step from one block of a model to the next in one pass (gfx950): the norm after a block, its gate and scale, the
// residual, and the norm before the next block.  For a token's row x (the block's output) and r (the residual stream):
//   u = x,  or  x * rsqrt(mean(x^2) + eps) * w_post
//   h = r + scale * act(g) * u                    act: g itself or its sigmoid; g one value a channel, a token or both
//   y = h * rsqrt(mean(h^2) + eps) * w
// with 1 + w for w where the weights are offsets.  fp32 throughout; h and y are each rounded once to their types, and y comes
// from the h before its rounding.
//
// A workgroup holds a row in registers between its sums.  Bound by memory at many rows, 8 bytes a value in 16 bits: 8192 rows of
// 5120 (336 MB, both norms, bf16) take 65 us, 5.1 TB/s, what a large copy reaches; by the chain load -> sum -> sum -> store at
// few (one row 3.4 us).
#include <algorithm>

#include "exl3_api.hpp"
#include "exl3_device.hpp"
#include "kv_device.hpp"

namespace exl3 {

typedef uint32_t an_u32x4_t __attribute__((ext_vector_type(4), aligned(2)));  // rows start at any value
typedef uint32_t an_b128_t __attribute__((ext_vector_type(4)));
typedef float an_f32x4_t __attribute__((ext_vector_type(4), aligned(4)));
typedef float an_f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 an_bf16x2_t __attribute__((ext_vector_type(2)));

enum { kGateNone = 0, kGateChannel = 1, kGateToken = 2, kGateFull = 3 };

struct AddNormArgs {
  const void *x, *residual, *weight, *post_weight, *gate;
  long long ld_x, ld_r, ld_g;
  int x_type, r_type, w_type, g_type;
  int gate_kind, sigmoid;
  float offset;  // 1 where the weights are offsets
  float scale, eps;
  int rows, dim;
  void *y, *h;
};

__device__ __forceinline__ void an_unpack(an_u32x4_t r, int type, float v[8]) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t u = r[i];
    if (type == EXL3_BF16) {
      v[2 * i] = __builtin_bit_cast(float, u << 16), v[2 * i + 1] = __builtin_bit_cast(float, u & 0xFFFF0000u);
    } else {
      const half2_t h = __builtin_bit_cast(half2_t, u);
      v[2 * i] = (float)h[0], v[2 * i + 1] = (float)h[1];
    }
  }
}

__device__ __forceinline__ float an_value(const void* p, int type, long long at) {
  if (type == EXL3_F32) return static_cast<const float*>(p)[at];
  const uint16_t u = static_cast<const uint16_t*>(p)[at];
  return type == EXL3_BF16 ? __builtin_bit_cast(float, (uint32_t)u << 16) : (float)__builtin_bit_cast(_Float16, u);
}

// values at .. at + 7 of a row, 0 past the first n (1 at least)
__device__ __forceinline__ void an_load(const void* p, int type, long long at, int n, float v[8]) {
  if (n < 8) {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = e < n ? an_value(p, type, at + e) : 0.f;
  } else if (type == EXL3_F32) {
    const an_f32x4_t* q = reinterpret_cast<const an_f32x4_t*>(static_cast<const float*>(p) + at);
    const an_f32x4_t a = q[0], b = q[1];
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = a[e], v[4 + e] = b[e];
  } else {
    an_unpack(*reinterpret_cast<const an_u32x4_t*>(static_cast<const uint16_t*>(p) + at), type, v);
  }
}

// two values in 16 bits, rounded to nearest even
template <int TYPE>
__device__ __forceinline__ uint32_t an_pair(float a, float b) {
  if constexpr (TYPE == EXL3_BF16)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((an_f32x2_t{a, b}), an_bf16x2_t));
  else
    return __builtin_bit_cast(uint32_t, half2_t{(_Float16)a, (_Float16)b});
}

template <int TYPE>
__device__ __forceinline__ void an_store(void* p, long long at, int n, const float v[8]) {
  if (n < 8) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      if (e >= n) continue;
      if constexpr (TYPE == EXL3_F32)
        static_cast<float*>(p)[at + e] = v[e];
      else
        static_cast<uint16_t*>(p)[at + e] = (uint16_t)an_pair<TYPE>(v[e], 0.f);
    }
  } else if constexpr (TYPE == EXL3_F32) {
    an_f32x4_t* q = reinterpret_cast<an_f32x4_t*>(static_cast<float*>(p) + at);
    q[0] = an_f32x4_t{v[0], v[1], v[2], v[3]}, q[1] = an_f32x4_t{v[4], v[5], v[6], v[7]};
  } else {
    an_u32x4_t r;
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = an_pair<TYPE>(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<an_u32x4_t*>(static_cast<uint16_t*>(p) + at) = r;
  }
}

__device__ __forceinline__ float an_act(const AddNormArgs& a, float g) { return a.sigmoid ? 1.0f / (1.0f + expf(-g)) : g; }

// the sum over the workgroup, in every lane; `slot` alternates, so that one barrier a sum is enough
struct AddNormSum {
  float (*part)[16];
  int waves, slot;
  __device__ __forceinline__ float operator()(float v) {
    v += lane_xor<1>(v);
    v += lane_xor<2>(v);
    v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x124, 0xF, 0xF, false));  // row_ror:4
    v += lane_xor<8>(v);
    v = sum_over_groups(v);
    if (waves == 1) return v;
    slot ^= 1;
    if ((threadIdx.x & 63) == 0) part[slot][threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
    for (int w = 0; w < waves; w++) s += part[slot][w];
    return s;
  }
};

// Rows of any width, stride and alignment: a workgroup a row, R times 8 values a thread
template <int R, int XT, int RT>
__global__ __launch_bounds__(512) void add_norm_any_kernel(const AddNormArgs a) {
  __shared__ float part[2][16];
  AddNormSum sum{part, (int)(blockDim.x >> 6), 0};
  const long long row = blockIdx.x, o0 = row * a.dim;
  float token = a.scale;
  if (a.gate_kind == kGateToken) token *= an_act(a, an_value(a.gate, a.g_type, row * a.ld_g));
  float u[R][8], ss = 0.f;
#pragma unroll
  for (int i = 0; i < R; i++) {
    const int d = (threadIdx.x + i * blockDim.x) * 8;
#pragma unroll
    for (int e = 0; e < 8; e++) u[i][e] = 0.f;
    if (d < a.dim) an_load(a.x, XT, row * a.ld_x + d, a.dim - d, u[i]);
#pragma unroll
    for (int e = 0; e < 8; e++) ss = __builtin_fmaf(u[i][e], u[i][e], ss);
  }
  float post = 1.f;
  if (a.post_weight) post = 1.0f / __builtin_sqrtf(sum(ss) / (float)a.dim + a.eps);
  ss = 0.f;
#pragma unroll
  for (int i = 0; i < R; i++) {
    const int d = (threadIdx.x + i * blockDim.x) * 8, n = a.dim - d;
    if (n <= 0) continue;
    float w[8], r[8];
    if (a.post_weight) {
      an_load(a.post_weight, a.w_type, d, n, w);
#pragma unroll
      for (int e = 0; e < 8; e++) u[i][e] *= post * (w[e] + a.offset);
    }
    if (a.gate_kind == kGateFull || a.gate_kind == kGateChannel) {
      an_load(a.gate, a.g_type, (a.gate_kind == kGateFull ? row * a.ld_g : 0) + d, n, w);
#pragma unroll
      for (int e = 0; e < 8; e++) u[i][e] *= an_act(a, w[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; e++) r[e] = 0.f;
    if (a.residual) an_load(a.residual, RT, row * a.ld_r + d, n, r);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      u[i][e] = e < n ? __builtin_fmaf(u[i][e], token, r[e]) : 0.f;
      ss = __builtin_fmaf(u[i][e], u[i][e], ss);
    }
    if (a.h) an_store<RT>(a.h, o0 + d, n, u[i]);
  }
  if (!a.y) return;
  const float pre = 1.0f / __builtin_sqrtf(sum(ss) / (float)a.dim + a.eps);
#pragma unroll
  for (int i = 0; i < R; i++) {
    const int d = (threadIdx.x + i * blockDim.x) * 8, n = a.dim - d;
    if (n <= 0) continue;
    float w[8];
    an_load(a.weight, a.w_type, d, n, w);
#pragma unroll
    for (int e = 0; e < 8; e++) w[e] = u[i][e] * pre * (w[e] + a.offset);
    an_store<XT>(a.y, o0 + d, n, w);
  }
}

// A row of n bytes as a buffer: what lies past it (all of it where p is null) reads as 0 and is not written
struct AddNormBuffer {
  __amdgpu_buffer_rsrc_t rsrc;
  __device__ __forceinline__ AddNormBuffer(const void* p, long long at, int n)
      : rsrc(__builtin_amdgcn_make_buffer_rsrc((void*)(static_cast<const char*>(p) + (p ? at : 0)), (short)0, p ? n : 0,
                                               0x00020000)) {}
  __device__ __forceinline__ an_u32x4_t load(int at) const {
    return __builtin_bit_cast(an_u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, 0, 0));
  }
  __device__ __forceinline__ void store(int at, an_u32x4_t v) const {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(an_b128_t, v), rsrc, at, 0, 0);
  }
};
template <int TYPE>
__device__ __forceinline__ void an_unpack_row(const an_u32x4_t* r, float v[8]) {
  if constexpr (TYPE == EXL3_F32) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const uint32_t u = r[e / 4][e & 3];
      v[e] = __builtin_bit_cast(float, u);
    }
  } else {
    an_unpack(r[0], TYPE, v);
  }
}
template <int TYPE>
__device__ __forceinline__ void an_put(const AddNormBuffer& to, int d, const float v[8]) {
  an_u32x4_t r[2];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (TYPE == EXL3_F32)
      r[0][i] = __builtin_bit_cast(uint32_t, v[i]), r[1][i] = __builtin_bit_cast(uint32_t, v[4 + i]);
    else
      r[0][i] = an_pair<TYPE>(v[2 * i], v[2 * i + 1]);
  }
  to.store(d * (TYPE == EXL3_F32 ? 4 : 2), r[0]);
  if constexpr (TYPE == EXL3_F32) to.store(d * 4 + 16, r[1]);
}

// Rows of multiples of 8 values that lie at multiples of 16 bytes, 8 values a thread.  A workgroup takes rows blockIdx.x,
// + gridDim.x, ..: the next row is loaded before this one is worked on; weights and a gate of one value a channel stay in
// registers.  Loads and stores go through buffers, without a branch: the wait for a row's loads then leaves the stores behind them
// out (with lane-conditional stores the compiler waits for everything: 112 us instead of 65 at 8192 rows of 5120).
template <int XT, int RT>
__global__ __launch_bounds__(1024) void add_norm_rows_kernel(const AddNormArgs a) {
  constexpr int WIDE = RT == EXL3_F32 ? 2 : 1;
  __shared__ float part[2][16];
  AddNormSum sum{part, (int)(blockDim.x >> 6), 0};
  const int x_bytes = a.dim * 2, r_bytes = a.dim * 2 * WIDE;
  const int d = threadIdx.x * 8, n = a.dim - d;
  float w[8], p[8];  // weight; post_weight times a channel's gate
#pragma unroll
  for (int e = 0; e < 8; e++) w[e] = 0.f, p[e] = 1.f;
  if (n > 0) {
    float g[8];
    if (a.post_weight) {
      an_load(a.post_weight, a.w_type, d, n, p);
#pragma unroll
      for (int e = 0; e < 8; e++) p[e] += a.offset;
    }
    if (a.gate_kind == kGateChannel) {
      an_load(a.gate, a.g_type, d, n, g);
#pragma unroll
      for (int e = 0; e < 8; e++) p[e] *= an_act(a, g[e]);
    }
    if (a.weight) an_load(a.weight, a.w_type, d, n, w);
#pragma unroll
    for (int e = 0; e < 8; e++) w[e] += a.offset;
  }
  const bool full = a.gate_kind == kGateFull;  // (in 16 bits)
  an_u32x4_t x, r[WIDE], f;
  auto load = [&](long long row) {
    const AddNormBuffer bx(a.x, row * a.ld_x * 2, x_bytes), br(a.residual, row * a.ld_r * 2 * WIDE, r_bytes),
        bf(full ? a.gate : nullptr, row * a.ld_g * 2, x_bytes);
    x = bx.load(2 * d);
#pragma unroll
    for (int j = 0; j < WIDE; j++) r[j] = br.load(2 * WIDE * d + 16 * j);
    f = bf.load(2 * d);
  };
  const float inv_dim = 1.0f / (float)a.dim;
  long long row = blockIdx.x;
  load(row);
  while (true) {
    float u[8], h[8], ss = 0.f;
    an_unpack(x, XT, u);
#pragma unroll
    for (int e = 0; e < 8; e++) ss = __builtin_fmaf(u[e], u[e], ss);
#pragma unroll
    for (int e = 0; e < 8; e++) u[e] *= p[e];
    if (full) {
      float q[8];
      an_unpack(f, a.g_type, q);
#pragma unroll
      for (int e = 0; e < 8; e++) u[e] *= an_act(a, q[e]);
    }
    an_unpack_row<RT>(r, h);
    const long long after = row + gridDim.x;
    load(min(after, (long long)a.rows - 1));
    float token = a.scale;
    if (a.gate_kind == kGateToken) token *= an_act(a, an_value(a.gate, a.g_type, row * a.ld_g));
    if (a.post_weight) token *= 1.0f / __builtin_sqrtf(sum(ss) * inv_dim + a.eps);
    ss = 0.f;
    const AddNormBuffer bh(a.h, row * r_bytes, r_bytes), by(a.y, row * x_bytes, x_bytes);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      h[e] = __builtin_fmaf(u[e], token, h[e]);
      ss = __builtin_fmaf(h[e], h[e], ss);
    }
    an_put<RT>(bh, d, h);
    const float pre = 1.0f / __builtin_sqrtf(sum(ss) * inv_dim + a.eps);
#pragma unroll
    for (int e = 0; e < 8; e++) h[e] *= pre * w[e];
    an_put<XT>(by, d, h);
    if (after >= a.rows) break;
    row = after;
  }
}

template <int XT, int RT>
static void add_norm_launch(const AddNormArgs& a, bool even, int threads, int each, int grid, hipStream_t st) {
  auto kern = even ? add_norm_rows_kernel<XT, RT>
              : each <= 1 ? add_norm_any_kernel<1, XT, RT>
              : each <= 4 ? add_norm_any_kernel<4, XT, RT>
                          : add_norm_any_kernel<8, XT, RT>;
  kern<<<grid, threads, 0, st>>>(a);
}

constexpr int kAddNormMaxDim = 32768;  // eight times 8 values of 512 threads

}  // namespace exl3

using namespace exl3;

extern "C" int exl3_add_norm(const void* x, int x_type, long long ld_x, const void* residual, int r_type, long long ld_r,
                             const void* weight, const void* post_weight, int w_type, int weight_offset, const void* gate,
                             int g_type, int gate_kind, long long ld_g, int gate_sigmoid, float scale, float eps, int rows,
                             int dim, void* y, void* h, void* stream) {
  EXL3_CHECK_ARG(rows >= 0 && dim >= 1 && dim <= kAddNormMaxDim, "exl3_add_norm: rows = %d, dim = %d (1 to %d)", rows, dim,
                 kAddNormMaxDim);
  EXL3_CHECK_ARG((x_type == EXL3_F16 || x_type == EXL3_BF16) && r_type >= EXL3_F16 && r_type <= EXL3_F32 &&
                     w_type >= EXL3_F16 && w_type <= EXL3_F32 && g_type >= EXL3_F16 && g_type <= EXL3_F32,
                 "exl3_add_norm: types %d (fp16, bf16), %d, %d, %d", x_type, r_type, w_type, g_type);
  EXL3_CHECK_ARG(gate_kind >= kGateNone && gate_kind <= kGateFull, "exl3_add_norm: gate kind %d", gate_kind);
  if (rows == 0) return EXL3_OK;
  EXL3_CHECK_ARG((gate_kind == kGateNone) == !gate, "exl3_add_norm: gate kind %d with%s a gate", gate_kind, gate ? "" : "out");
  EXL3_CHECK_ARG(!y == !weight && (y || h), "exl3_add_norm: a weight and its output y, or h alone");
  EXL3_CHECK_ARG(x, "exl3_add_norm: null pointer");
  EXL3_CHECK_ARG(ld_x >= dim && (!residual || ld_r >= dim) && (gate_kind != kGateFull || ld_g >= dim) &&
                     (gate_kind != kGateToken || ld_g >= 1),
                 "exl3_add_norm: row strides %lld / %lld / %lld of %d values", ld_x, ld_r, ld_g, dim);
  auto bytes = [](int type) { return type == EXL3_F32 ? (size_t)4 : (size_t)2; };
  auto aligned = [&](const void* p, int type) { return !p || (uintptr_t)p % bytes(type) == 0; };
  EXL3_CHECK_ARG(aligned(x, x_type) && aligned(residual, r_type) && aligned(weight, w_type) && aligned(post_weight, w_type) &&
                     aligned(gate, g_type) && aligned(y, x_type) && aligned(h, r_type),
                 "exl3_add_norm: a tensor is not aligned to its type");
  const size_t last = rows - 1, n = dim;
  const Span xs{x, (last * ld_x + n) * bytes(x_type)}, rs{residual, (last * ld_r + n) * bytes(r_type)};
  const size_t gate_values = gate_kind == kGateFull ? last * ld_g + n : gate_kind == kGateToken ? last * ld_g + 1 : n;
  const bool in_place = h && h == residual && ld_r == dim;
  const Span all[] = {{y, rows * n * bytes(x_type)}, {h, rows * n * bytes(r_type)}, xs,
                      in_place ? Span{nullptr, 0} : rs, {weight, n * bytes(w_type)}, {post_weight, n * bytes(w_type)},
                      {gate, gate_values * bytes(g_type)}};
  EXL3_CHECK_ARG(apart(all, 2), "exl3_add_norm: an output overlaps another tensor of the call");
  const AddNormArgs a{x, residual, weight, post_weight, gate, ld_x, ld_r, ld_g, x_type, r_type, w_type, g_type, gate_kind,
                      gate_sigmoid, weight_offset ? 1.f : 0.f, scale, eps, rows, dim, y, h};
  const int chunks = (dim + 7) / 8;
  const bool even = dim % 8 == 0 && chunks <= 1024 && ld_x % 8 == 0 && (!residual || ld_r % 8 == 0) &&
                    (gate_kind != kGateFull || (ld_g % 8 == 0 && g_type != EXL3_F32)) &&
                    (((uintptr_t)x | (uintptr_t)residual | (uintptr_t)y | (uintptr_t)h |
                      (gate_kind == kGateFull ? (uintptr_t)gate : 0)) & 15) == 0;
  const int threads = (std::min(chunks, even ? 1024 : 512) + 63) / 64 * 64;
  // Even rows: workgroups that stay for as many rows each, six waves a SIMD (16 values a thread, half the threads, took 73 us
  // at 8192 rows of 5120, for fewer waves by their registers; 8 take 65)
  const int fit = 256 * std::max(1, 1536 / threads), rounds = even ? (rows + fit - 1) / fit : 1;
  const int grid = (rows + rounds - 1) / rounds;
  const int each = (chunks + threads - 1) / threads;
  hipStream_t st = as_stream(stream);
  auto launch = x_type == EXL3_BF16 ? (r_type == EXL3_F32    ? add_norm_launch<EXL3_BF16, EXL3_F32>
                                       : r_type == EXL3_BF16 ? add_norm_launch<EXL3_BF16, EXL3_BF16>
                                                             : add_norm_launch<EXL3_BF16, EXL3_F16>)
                                    : (r_type == EXL3_F32    ? add_norm_launch<EXL3_F16, EXL3_F32>
                                       : r_type == EXL3_BF16 ? add_norm_launch<EXL3_F16, EXL3_BF16>
                                                             : add_norm_launch<EXL3_F16, EXL3_F16>);
  launch(a, even, threads, each, grid, st);
  EXL3_CHECK_LAUNCH();
  return EXL3_OK;
}
