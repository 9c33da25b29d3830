// The step from one block of a model to the next in one pass (gfx950): the norm after a block, its gate and scale, the
// residual, and the norm before the next block.  For a token's row x (the block's output) and r (the residual stream):
//   u = x,  or  x * rsqrt(mean(x^2) + eps) * w_post
//   h = r + scale * act(g) * u                    act: g itself or its sigmoid; g one value a channel, a token or both
//   y = h * rsqrt(mean(h^2) + eps) * w
// with 1 + w for w where the weights are offsets.  fp32 throughout; h and y are each rounded once to their types, and y comes
// from the h before its rounding.
//
// A workgroup holds a row in registers between its sums.  Bound by memory at many rows, 8 bytes a value in 16 bits; by the
// chain load -> sum -> sum -> store at few.
#include <algorithm>

#include "exl3_api.hpp"
#include "exl3_device.hpp"

namespace exl3 {

typedef uint32_t an_u32x4_t __attribute__((ext_vector_type(4)));

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

template <int VEC>
__device__ __forceinline__ void an_load(const void* p, int type, long long at, float v[VEC]) {
  if constexpr (VEC == 1) {
    if (type == EXL3_F32) {
      v[0] = static_cast<const float*>(p)[at];
    } else {
      const uint16_t u = static_cast<const uint16_t*>(p)[at];
      v[0] = type == EXL3_BF16 ? __builtin_bit_cast(float, (uint32_t)u << 16) : (float)__builtin_bit_cast(_Float16, u);
    }
  } else {
    if (type == EXL3_F32) {
      const float4_t* q = reinterpret_cast<const float4_t*>(static_cast<const float*>(p) + at);
      const float4_t a = q[0], b = q[1];
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = a[e], v[4 + e] = b[e];
      return;
    }
    const an_u32x4_t r = *reinterpret_cast<const an_u32x4_t*>(static_cast<const uint16_t*>(p) + at);
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
}

template <int VEC>
__device__ __forceinline__ void an_store(void* p, int type, long long at, const float v[VEC]) {
  if constexpr (VEC == 1) {
    if (type == EXL3_F32)
      static_cast<float*>(p)[at] = v[0];
    else
      static_cast<uint16_t*>(p)[at] =
          type == EXL3_BF16 ? f32_to_bf16(v[0]) : __builtin_bit_cast(uint16_t, (_Float16)v[0]);
  } else {
    if (type == EXL3_F32) {
      float4_t* q = reinterpret_cast<float4_t*>(static_cast<float*>(p) + at);
      q[0] = float4_t{v[0], v[1], v[2], v[3]}, q[1] = float4_t{v[4], v[5], v[6], v[7]};
      return;
    }
    an_u32x4_t r;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (type == EXL3_BF16)
        r[i] = (uint32_t)f32_to_bf16(v[2 * i]) | ((uint32_t)f32_to_bf16(v[2 * i + 1]) << 16);
      else
        r[i] = __builtin_bit_cast(uint32_t, half2_t{(_Float16)v[2 * i], (_Float16)v[2 * i + 1]});
    }
    *reinterpret_cast<an_u32x4_t*>(static_cast<uint16_t*>(p) + at) = r;
  }
}

// the sum over the workgroup, in every lane; `part`: LDS, a float a wave, of its own for each call
__device__ __forceinline__ float an_sum(float v, float* part, int waves) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
  if (waves == 1) return v;
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
  for (int w = 0; w < waves; w++) s += part[w];
  return s;
}

// VEC values at a time, R times a thread
template <int VEC, int R>
__global__ __launch_bounds__(1024) void add_norm_kernel(const AddNormArgs a) {
  __shared__ float part[2][16];
  const long long row = blockIdx.x;
  const int waves = blockDim.x >> 6;
  const long long x0 = row * a.ld_x, r0 = row * a.ld_r, o0 = row * a.dim;
  float u[R][VEC];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < R; i++) {
    const int d = (threadIdx.x + i * blockDim.x) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; e++) u[i][e] = 0.f;
    if (d < a.dim) an_load<VEC>(a.x, a.x_type, x0 + d, u[i]);
#pragma unroll
    for (int e = 0; e < VEC; e++) ss = __builtin_fmaf(u[i][e], u[i][e], ss);
  }
  float post = 1.f;
  if (a.post_weight) post = 1.0f / __builtin_sqrtf(an_sum(ss, part[0], waves) / (float)a.dim + a.eps);
  float g_token = 1.f;
  if (a.gate_kind == kGateToken) an_load<1>(a.gate, a.g_type, row * a.ld_g, &g_token);
  auto act = [&](float g) { return a.sigmoid ? 1.0f / (1.0f + expf(-g)) : g; };
  const float token = a.scale * (a.gate_kind == kGateToken ? act(g_token) : 1.f);
  ss = 0.f;
#pragma unroll
  for (int i = 0; i < R; i++) {
    const int d = (threadIdx.x + i * blockDim.x) * VEC;
    if (d >= a.dim) continue;
    float w[VEC];
    if (a.post_weight) {
      an_load<VEC>(a.post_weight, a.w_type, d, w);
#pragma unroll
      for (int e = 0; e < VEC; e++) u[i][e] *= post * (w[e] + a.offset);
    }
    if (a.gate_kind == kGateChannel || a.gate_kind == kGateFull) {
      an_load<VEC>(a.gate, a.g_type, (a.gate_kind == kGateFull ? row * a.ld_g : 0) + d, w);
#pragma unroll
      for (int e = 0; e < VEC; e++) u[i][e] *= act(w[e]);
    }
    float r[VEC];
#pragma unroll
    for (int e = 0; e < VEC; e++) r[e] = 0.f;
    if (a.residual) an_load<VEC>(a.residual, a.r_type, r0 + d, r);
#pragma unroll
    for (int e = 0; e < VEC; e++) {
      u[i][e] = __builtin_fmaf(u[i][e], token, r[e]);
      ss = __builtin_fmaf(u[i][e], u[i][e], ss);
    }
    if (a.h) an_store<VEC>(a.h, a.r_type, o0 + d, u[i]);
  }
  if (!a.y) return;
  const float pre = 1.0f / __builtin_sqrtf(an_sum(ss, part[1], waves) / (float)a.dim + a.eps);
#pragma unroll
  for (int i = 0; i < R; i++) {
    const int d = (threadIdx.x + i * blockDim.x) * VEC;
    if (d >= a.dim) continue;
    float w[VEC];
    an_load<VEC>(a.weight, a.w_type, d, w);
#pragma unroll
    for (int e = 0; e < VEC; e++) w[e] = u[i][e] * pre * (w[e] + a.offset);
    an_store<VEC>(a.y, a.x_type, o0 + d, w);
  }
}

constexpr int kAddNormMaxDim = 65536;

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
  // 8 values at a time where every row of every tensor starts at a multiple of 16 bytes
  const bool vec = dim % 8 == 0 && ld_x % 8 == 0 && (!residual || ld_r % 8 == 0) && (gate_kind != kGateFull || ld_g % 8 == 0) &&
                   (((uintptr_t)x | (uintptr_t)residual | (uintptr_t)weight | (uintptr_t)post_weight | (uintptr_t)y |
                     (uintptr_t)h | (gate_kind == kGateToken ? 0 : (uintptr_t)gate)) & 15) == 0;
  const int chunks = vec ? dim / 8 : dim;
  const int threads = std::min(1024, (chunks + 63) / 64 * 64), each = (chunks + threads - 1) / threads;
  hipStream_t st = as_stream(stream);
  if (vec) {
    auto kern = each <= 1 ? add_norm_kernel<8, 1> : each <= 2 ? add_norm_kernel<8, 2> : each <= 4 ? add_norm_kernel<8, 4>
                                                                                            : add_norm_kernel<8, 8>;
    kern<<<rows, threads, 0, st>>>(a);
  } else {
    auto kern = each <= 4 ? add_norm_kernel<1, 4> : each <= 16 ? add_norm_kernel<1, 16> : add_norm_kernel<1, 64>;
    kern<<<rows, threads, 0, st>>>(a);
  }
  EXL3_CHECK_LAUNCH();
  return EXL3_OK;
}
