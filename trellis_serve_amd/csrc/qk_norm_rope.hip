// Norms of every query and key head with the position rotation, in one pass (gfx950).
//
// For a head's 128 values x of a token at position t:
//   y = x * rsqrt(mean(x^2) + eps) * w                      (w: the queries' or the keys' weight, fp32 throughout)
//   z_a = y_a cos - y_b sin,  z_b = y_b cos + y_a sin       for the pairs (a, b) of the first `rotary` values:
//                                                           (i, i + rotary/2), or (2i, 2i + 1) when interleaved
// with cos, sin = row t of the table, rounded once to the output type.
//
// 16 lanes hold one head (8 values, 16 bytes each), so a wave works on 4 heads at a time; the sum of squares is four
// DPP row rotations.  A wave stays with one token: the weights and the token's cos / sin are loaded once, in registers, for
// up to `per` groups of 4 heads.  The partner of a half-split pair sits rotary/16 lanes away (a row rotate by 8 for
// rotary = 128, else a ds_bpermute); interleaved pairs are in the lane.  Bound by memory at many tokens, 4 bytes a value: 8192
// tokens of 40 + 8 heads (206 MB) take 40.8 us, 5.0 TB/s, what a large copy reaches; by the launch at few (1 token 3.1 us,
// 77 of 32 + 2 heads 3.6).
#include <algorithm>

#include "exl3_api.hpp"
#include "exl3_device.hpp"

namespace exl3 {

typedef uint32_t nr_u32x4_t __attribute__((ext_vector_type(4)));

constexpr int kNormDim = 128;

struct NormRopeArgs {
  const uint16_t *q, *k;
  long long ld_q, ld_k;  // elements from one token's heads to the next's
  const void *q_weight, *k_weight;
  int w_type;
  float eps;
  const float* cos_sin;
  int max_pos, rotary, interleaved;
  const void* positions;
  int pos_i64;
  uint16_t *q_out, *k_out;
  int tokens, Hq, Hkv;
  int groups, per, slices;  // groups of 4 heads per token, per wave; waves per token
};

template <bool BF16>
__device__ __forceinline__ void unpack8(nr_u32x4_t r, float v[8]) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (BF16) {
      v[2 * i] = __builtin_bit_cast(float, r[i] << 16);
      v[2 * i + 1] = __builtin_bit_cast(float, r[i] & 0xFFFF0000u);
    } else {
      const uint32_t u = r[i];  // a value of its own: the bit cast of a vector's element takes element 0
      const half2_t h = __builtin_bit_cast(half2_t, u);
      v[2 * i] = (float)h[0], v[2 * i + 1] = (float)h[1];
    }
  }
}

template <bool BF16>
__device__ __forceinline__ nr_u32x4_t pack8(const float v[8]) {
  nr_u32x4_t r;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (BF16)
      r[i] = (uint32_t)f32_to_bf16(v[2 * i]) | ((uint32_t)f32_to_bf16(v[2 * i + 1]) << 16);
    else
      r[i] = __builtin_bit_cast(uint32_t, half2_t{(_Float16)v[2 * i], (_Float16)v[2 * i + 1]});
  }
  return r;
}

__device__ __forceinline__ void load_weight(const void* w, int type, int d0, float v[8]) {
  if (type == EXL3_F32) {
    const float4_t* p = reinterpret_cast<const float4_t*>(static_cast<const float*>(w) + d0);
    const float4_t a = p[0], b = p[1];
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = a[e], v[4 + e] = b[e];
    return;
  }
  const nr_u32x4_t r = *reinterpret_cast<const nr_u32x4_t*>(static_cast<const uint16_t*>(w) + d0);
  if (type == EXL3_BF16)
    unpack8<true>(r, v);
  else
    unpack8<false>(r, v);
}

// sum over the 16 lanes of a row, in every lane
__device__ __forceinline__ float row_sum(float v) {
  v += lane_xor<8>(v);
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x124, 0xF, 0xF, false));
  v += lane_xor<2>(v);
  return v + lane_xor<1>(v);
}

template <bool XB, bool OB>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(const NormRopeArgs a) {
  const int lane = threadIdx.x & 63, sub = lane >> 4, j = lane & 15, d0 = 8 * j;
  const unsigned wave = blockIdx.x * 4u + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned t = wave / (unsigned)a.slices;
  if (t >= (unsigned)a.tokens) return;
  const int g0 = (int)(wave - t * (unsigned)a.slices) * a.per, g1 = min(g0 + a.per, a.groups);
  const int H = a.Hq + a.Hkv;

  float wq[8], wk[8], c[8], s[8];  // s: the sine as it multiplies the partner (negative for the pair's first value)
#pragma unroll
  for (int e = 0; e < 8; e++) wq[e] = wk[e] = c[e] = 1.f, s[e] = 0.f;
  if (a.q_weight) {
    load_weight(a.q_weight, a.w_type, d0, wq);
    load_weight(a.k_weight, a.w_type, d0, wk);
  }
  const int half = a.rotary / 16;  // lanes from a value to its partner, half-split pairs
  int partner = lane;
  if (a.cos_sin && d0 < a.rotary) {
    const long long at = a.pos_i64 ? static_cast<const long long*>(a.positions)[t]
                                   : (long long)static_cast<const int*>(a.positions)[t];
    const int pos = (int)(at < 0 ? 0 : at >= a.max_pos ? a.max_pos - 1 : at);
    const float* row = a.cos_sin + (size_t)pos * a.rotary;
    const int r2 = a.rotary / 2;
    if (a.interleaved) {
      const float4_t cv = *reinterpret_cast<const float4_t*>(row + 4 * j);
      const float4_t sv = *reinterpret_cast<const float4_t*>(row + r2 + 4 * j);
#pragma unroll
      for (int e = 0; e < 8; e++) c[e] = cv[e / 2], s[e] = (e & 1) ? sv[e / 2] : -sv[e / 2];
    } else {
      const bool first = j < half;
      const float* p = row + 8 * (first ? j : j - half);
      partner = first ? lane + half : lane - half;
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const float4_t cv = *reinterpret_cast<const float4_t*>(p + 4 * i);
        const float4_t sv = *reinterpret_cast<const float4_t*>(p + r2 + 4 * i);
#pragma unroll
        for (int e = 0; e < 4; e++) c[4 * i + e] = cv[e], s[4 * i + e] = first ? -sv[e] : sv[e];
      }
    }
  }

  for (int g = g0; g < g1; g++) {
    const int h = 4 * g + sub;
    const bool is_q = h < a.Hq;
    if (h >= H) break;  // the lanes of a row leave together; every cross-lane step stays in its row
    const uint16_t* src = is_q ? a.q + t * a.ld_q + h * kNormDim : a.k + t * a.ld_k + (h - a.Hq) * kNormDim;
    float v[8];
    unpack8<XB>(*reinterpret_cast<const nr_u32x4_t*>(src + d0), v);
    if (a.q_weight) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; e++) ss = __builtin_fmaf(v[e], v[e], ss);
      const float r = 1.0f / __builtin_sqrtf(__builtin_fmaf(row_sum(ss), 1.0f / kNormDim, a.eps));
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] *= r * (is_q ? wq[e] : wk[e]);
    }
    if (a.cos_sin) {
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float p = a.interleaved ? v[e ^ 1] : a.rotary == kNormDim ? lane_xor<8>(v[e]) : __shfl(v[e], partner);
        o[e] = __builtin_fmaf(v[e], c[e], s[e] * p);
      }
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = d0 < a.rotary ? o[e] : v[e];
    }
    uint16_t* dst = is_q ? a.q_out + ((size_t)t * a.Hq + h) * kNormDim
                         : a.k_out + ((size_t)t * a.Hkv + (h - a.Hq)) * kNormDim;
    *reinterpret_cast<nr_u32x4_t*>(dst + d0) = pack8<OB>(v);
  }
}

}  // namespace exl3

using namespace exl3;

extern "C" int exl3_qk_norm_rope(const void* q, const void* k, int x_bf16, long long ld_q, long long ld_k, int tokens,
                                 int num_q_heads, int num_kv_heads, int head_dim, const void* q_weight,
                                 const void* k_weight, int w_type, float eps, const float* cos_sin, int max_pos,
                                 int rotary_dim, int interleaved, const void* positions, int positions_i64,
                                 void* q_out, void* k_out, int out_bf16, void* stream) {
  EXL3_CHECK_ARG(head_dim == kNormDim, "exl3_qk_norm_rope: head_dim = %d (supported: 128)", head_dim);
  EXL3_CHECK_ARG(tokens >= 0 && num_q_heads >= 1 && num_kv_heads >= 1 && num_q_heads <= 65536 && num_kv_heads <= 65536,
                 "exl3_qk_norm_rope: tokens = %d, heads %d / %d", tokens, num_q_heads, num_kv_heads);
  EXL3_CHECK_ARG(!q_weight == !k_weight, "exl3_qk_norm_rope: both weights or neither");
  EXL3_CHECK_ARG(!q_weight || (w_type >= EXL3_F16 && w_type <= EXL3_F32), "exl3_qk_norm_rope: weight type %d", w_type);
  EXL3_CHECK_ARG(q_weight || cos_sin, "exl3_qk_norm_rope: neither weights nor a rotation table");
  EXL3_CHECK_ARG(!cos_sin || (max_pos >= 1 && rotary_dim >= 16 && rotary_dim <= head_dim && rotary_dim % 16 == 0),
                 "exl3_qk_norm_rope: rotary_dim = %d (a multiple of 16 up to 128), max_pos = %d", rotary_dim, max_pos);
  if (tokens == 0) return EXL3_OK;
  EXL3_CHECK_ARG(q && k && q_out && k_out && (!cos_sin || positions), "exl3_qk_norm_rope: null pointer");
  EXL3_CHECK_ARG(ld_q >= (long long)num_q_heads * head_dim && ld_k >= (long long)num_kv_heads * head_dim &&
                     ld_q % 8 == 0 && ld_k % 8 == 0,
                 "exl3_qk_norm_rope: token strides %lld / %lld (multiples of 8, a token's heads at least)", ld_q, ld_k);
  EXL3_CHECK_ARG((((uintptr_t)q | (uintptr_t)k | (uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)q_weight |
                   (uintptr_t)k_weight | (uintptr_t)cos_sin) & 15) == 0,
                 "exl3_qk_norm_rope: a tensor is not 16-byte aligned");
  const int groups = (num_q_heads + num_kv_heads + 3) / 4;
  // groups per wave: one while that fills the card (8192 waves), then enough to load weights and angles once a token
  const int per = (int)std::min<long long>(groups, std::max<long long>(1, (long long)tokens * groups / 8192));
  const int slices = (groups + per - 1) / per;
  EXL3_CHECK_ARG((long long)tokens * slices < (1LL << 26), "exl3_qk_norm_rope: %d tokens of %d heads", tokens,
                 num_q_heads + num_kv_heads);
  const NormRopeArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), ld_q, ld_k, q_weight, k_weight,
                       w_type, eps, cos_sin, max_pos, cos_sin ? rotary_dim : 0, interleaved, positions, positions_i64,
                       static_cast<uint16_t*>(q_out), static_cast<uint16_t*>(k_out), tokens, num_q_heads, num_kv_heads,
                       groups, per, slices};
  const unsigned blocks = ((unsigned)tokens * (unsigned)slices + 3u) / 4u;
  auto kern = x_bf16 ? (out_bf16 ? qk_norm_rope_kernel<true, true> : qk_norm_rope_kernel<true, false>)
                     : (out_bf16 ? qk_norm_rope_kernel<false, true> : qk_norm_rope_kernel<false, false>);
  kern<<<blocks, 256, 0, as_stream(stream)>>>(a);
  EXL3_CHECK_LAUNCH();
  return EXL3_OK;
}
