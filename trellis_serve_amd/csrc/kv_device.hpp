// Building blocks of the kernels that work on the paged quantized KV cache (decode attention, draft-tree attention,
// cache writes and read-back): the layout's constants, the codes one lane takes from a page as MFMA operands, and
// reductions over a wave.
#pragma once
#include <stdint.h>

#include "exl3_device.hpp"

namespace exl3 {

typedef uint32_t kv_u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t kv_u32x4_t __attribute__((ext_vector_type(4)));

constexpr int kHeadDim = 128;
constexpr int kPage = 16;
constexpr int kMaxGroup = 16;

// 4 biased code bytes -> 4 fp16 (1024 + byte - sub); the fp16 subtract is exact for the code range
__device__ __forceinline__ half4_t codes_f16(uint32_t u, _Float16 sub) {
  const uint32_t lo = __builtin_amdgcn_perm(0x64646464u, u, 0x05010400u);  // bytes: u0, 0x64, u1, 0x64
  const uint32_t hi = __builtin_amdgcn_perm(0x64646464u, u, 0x05030402u);  // bytes: u2, 0x64, u3, 0x64
  return __builtin_bit_cast(half4_t, kv_u32x2_t{lo, hi}) - half4_t{sub, sub, sub, sub};
}

// 4 x 4 byte transpose: in[i] holds bytes 0..3 of row i; out[j] holds byte j of rows 0..3 (row order)
__device__ __forceinline__ void transpose4x4(const uint32_t in[4], uint32_t out[4]) {
  const uint32_t a = __builtin_amdgcn_perm(in[1], in[0], 0x05010400u);  // r0b0 r1b0 r0b1 r1b1
  const uint32_t b = __builtin_amdgcn_perm(in[3], in[2], 0x05010400u);  // r2b0 r3b0 r2b1 r3b1
  const uint32_t c = __builtin_amdgcn_perm(in[1], in[0], 0x07030602u);  // r0b2 r1b2 r0b3 r1b3
  const uint32_t d = __builtin_amdgcn_perm(in[3], in[2], 0x07030602u);  // r2b2 r3b2 r2b3 r3b3
  out[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
  out[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
  out[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
  out[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

// reductions over the 4 lanes l, l^16, l^32, l^48 (the 16 keys of a page for one query): v_permlane16_swap and
// v_permlane32_swap with both operands x return (x of row r, x of row r^1) and (x of half h, x of half h^1)
__device__ __forceinline__ float max_over_groups(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum_over_groups(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// magnitudes of halves order as integers: maxima of pairs, and over a wave
typedef uint16_t kv_u16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(kv_u16x2_t, a),
                                                                __builtin_bit_cast(kv_u16x2_t, b)));
}
template <int ROR>
__device__ __forceinline__ uint32_t max_ror(uint32_t v) {  // with the lane ROR places off in its row of 16
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + ROR, 0xF, 0xF, true));
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  v = max_ror<1>(max_ror<2>(max_ror<4>(max_ror<8>(v))));
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return __builtin_amdgcn_readfirstlane(max(b[0], b[1]));
}

// Keeps the loads above it issued here: otherwise they are free to sink to their first use, which turns the
// next-page prefetch into a load-and-wait.  Registers are not touched, so no wait is implied.  (The cache pointers
// carry no __restrict__: loads of restrict read-only memory count as invariant and would cross the fence.)
__device__ __forceinline__ void issue_fence() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);  // and no instruction that waits on older loads is scheduled above them
}

// The codes one lane needs from one (page, kv head) block, and the block's scales.
template <int BITS>
struct KvRegs {
  static constexpr int ROW = BITS == 8 ? kHeadDim : kHeadDim / 2;  // bytes per token row
  static constexpr int KW = BITS == 8 ? 8 : 4;                      // K dwords per lane
  static constexpr int VW = BITS == 8 ? 8 : 4;                      // V dwords per lane
  uint32_t k[KW], v[VW];
  uint32_t ksw, vsw;  // the block's two fp16 scales, each zero-extended in a register of its own

  // lane (n, g): K row n, bytes [ROW/4 * g, +ROW/4); V rows 4g .. 4g+3, bytes [ROW/16 * n, +ROW/16)
  __device__ __forceinline__ void load(const uint8_t* kblk, const uint8_t* vblk, const uint16_t* ksc,
                                       const uint16_t* vsc, size_t bi, int n, int g) {
    // The scales first, each zero-extended into a 32-bit register that nothing copies or packs before the scales are
    // used: packed as fp16 halves of one register (a copy that must wait for both loads), and issued as the page's
    // youngest loads, their wait covered every load in flight.
    ksw = ksc[bi];
    vsw = vsc[bi];
    const kv_u32x4_t* kp = reinterpret_cast<const kv_u32x4_t*>(kblk + n * ROW + (ROW / 4) * g);
    if constexpr (BITS == 8) {
      const kv_u32x4_t a = kp[0], b = kp[1];
      k[0] = a.x, k[1] = a.y, k[2] = a.z, k[3] = a.w, k[4] = b.x, k[5] = b.y, k[6] = b.z, k[7] = b.w;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const kv_u32x2_t t = *reinterpret_cast<const kv_u32x2_t*>(vblk + (4 * g + i) * ROW + 8 * n);
        v[i] = t.x, v[4 + i] = t.y;
      }
    } else {
      const kv_u32x4_t a = kp[0];
      k[0] = a.x, k[1] = a.y, k[2] = a.z, k[3] = a.w;
#pragma unroll
      for (int i = 0; i < 4; i++) v[i] = *reinterpret_cast<const uint32_t*>(vblk + (4 * g + i) * ROW + 4 * n);
    }
  }
  __device__ __forceinline__ _Float16 kscale() const { return __builtin_bit_cast(_Float16, (uint16_t)ksw); }
  __device__ __forceinline__ _Float16 vscale() const { return __builtin_bit_cast(_Float16, (uint16_t)vsw); }

  // K fragment c, biased: 1024 + bias + code (bias 128 / 8; removed after the MFMA, per page, from the query sums).
  // Dims of lane group g, in the order the Q fragment uses: 8 bits, dwords 2c, 2c+1 = dims 32g + 8c + 0..7;
  // 4 bits, dword c = dims 32g + 8c + 0..7 as nibbles 0..7, taken in pairs (s, s+4) straight into fp16 halves.
  __device__ __forceinline__ half8_t kfrag(int c) const {
    if constexpr (BITS == 8) {
      const uint32_t x = k[2 * c] ^ 0x80808080u, y = k[2 * c + 1] ^ 0x80808080u;
      return __builtin_bit_cast(half8_t, kv_u32x4_t{__builtin_amdgcn_perm(0x64646464u, x, 0x05010400u),
                                                     __builtin_amdgcn_perm(0x64646464u, x, 0x05030402u),
                                                     __builtin_amdgcn_perm(0x64646464u, y, 0x05010400u),
                                                     __builtin_amdgcn_perm(0x64646464u, y, 0x05030402u)});
    } else {
      const uint32_t x = k[c];
      return __builtin_bit_cast(half8_t, kv_u32x4_t{(x & 0x000F000Fu) ^ 0x64086408u, ((x >> 4) & 0x000F000Fu) ^ 0x64086408u,
                                                     ((x >> 8) & 0x000F000Fu) ^ 0x64086408u,
                                                     ((x >> 12) & 0x000F000Fu) ^ 0x64086408u});
    }
  }

  // V^T fragments: vt[db] = the 4 keys' biased codes at dim 8n + db
  __device__ __forceinline__ void vtrans(uint32_t vt[8]) const {
    if constexpr (BITS == 8) {
      uint32_t lo[4] = {v[0] ^ 0x80808080u, v[1] ^ 0x80808080u, v[2] ^ 0x80808080u, v[3] ^ 0x80808080u};
      uint32_t hi[4] = {v[4] ^ 0x80808080u, v[5] ^ 0x80808080u, v[6] ^ 0x80808080u, v[7] ^ 0x80808080u};
      transpose4x4(lo, vt);
      transpose4x4(hi, vt + 4);
    } else {
      uint32_t tb[4];
      transpose4x4(v, tb);  // tb[j]: byte j (dims 8n + 2j, 8n + 2j + 1) of the 4 keys
#pragma unroll
      for (int j = 0; j < 4; j++) {
        vt[2 * j] = (tb[j] & 0x0F0F0F0Fu) ^ 0x08080808u;
        vt[2 * j + 1] = ((tb[j] >> 4) & 0x0F0F0F0Fu) ^ 0x08080808u;
      }
    }
  }
};

__device__ __forceinline__ int wave_scan(int v) {  // inclusive prefix sum over the 64 lanes
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);   // row_shr:1, 2, 4, 8: inside each row of 16
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ int wave_total(int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }

}  // namespace exl3
