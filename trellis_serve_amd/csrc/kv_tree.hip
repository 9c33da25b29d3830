// Attention of drafted tokens, a tree or a chain per sequence, over the paged quantized KV cache (gfx950).
//
//   o[i] = softmax(sm_scale q_i [K_cache ; K_nodes]^T) [V_cache ; V_nodes]
// for nodes i < 64 of every sequence: all of them see the cached tokens, and those nodes whose bits their mask sets.  The
// nodes' keys and values come in fp16 (they enter the cache, quantized, once verified).  Cache layout and the MFMA forms of a
// page: kv_attention.hip; a query row here is a (node, query head) pair of one kv head.
//
// A wave keeps RG groups of 16 rows and works on two pages (32 keys) a step:
//   S^T = K Q^T     4 x MFMA 16x16x32 per page and group; the K fragments are decoded once for all groups
//   O^T += V^T P^T  8 x MFMA 16x16x32 per group: slots 0..3 of a lane's 8 keys are its keys of the first page, 4..7 of the
//                   second, so the C layout of the two S^T is the B operand as it stands
// Softmax in base 2 with a lazy reference: O, l are rescaled only when a logit passes the reference by more than 4.  The
// page's value scale is folded into the exponent (p' = 2^(s + log2 vs - m)), so P' stays within 16 of fp16 whatever the
// scales are, and a step has no multiplication per probability; the sum takes p' / vs, once per page and row.
//
// Work split: a unit is (sequence, kv head, tile of rows), its steps 4 x 2 pages each (four waves take two pages each) and a
// last one for the nodes.  The steps of all units in a row are dealt to the workgroups in equal runs, whatever the lengths:
// a unit inside one run is written directly, the parts of a split one go to the workspace and kv_tree_merge_kernel joins
// them in order (deterministic).  Tiles of more than 64 rows take 8 waves (RS = 2 halves of the rows on the same pages).
#include <algorithm>

#include "exl3_api.hpp"
#include "kv_device.hpp"

namespace exl3 {

constexpr int kTreeNodes = 64;        // a bit of the mask each
constexpr int kTreePageWaves = 4;     // waves that take two pages each per step
constexpr int kTreeStep = 2 * kTreePageWaves;
constexpr float kTreeLow = -1e30f;    // below any logit, finite: differences of empty states are 0, not NaN

struct KvTreeArgs {
  const _Float16 *q, *k_new, *v_new;
  long long ld_q, ld_k, ld_v;
  const unsigned long long* mask;
  const int* num_nodes;
  const uint8_t *kc, *vc;
  const uint16_t *ksc, *vsc;
  int num_pages;
  const int* page_table;
  int max_pages;
  const int* seq_lens;
  int batch, nodes, Hq, Hkv, G;
  float qk_scale;  // sm_scale * log2(e)
  int wgs;
  float *part_o, *part_ml;
  _Float16* out;
};

// A place in the row of all steps
struct TreeUnit {
  int b, len, nodes, pages, steps;  // the sequence; steps of one of its units
  int first;                        // the sequence's first step
};

// Steps of sequence base + lane (0 past the batch), and what they come from
__device__ __forceinline__ int tree_steps(const KvTreeArgs& a, int tile, int b, int& len, int& nodes) {
  const int at = min(b, a.batch - 1);
  len = max(min(a.seq_lens[at], a.max_pages * kPage), 0);
  nodes = a.num_nodes ? max(min(a.num_nodes[at], a.nodes), 0) : a.nodes;
  nodes = b < a.batch ? nodes : 0;
  const int pages = (len + kPage - 1) / kPage;
  return a.Hkv * ((nodes * a.G + tile - 1) / tile) * ((pages + kTreeStep - 1) / kTreeStep + 1);
}

__device__ __forceinline__ int tree_total(const KvTreeArgs& a, int tile) {
  const int lane = threadIdx.x & 63;
  int total = 0;
  for (int base = 0; base < a.batch; base += 64) {
    int len, nodes;
    total += wave_total(tree_steps(a, tile, base + lane, len, nodes));
  }
  return total;
}

__device__ __forceinline__ TreeUnit tree_unit(int b, int len, int nodes, int first) {
  const int pages = (len + kPage - 1) / kPage;
  return TreeUnit{b, len, nodes, pages, (pages + kTreeStep - 1) / kTreeStep + 1, first};
}

// The sequence that step s (below the total) belongs to
__device__ __forceinline__ TreeUnit tree_at_step(const KvTreeArgs& a, int tile, int s) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int base = 0;; base += 64) {
    int len, nodes;
    const int mine = tree_steps(a, tile, base + lane, len, nodes), upto = before + wave_scan(mine);
    const unsigned long long later = __builtin_amdgcn_ballot_w64(upto > s);
    if (later || base + 64 >= a.batch) {
      const int at = later ? __builtin_ctzll(later) : 63;
      return tree_unit(base + at, __builtin_amdgcn_readlane(len, at), __builtin_amdgcn_readlane(nodes, at),
                       __builtin_amdgcn_readlane(upto - mine, at));
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
}

// The runs: workgroup w takes steps [start(w), start(w + 1))
struct TreeRuns {
  int count, per, longer;  // the first `longer` runs are one step longer
  __device__ __forceinline__ TreeRuns(int total, int wgs) {
    count = max(min(wgs, total), 1);
    per = total / count;
    longer = total - per * count;
  }
  __device__ __forceinline__ int start(int w) const { return w * per + min(w, longer); }
  __device__ __forceinline__ int of(int s) const {
    const int edge = longer * (per + 1);
    return s < edge ? s / (per + 1) : longer + (s - edge) / max(per, 1);
  }
};

template <int BITS, int RG, int RS>
struct KvTree {
  static constexpr int ROW = KvRegs<BITS>::ROW;
  static constexpr int TILE = 16 * RG * RS;
  static constexpr int WAVES = kTreePageWaves * RS;
  static constexpr bool Q_IN_LDS = RG > 2;  // else in registers: 16 of them per group
  static constexpr float kBias = BITS == 8 ? 1152.0f : 1032.0f;

  struct Shared {
    half8_t q[Q_IN_LDS ? RS * RG * 4 * 64 : 1];
    float red_o[WAVES][16][kHeadDim + 1];
    float red_ml[WAVES][16][2];
  };

  half8_t q[Q_IN_LDS ? 1 : RG][4];
  float qsum[RG];
  float m[RG], l[RG];  // l: this lane's keys only, until the merge
  float4_t o[RG][8];

  __device__ __forceinline__ half8_t query(const Shared& sh, int gi, int c, int rw, int lane) const {
    if constexpr (Q_IN_LDS)
      return sh.q[((rw * RG + gi) * 4 + c) * 64 + lane];
    else
      return q[gi][c];
  }

  // 16 rows' fragment c (dims in K-fragment order); rows past the last repeat it
  static __device__ __forceinline__ half8_t load_query(const KvTreeArgs& a, const TreeUnit& u, int hk, int row, int g,
                                                       int c) {
    const int r = min(row, u.nodes * a.G - 1), node = r / a.G;
    const _Float16* p = a.q + ((size_t)u.b * a.nodes + node) * a.ld_q + (hk * a.G + r - node * a.G) * kHeadDim +
                        32 * g + 8 * c;
    return in_key_order(*reinterpret_cast<const half8_t*>(p));
  }
  // 8 consecutive dims in the order of a K fragment: 4-bit codes come in pairs (s, s + 4)
  static __device__ __forceinline__ half8_t in_key_order(half8_t h) {
    if constexpr (BITS == 8)
      return h;
    else
      return half8_t{h[0], h[4], h[1], h[5], h[2], h[6], h[3], h[7]};
  }

  // Raises the references to the largest logits where any lane needs it; sv: NS logits per group, value scales included
  template <int NS>
  __device__ __forceinline__ void raise(const float (&sv)[RG][NS]) {
    float top[RG];
    bool any = false;
#pragma unroll
    for (int gi = 0; gi < RG; gi++) {
      top[gi] = sv[gi][0];
#pragma unroll
      for (int i = 1; i < NS; i++) top[gi] = fmaxf(top[gi], sv[gi][i]);
      any |= top[gi] > m[gi] + 4.f;
    }
    if (!__builtin_amdgcn_ballot_w64(any)) return;
#pragma unroll
    for (int gi = 0; gi < RG; gi++) {
      const float mn = fmaxf(m[gi], max_over_groups(top[gi]));
      const float alpha = __builtin_amdgcn_exp2f(m[gi] - mn);
      m[gi] = mn;
      l[gi] *= alpha;
#pragma unroll
      for (int db = 0; db < 8; db++) o[gi][db] *= alpha;
    }
  }

  // log2 |vs| and 1 / |vs|, a page of zero scale as if 2^-24 (its probabilities are dropped from O by fix_page)
  static __device__ __forceinline__ void value_scale(float vs, float& lv, float& rv) {
    const float av = vs == 0.f ? 0x1p-24f : fabsf(vs);
    lv = __builtin_amdgcn_logf(av);
    rv = __builtin_amdgcn_rcpf(av);
  }

  // Two pages, keys key0 .. key0 + 31
  __device__ __forceinline__ void process(const Shared& sh, const KvRegs<BITS>& ra, const KvRegs<BITS>& rb, int key0,
                                          int len, float qk_scale, int rw, int lane) {
    const int g = lane >> 4;
    float4_t sa[RG], sb[RG];
#pragma unroll
    for (int gi = 0; gi < RG; gi++) sa[gi] = sb[gi] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < 4; c++) {
      const half8_t ka = ra.kfrag(c), kb = rb.kfrag(c);
#pragma unroll
      for (int gi = 0; gi < RG; gi++) {
        const half8_t qv = query(sh, gi, c, rw, lane);
        sa[gi] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qv, sa[gi], 0, 0, 0);
        sb[gi] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb, qv, sb[gi], 0, 0, 0);
      }
    }
    const float sca = (float)ra.kscale() * qk_scale, scb = (float)rb.kscale() * qk_scale;
    const float va = (float)ra.vscale(), vb = (float)rb.vscale();
    float la, lb, na, nb;
    value_scale(va, la, na);
    value_scale(vb, lb, nb);
    float sv[RG][8];
#pragma unroll
    for (int gi = 0; gi < RG; gi++) {
      const float oa = __builtin_fmaf(-kBias * qsum[gi], sca, la), ob = __builtin_fmaf(-kBias * qsum[gi], scb, lb);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        sv[gi][i] = __builtin_fmaf(sa[gi][i], sca, oa);
        sv[gi][4 + i] = __builtin_fmaf(sb[gi][i], scb, ob);
      }
    }
    if (key0 + 2 * kPage > len) {  // the sequence ends inside these pages
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const bool in = key0 + (i < 4 ? 0 : kPage) + 4 * g + (i & 3) < len;
#pragma unroll
        for (int gi = 0; gi < RG; gi++) sv[gi][i] = in ? sv[gi][i] : -INFINITY;
      }
    }
    raise<8>(sv);
    half8_t pf[RG];
#pragma unroll
    for (int gi = 0; gi < RG; gi++) {
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; i++) {
        p[i] = __builtin_amdgcn_exp2f(sv[gi][i] - m[gi]);
        pf[gi][i] = (_Float16)p[i];
      }
      l[gi] = __builtin_fmaf((p[0] + p[1]) + (p[2] + p[3]), na, l[gi]);
      l[gi] = __builtin_fmaf((p[4] + p[5]) + (p[6] + p[7]), nb, l[gi]);
    }
    if (!(fminf(va, vb) > 0.f)) {  // a scale of zero or below: drop or flip that page's probabilities
#pragma unroll
      for (int gi = 0; gi < RG; gi++)
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float v = i < 4 ? va : vb;
          pf[gi][i] = v == 0.f ? (_Float16)0.f : v < 0.f ? -pf[gi][i] : pf[gi][i];
        }
    }
    uint32_t ta[8], tb[8];
    ra.vtrans(ta);
    rb.vtrans(tb);
#pragma unroll
    for (int db = 0; db < 8; db++) {
      const half4_t xa = codes_f16(ta[db], (_Float16)kBias), xb = codes_f16(tb[db], (_Float16)kBias);
      const half8_t v = __builtin_shufflevector(xa, xb, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
      for (int gi = 0; gi < RG; gi++)
        o[gi][db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pf[gi], o[gi][db], 0, 0, 0);
    }
  }

  // The nodes 16 t .. 16 t + 15 as keys
  __device__ __forceinline__ void process_nodes(const KvTreeArgs& a, const Shared& sh, const TreeUnit& u, int hk, int t,
                                                int row0, int rw, int lane) {
    const int n = lane & 15, g = lane >> 4, last = u.nodes - 1;
    const size_t seq = (size_t)u.b * a.nodes;
    half8_t kf[4], vr[4];
    const _Float16* kp = a.k_new + (seq + min(16 * t + n, last)) * a.ld_k + hk * kHeadDim + 32 * g;
#pragma unroll
    for (int c = 0; c < 4; c++) kf[c] = in_key_order(*reinterpret_cast<const half8_t*>(kp + 8 * c));
    unsigned long long odd[4], any_odd = 0;  // lanes whose 8 values of key 4g + i hold an infinity or NaN
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int key = 16 * t + 4 * g + i;
      vr[i] = *reinterpret_cast<const half8_t*>(a.v_new + (seq + min(key, last)) * a.ld_v + hk * kHeadDim + 8 * n);
      const kv_u32x4_t w = __builtin_bit_cast(kv_u32x4_t, vr[i]);
      bool bad = false;
#pragma unroll
      for (int e = 0; e < 4; e++) bad |= (w[e] & 0x7C00u) == 0x7C00u || (w[e] & 0x7C000000u) == 0x7C000000u;
      odd[i] = __builtin_amdgcn_ballot_w64(bad && key <= last);
      any_odd |= odd[i];
      // such a key would reach the rows that do not see it as 0 * inf: it leaves the product and is added below
      if ((odd[i] >> (16 * g) & 0xFFFF) || key > last) vr[i] = half8_t{};
    }
    float sv[RG][4];
    unsigned seen[RG];  // bit j: this row sees node 16 t + j
#pragma unroll
    for (int gi = 0; gi < RG; gi++) {
      const int node = min((row0 + 16 * gi + n) / a.G, last);
      const unsigned long long bits = a.mask ? a.mask[seq + node] : (2ull << node) - 1;
      seen[gi] = (unsigned)(bits >> (16 * t)) & (16 * t + 15 <= last ? 0xFFFFu : (1u << (last + 1 - 16 * t)) - 1);
      float4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 4; c++)
        s = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[c], query(sh, gi, c, rw, lane), s, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; i++) sv[gi][i] = (seen[gi] >> (4 * g + i) & 1) ? s[i] * a.qk_scale : -INFINITY;
    }
    raise<4>(sv);
#pragma unroll
    for (int gi = 0; gi < RG; gi++) {
      float p[4];
      half4_t pf;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        p[i] = __builtin_amdgcn_exp2f(sv[gi][i] - m[gi]);
        pf[i] = (_Float16)p[i];
      }
      l[gi] += (p[0] + p[1]) + (p[2] + p[3]);
#pragma unroll
      for (int db = 0; db < 8; db++)
        o[gi][db] = __builtin_amdgcn_mfma_f32_16x16x16f16(half4_t{vr[0][db], vr[1][db], vr[2][db], vr[3][db]}, pf,
                                                          o[gi][db], 0, 0, 0);
      if (any_odd) {
#pragma unroll 1
        for (int j = 0; j < 16; j++) {
          const unsigned long long lanes = (j & 3) == 0 ? odd[0] : (j & 3) == 1 ? odd[1] : (j & 3) == 2 ? odd[2] : odd[3];
          if (!(lanes >> (16 * (j >> 2)) & 0xFFFF)) continue;
          const float pj = (j & 3) == 0 ? p[0] : (j & 3) == 1 ? p[1] : (j & 3) == 2 ? p[2] : p[3];
          const float pk = __shfl(pj, n + 16 * (j >> 2));
          if (seen[gi] >> j & 1) {
            const _Float16* vp = a.v_new + (seq + 16 * t + j) * a.ld_v + hk * kHeadDim + 32 * g;
#pragma unroll
            for (int db = 0; db < 8; db++)
#pragma unroll
              for (int i = 0; i < 4; i++) o[gi][db][i] = __builtin_fmaf(pk, (float)vp[8 * i + db], o[gi][db][i]);
          }
        }
      }
    }
  }
};

template <int BITS, int RG, int RS>
__global__ __launch_bounds__(256 * RS, 2) void kv_tree_kernel(const KvTreeArgs a) {
  using T = KvTree<BITS, RG, RS>;
  constexpr int PS = kTreePageWaves;
  __shared__ typename T::Shared sh;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), pw = w % PS, rw = w / PS;
  const int total = tree_total(a, T::TILE);
  const TreeRuns runs(total, a.wgs);
  const int wg = blockIdx.x;
  if (wg >= runs.count) return;
  int s = runs.start(wg);
  const int s_end = runs.start(wg + 1);
  const size_t blk_bytes = (size_t)kPage * T::ROW;
  while (s < s_end) {
    const TreeUnit u = tree_at_step(a, T::TILE, s);
    const int tiles = (u.nodes * a.G + T::TILE - 1) / T::TILE;
    const int unit = (s - u.first) / u.steps;
    const int t0 = s - u.first - unit * u.steps, t1 = min(u.steps, t0 + s_end - s);
    const int hk = unit / tiles, row0 = (unit - hk * tiles) * T::TILE + rw * 16 * RG, rows = u.nodes * a.G;
    const int cache_end = min(t1, u.steps - 1);

    KvRegs<BITS> ra[2], rb[2];
    const int* ptab = a.page_table + (size_t)u.b * a.max_pages;
    auto page_of = [&](int lp) { return min(max(ptab[min(lp, u.pages - 1)], 0), a.num_pages - 1); };
    auto load = [&](int j, int pa, int pb) {
      const size_t ba = (size_t)pa * a.Hkv + hk, bb = (size_t)pb * a.Hkv + hk;
      ra[j].load(a.kc + ba * blk_bytes, a.vc + ba * blk_bytes, a.ksc, a.vsc, ba, n, g);
      rb[j].load(a.kc + bb * blk_bytes, a.vc + bb * blk_bytes, a.ksc, a.vsc, bb, n, g);
    };
    int t = t0, lp = t0 * kTreeStep + 2 * pw, pa = 0, pb = 0;
    if (t < cache_end) {
      load(0, page_of(lp), page_of(lp + 1));
      pa = page_of(lp + kTreeStep), pb = page_of(lp + kTreeStep + 1);
    }

    T x;
#pragma unroll
    for (int gi = 0; gi < RG; gi++) {
      x.m[gi] = kTreeLow, x.l[gi] = 0.f;
#pragma unroll
      for (int db = 0; db < 8; db++) x.o[gi][db] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
    if constexpr (T::Q_IN_LDS) {
      for (int i = pw; i < RG; i += PS)
#pragma unroll
        for (int c = 0; c < 4; c++)
          sh.q[((rw * RG + i) * 4 + c) * 64 + lane] = T::load_query(a, u, hk, row0 + 16 * i + n, g, c);
      __syncthreads();
    } else {
#pragma unroll
      for (int gi = 0; gi < RG; gi++)
#pragma unroll
        for (int c = 0; c < 4; c++) x.q[gi][c] = T::load_query(a, u, hk, row0 + 16 * gi + n, g, c);
    }
#pragma unroll
    for (int gi = 0; gi < RG; gi++) {
      float part = 0.f;
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const half8_t qv = x.query(sh, gi, c, rw, lane);
#pragma unroll
        for (int e = 0; e < 8; e++) part += (float)qv[e];
      }
      x.qsum[gi] = sum_over_groups(part);
    }

    // two register sets rotate: the next step's pages are in flight, and the ids of those after, while one is worked on
    bool more = t < cache_end;
    while (more) {
#pragma unroll
      for (int j = 0; j < 2; j++) {
        if (more) {
          load(j ^ 1, pa, pb);
          pa = page_of(lp + 2 * kTreeStep), pb = page_of(lp + 2 * kTreeStep + 1);
          issue_fence();
          x.process(sh, ra[j], rb[j], lp * kPage, u.len, a.qk_scale, rw, lane);
          lp += kTreeStep;
          more = ++t < cache_end;
        }
      }
    }
    if (t1 == u.steps && 16 * pw < u.nodes) x.process_nodes(a, sh, u, hk, pw, row0, rw, lane);

    // merge the page waves, 16 rows at a time; lane (n, g) holds dims 32g + 8i + db of row n
    const bool whole = t0 == 0 && t1 == u.steps;
    const int tid = threadIdx.x & 255, tq = tid >> 4, td = (tid & 15) * 8;
#pragma unroll
    for (int gi = 0; gi < RG; gi++) {
      const float lsum = sum_over_groups(x.l[gi]);
      if (gi > 0) __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int db = 0; db < 8; db++) sh.red_o[w][n][32 * g + 8 * i + db] = x.o[gi][db][i];
      if (g == 0) sh.red_ml[w][n][0] = x.m[gi], sh.red_ml[w][n][1] = lsum;
      __syncthreads();
      float mx = kTreeLow;
#pragma unroll
      for (int i = 0; i < PS; i++) mx = fmaxf(mx, sh.red_ml[rw * PS + i][tq][0]);
      float sum = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < PS; i++) {
        const float f = __builtin_amdgcn_exp2f(sh.red_ml[rw * PS + i][tq][0] - mx);
        sum += sh.red_ml[rw * PS + i][tq][1] * f;
#pragma unroll
        for (int e = 0; e < 8; e++) acc[e] += sh.red_o[rw * PS + i][tq][td + e] * f;
      }
      const int row = row0 + 16 * gi + tq;
      if (row < rows) {
        if (whole) {
          const int node = row / a.G, h = hk * a.G + row - node * a.G;
          half8_t r;
#pragma unroll
          for (int e = 0; e < 8; e++) r[e] = (_Float16)(sum == 0.f ? 0.f : acc[e] / sum);
          *reinterpret_cast<half8_t*>(a.out + (((size_t)u.b * a.nodes + node) * a.Hq + h) * kHeadDim + td) = r;
        } else {
          // a run has at most two parts of split units: the end of one (slot 0) and the beginning of another (slot 1)
          const size_t at = ((size_t)wg * 2 + (t0 == 0)) * T::TILE + rw * 16 * RG + 16 * gi + tq;
          float4_t* po = reinterpret_cast<float4_t*>(a.part_o + at * kHeadDim + td);
          po[0] = float4_t{acc[0], acc[1], acc[2], acc[3]};
          po[1] = float4_t{acc[4], acc[5], acc[6], acc[7]};
          if (td == 0) a.part_ml[at * 2] = mx, a.part_ml[at * 2 + 1] = sum;
        }
      }
    }
    __syncthreads();
    s += t1 - t0;
  }
}

// Joins the parts of split units: one workgroup per (16 rows, unit of the sequence, sequence)
template <int TILE>
__global__ __launch_bounds__(256) void kv_tree_merge_kernel(const KvTreeArgs a) {
  const int total = tree_total(a, TILE);
  const TreeRuns runs(total, a.wgs);
  const int b = blockIdx.z, unit = blockIdx.y, group = blockIdx.x;
  int first = 0, len = 0, nodes = 0, steps = 0;
  for (int base = 0; base <= b; base += 64) {  // the sequence's first step
    const int mine = tree_steps(a, TILE, base + (threadIdx.x & 63), len, nodes), upto = first + wave_scan(mine);
    if (b < base + 64) {
      first = __builtin_amdgcn_readlane(upto - mine, b - base);
      len = __builtin_amdgcn_readlane(len, b - base);
      nodes = __builtin_amdgcn_readlane(nodes, b - base);
      steps = tree_unit(b, len, nodes, first).steps;
    } else {
      first = __builtin_amdgcn_readlane(upto, 63);
    }
  }
  const int rows = nodes * a.G, tiles = (rows + TILE - 1) / TILE;
  if (unit >= a.Hkv * tiles) return;
  const int hk = unit / tiles, row = (unit - hk * tiles) * TILE + 16 * group + (threadIdx.x >> 4);
  const int td = (threadIdx.x & 15) * 8;
  const int s0 = first + unit * steps, w0 = runs.of(s0), w1 = runs.of(s0 + steps - 1);
  if (w0 == w1 || row >= rows) return;
  float mx = kTreeLow, sum = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int w = w0; w <= w1; w++) {
    const size_t at = ((size_t)w * 2 + (w == w0)) * TILE + 16 * group + (threadIdx.x >> 4);
    const float mw = a.part_ml[at * 2], lw = a.part_ml[at * 2 + 1];
    const float4_t* po = reinterpret_cast<const float4_t*>(a.part_o + at * kHeadDim + td);
    const float4_t x = po[0], y = po[1];
    const float mn = fmaxf(mx, mw);
    const float fa = __builtin_amdgcn_exp2f(mx - mn), fw = __builtin_amdgcn_exp2f(mw - mn);
    sum = sum * fa + lw * fw;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      acc[e] = acc[e] * fa + x[e] * fw;
      acc[4 + e] = acc[4 + e] * fa + y[e] * fw;
    }
    mx = mn;
  }
  const int node = row / a.G, h = hk * a.G + row - node * a.G;
  half8_t r;
#pragma unroll
  for (int e = 0; e < 8; e++) r[e] = (_Float16)(sum == 0.f ? 0.f : acc[e] / sum);
  *reinterpret_cast<half8_t*>(a.out + (((size_t)b * a.nodes + node) * a.Hq + h) * kHeadDim + td) = r;
}

// Groups of 16 rows per wave, halves of the rows per workgroup, and the most workgroups of the launch (a run each)
struct TreePlan {
  int rg, rs, tile, tiles, wgs;
  long long steps;  // of a batch that fills its tables
};
static TreePlan tree_plan(int batch, int nodes, int num_q_heads, int num_kv_heads, int max_pages) {
  const int groups = (nodes * (num_q_heads / num_kv_heads) + 15) / 16;
  TreePlan p;
  if (groups <= 4) {
    p.rg = groups, p.rs = 1;
  } else if (groups <= 8) {
    p.rg = (groups + 1) / 2, p.rs = 2;
  } else {
    p.rg = 4, p.rs = 1;
  }
  p.tile = 16 * p.rg * p.rs;
  p.tiles = (groups * 16 + p.tile - 1) / p.tile;
  p.steps = (long long)batch * num_kv_heads * p.tiles * ((max_pages + kTreeStep - 1) / kTreeStep + 1);
  p.wgs = (int)std::min<long long>(512 / p.rs, p.steps);
  return p;
}

}  // namespace exl3

using namespace exl3;

extern "C" size_t exl3_kv_tree_workspace_bytes(int batch, int nodes, int num_q_heads, int num_kv_heads, int max_pages) {
  if (batch <= 0 || nodes <= 0 || nodes > kTreeNodes || num_kv_heads <= 0 || num_q_heads % num_kv_heads ||
      num_q_heads / num_kv_heads < 1 || num_q_heads / num_kv_heads > kMaxGroup || max_pages <= 0)
    return 0;
  const TreePlan p = tree_plan(batch, nodes, num_q_heads, num_kv_heads, max_pages);
  return (size_t)p.wgs * 2 * p.tile * (kHeadDim + 2) * sizeof(float);
}

extern "C" int exl3_kv_tree_attention(const void* q, long long ld_q, const void* k_new, const void* v_new,
                                      long long ld_k, long long ld_v, const void* tree_mask, int nodes,
                                      const int* num_nodes, const void* k_cache, const void* v_cache,
                                      const void* k_scale, const void* v_scale, int num_pages, const int* page_table,
                                      int max_pages, const int* seq_lens, int batch, int num_q_heads, int num_kv_heads,
                                      int head_dim, int page_size, int bits, float sm_scale, void* out, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  EXL3_CHECK_ARG(k_cache && v_cache && k_scale && v_scale, "exl3_kv_tree_attention: null pointer");
  EXL3_CHECK_ARG(head_dim == kHeadDim && page_size == kPage,
                 "exl3_kv_tree_attention: head_dim = %d, page_size = %d (supported: 128, 16)", head_dim, page_size);
  EXL3_CHECK_ARG(bits == 4 || bits == 8, "exl3_kv_tree_attention: bits = %d (4 or 8)", bits);
  EXL3_CHECK_ARG(nodes >= 1 && nodes <= kTreeNodes, "exl3_kv_tree_attention: nodes = %d (1 to 64)", nodes);
  EXL3_CHECK_ARG(batch >= 0 && batch <= 65535 && num_pages >= 1 && num_pages <= (1 << 26) && max_pages >= 1 &&
                     max_pages <= (1 << 26) && num_kv_heads >= 1 && num_kv_heads <= 1024 &&
                     num_q_heads % num_kv_heads == 0 && num_q_heads / num_kv_heads >= 1 &&
                     num_q_heads / num_kv_heads <= kMaxGroup,
                 "exl3_kv_tree_attention: batch = %d, pages = %d, max_pages = %d, heads %d / %d (group <= 16)", batch,
                 num_pages, max_pages, num_q_heads, num_kv_heads);
  if (batch == 0) return EXL3_OK;
  EXL3_CHECK_ARG(q && k_new && v_new && page_table && seq_lens && out, "exl3_kv_tree_attention: null pointer");
  EXL3_CHECK_ARG(ld_q >= (long long)num_q_heads * head_dim && ld_k >= (long long)num_kv_heads * head_dim &&
                     ld_v >= (long long)num_kv_heads * head_dim && (ld_q | ld_k | ld_v) % 8 == 0,
                 "exl3_kv_tree_attention: token strides %lld / %lld / %lld (multiples of 8, a token's heads at least)",
                 ld_q, ld_k, ld_v);
  EXL3_CHECK_ARG((((uintptr_t)q | (uintptr_t)k_new | (uintptr_t)v_new | (uintptr_t)k_cache | (uintptr_t)v_cache |
                   (uintptr_t)out | (uintptr_t)workspace) & 15) == 0,
                 "exl3_kv_tree_attention: a tensor is not 16-byte aligned");
  const TreePlan p = tree_plan(batch, nodes, num_q_heads, num_kv_heads, max_pages);
  EXL3_CHECK_ARG(p.steps < (1LL << 31), "exl3_kv_tree_attention: batch = %d of %d pages is too large", batch, max_pages);
  const size_t slots = (size_t)p.wgs * 2 * p.tile, need = slots * (kHeadDim + 2) * sizeof(float);
  EXL3_CHECK_ARG(workspace && workspace_bytes >= need, "exl3_kv_tree_attention: workspace %zu bytes, need %zu",
                 workspace_bytes, need);
  float* part_o = static_cast<float*>(workspace);
  const KvTreeArgs a{static_cast<const _Float16*>(q), static_cast<const _Float16*>(k_new),
                     static_cast<const _Float16*>(v_new), ld_q, ld_k, ld_v,
                     static_cast<const unsigned long long*>(tree_mask), num_nodes,
                     static_cast<const uint8_t*>(k_cache), static_cast<const uint8_t*>(v_cache),
                     static_cast<const uint16_t*>(k_scale), static_cast<const uint16_t*>(v_scale), num_pages, page_table,
                     max_pages, seq_lens, batch, nodes, num_q_heads, num_kv_heads, num_q_heads / num_kv_heads,
                     sm_scale * 1.4426950408889634f, p.wgs, part_o, part_o + slots * kHeadDim,
                     static_cast<_Float16*>(out)};
  hipStream_t st = as_stream(stream);
  using Kern = decltype(&kv_tree_kernel<8, 1, 1>);
#define EXL3_TREE_BITS(RG, RS) {kv_tree_kernel<4, RG, RS>, kv_tree_kernel<8, RG, RS>}
  static const Kern one[4][2] = {EXL3_TREE_BITS(1, 1), EXL3_TREE_BITS(2, 1), EXL3_TREE_BITS(3, 1), EXL3_TREE_BITS(4, 1)};
  static const Kern two[2][2] = {EXL3_TREE_BITS(3, 2), EXL3_TREE_BITS(4, 2)};
#undef EXL3_TREE_BITS
  (p.rs == 1 ? one[p.rg - 1] : two[p.rg - 3])[bits == 8]<<<p.wgs, 256 * p.rs, 0, st>>>(a);
  EXL3_CHECK_LAUNCH();
  auto merge = p.tile == 16   ? kv_tree_merge_kernel<16>
               : p.tile == 32 ? kv_tree_merge_kernel<32>
               : p.tile == 48 ? kv_tree_merge_kernel<48>
               : p.tile == 64 ? kv_tree_merge_kernel<64>
               : p.tile == 96 ? kv_tree_merge_kernel<96>
                              : kv_tree_merge_kernel<128>;
  merge<<<dim3(p.tile / 16, num_kv_heads * p.tiles, batch), 256, 0, st>>>(a);
  EXL3_CHECK_LAUNCH();
  return EXL3_OK;
}
