// Attention of drafted tokens, a tree or a chain per sequence, over the paged quantized KV cache (gfx950).
//
//   o[i] = softmax(sm_scale q_i [K_cache ; K_nodes]^T) [V_cache ; V_nodes]
// for nodes i < 64 of every sequence: all of them see the cached tokens, and those nodes whose bits their mask sets.  The
// nodes' keys and values come in fp16 (they enter the cache, quantized, once verified).  Cache layout and the MFMA forms of a
// page: kv_attention.hip; a query row here is a (node, query head) pair of one kv head.
//
// A wave keeps RG groups of 16 rows and takes two pages (32 keys) at a time:
//   S^T = K Q^T     4 x MFMA 16x16x32 per page and group
//   O^T += V^T P^T  8 x MFMA 16x16x32 per group: slots 0..3 of a lane's 8 keys are its keys of the first page, 4..7 of the
//                   second, so the C layout of the two S^T is the B operand as it stands
// Softmax in base 2 with a lazy reference: O, l are rescaled only when a logit passes the reference by more than 15.  The
// page's value scale is folded into the exponent (p' = 2^(s + log2 vs - m)), so a step has no multiplication per
// probability; the sum takes p' / vs, once per page and row, in fp32.  P' is rounded to fp16 for the second product, which
// takes both operands in one 16-bit type: fp16 holds every code and 3 bits more of P' than bf16 would (half a step: 2^-12 to
// 2^-11 of a key's share).  Its range is the other limit, steps of 2^-24 at the bottom.  The reference therefore lies 11 below
// a row's largest exponent when it is set, so the largest P' stays between 2^11 and 2^15, and a tile of nodes is brought to
// the size of codes by a power of two, like a page of that scale.  With P' of at least 2^11 against codes of 127 each key
// below fp16's range costs an output at most 2^-25 * 2^-11 of the largest value (2^-35 where that is a node's).
//
// Two forms.  Up to 96 rows (split): every wave of a workgroup of 4 works on pages of its own, codes straight into LDS stages
// of the wave, no barrier until the waves' states are merged in LDS; up to 32 rows two workgroups share a CU, with more rows a
// wave has a SIMD's registers to itself.  Long contexts (16 sequences up to 32768 tokens, 40 / 8 heads, 8 bits) run at 5.2, 4.8
// and 4.7 TB/s with 3, 5 and 9 nodes, what the memory gives here; with more rows issue takes over (16 nodes 3.2 to 3.5 TB/s,
// 520 to 560 TFLOP/s; 4 bits 590): a step of 80 rows holds 1280 cycles of MFMA in some 5000, one wave's chain of products,
// softmax and products.  More rows (shared): decoding codes for 64 rows costs as much as their softmax, so the 8 waves of a
// workgroup decode a tile of 4 pages together, as MFMA fragments in LDS, and each runs it against rows of its own (64 nodes:
// 810 to 830 TFLOP/s at 8 bits, 870 to 920 at 4; a large fp16 matrix product reaches 1140 here).  Bound by issue there: MFMA
// takes 41 % and VALU 56 % of a SIMD's cycles, at a clock of 2.0 GHz under that load, and the two waves of a SIMD hardly
// overlap them (the products at a higher wave priority: 3 %; staggering the waves' shares of decoding: nothing).
// 24 nodes (one group of rows a wave: each fragment read from LDS feeds one product): 520 to 590 TFLOP/s.
//
// Work split: a unit is (sequence, kv head, tile of rows), its step 0 the nodes, each further one a workgroup's pages at a
// time.  The steps of all units in a row are dealt to the workgroups in equal runs, whatever the lengths: a unit inside
// one run is written directly, the parts of a split one go to the workspace and kv_tree_merge_kernel joins them in order
// (deterministic).
#include <algorithm>

#include "exl3_api.hpp"
#include "kv_device.hpp"

namespace exl3 {

constexpr int kTreeNodes = 64;        // a bit of the mask each
constexpr int kSplitWaves = 4;        // split: waves that take two pages each per step
constexpr int kSharedSlots = 8;       // shared: waves; each takes rows, and all decode a step's pages
constexpr int kSharedPages = 4;       // pages per step
constexpr int kSharedGroups = 3;      // most groups of 16 rows per wave
constexpr int kSplitGroups = 6;
constexpr int kPairedGroups = 2;      // split: up to as many, two workgroups share a CU
constexpr int kTreeExtra = 6;         // most steps that the beginning of a unit counts for
constexpr float kTreeHead = 11.f;     // what a row's largest exponent is brought to (P' in fp16: to 2^15, no overflow)
constexpr float kTreeBar = 15.f;      // exponents above it move a row's reference
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
  int tile, step;  // rows of a unit, pages of a step
  float *part_o, *part_ml;
  _Float16* out;
};

// The row of all steps.  Workgroup w takes the steps [start(w), start(w + 1)) of the `total`.  A part of a unit costs about
// as much to begin and to merge as several steps, and a run has one part more for every unit that begins in it: so a unit
// counts `extra` steps more than it has (16 sequences of 256 .. 4096 tokens, 64 nodes, 40 / 8 heads, 8 bits, both launches:
// 123 us with 2, 108.5 with 6; 16 nodes 52.6 and 51.1, this kernel 56 without any and 45).
struct TreeRuns {
  int extra, total, count, per, longer;  // the first `longer` runs are one step longer
  int len0, nodes0, units0;              // of sequence `lane` (KEPT: for tree_find, for 3 registers)

  __device__ __forceinline__ explicit TreeRuns(const KvTreeArgs& a) {
    const int lane = threadIdx.x & 63;
    int steps = 0, units = 0;
    for (int base = 0; base < a.batch; base += 64) {
      int len, nodes;
      const int u = units_of(a, base + lane, len, nodes);
      if (base == 0) len0 = len, nodes0 = nodes, units0 = u;
      units += wave_total(u);
      steps += wave_total(u * steps_of(a, len));
    }
    extra = min(max(steps / a.wgs / 3, 0), kTreeExtra);
    total = steps + extra * units;
    count = max(min(a.wgs, total), 1);
    per = total / count;
    longer = total - per * count;
  }
  __device__ __forceinline__ int start(int w) const { return w * per + min(w, longer); }
  __device__ __forceinline__ int of(int s) const {
    const int edge = longer * (per + 1);
    return s < edge ? s / (per + 1) : longer + (s - edge) / max(per, 1);
  }

  // units of sequence b (0 past the batch), and what they come from
  static __device__ __forceinline__ int units_of(const KvTreeArgs& a, int b, int& len, int& nodes) {
    const int at = min(b, a.batch - 1);
    len = max(min(a.seq_lens[at], a.max_pages * kPage), 0);
    nodes = a.num_nodes ? max(min(a.num_nodes[at], a.nodes), 0) : a.nodes;
    nodes = b < a.batch ? nodes : 0;
    return a.Hkv * ((nodes * a.G + a.tile - 1) / a.tile);
  }
  static __device__ __forceinline__ int steps_of(const KvTreeArgs& a, int len) {
    return ((len + kPage - 1) / kPage + a.step - 1) / a.step + 1;
  }
};

// A sequence, and its place in the row
struct TreeUnit {
  int b, len, nodes, pages, steps;  // steps: of one of its units
  int first;                        // the sequence's first step
};

__device__ __forceinline__ TreeUnit tree_unit(const KvTreeArgs& a, const TreeRuns& runs, int b, int len, int nodes,
                                              int first) {
  return TreeUnit{b, len, nodes, (len + kPage - 1) / kPage, runs.steps_of(a, len) + runs.extra, first};
}

// The sequence that `found(first, end)` picks by its first step and the one after its last, among the lanes' sequences
template <bool KEPT, typename Found>
__device__ __forceinline__ TreeUnit tree_find(const KvTreeArgs& a, const TreeRuns& runs, Found found) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int base = 0;; base += 64) {
    int len = runs.len0, nodes = runs.nodes0;
    const int units = !KEPT || base > 0 ? runs.units_of(a, base + lane, len, nodes) : runs.units0;
    const int mine = units * (runs.steps_of(a, len) + runs.extra);
    const int upto = before + wave_scan(mine);
    const unsigned long long hit = __builtin_amdgcn_ballot_w64(found(base + lane, upto));
    if (hit || base + 64 >= a.batch) {
      const int at = hit ? __builtin_ctzll(hit) : 63;
      return tree_unit(a, runs, base + at, __builtin_amdgcn_readlane(len, at), __builtin_amdgcn_readlane(nodes, at),
                       __builtin_amdgcn_readlane(upto - mine, at));
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
}
// ... the one that step s (below the total) belongs to
template <bool KEPT>
__device__ __forceinline__ TreeUnit tree_at_step(const KvTreeArgs& a, const TreeRuns& runs, int s) {
  return tree_find<KEPT>(a, runs, [&](int, int end) { return end > s; });
}

// The state of RG groups of 16 rows in a wave: lane (n, g) = (l % 16, l / 16) holds row n of each group
template <int BITS, int RG>
struct TreeRows {
  static constexpr float kBias = BITS == 8 ? 1152.0f : 1032.0f;

  half8_t q[RG][4];
  float qsum[RG];      // -bias times the row's sum: what the biased codes of K add to its logits
  float m[RG], l[RG];  // the row's reference; l: this lane's keys only, until the end
  float bar[RG];       // -inf until the row has seen a key
  float4_t o[RG][8];

  // 8 consecutive dims in the order of a K fragment: 4-bit codes come in pairs (s, s + 4)
  static __device__ __forceinline__ half8_t in_key_order(half8_t h) {
    if constexpr (BITS == 8)
      return h;
    else
      return half8_t{h[0], h[4], h[1], h[5], h[2], h[6], h[3], h[7]};
  }

  // 16 rows from row0 on per group (rows past the unit's last repeat it)
  __device__ __forceinline__ void load_queries(const KvTreeArgs& a, const TreeUnit& u, int hk, int row0, int n, int g) {
#pragma unroll
    for (int gi = 0; gi < RG; gi++) {
      const int r = min(row0 + 16 * gi + n, u.nodes * a.G - 1), node = r / a.G;
      const _Float16* p = a.q + ((size_t)u.b * a.nodes + node) * a.ld_q + (hk * a.G + r - node * a.G) * kHeadDim + 32 * g;
#pragma unroll
      for (int c = 0; c < 4; c++) q[gi][c] = in_key_order(*reinterpret_cast<const half8_t*>(p + 8 * c));
    }
  }
  // The same by a workgroup of 4 waves: wave w brings rows 4 w .. 4 w + 3 of each group into LDS, one 256-byte row per 16
  // lanes, piece p (8 dims) of row r at place p ^ r.  Each wave loading its own fragments takes four times as many loads,
  // of 16 bytes from 64 places each.
  using Staging = half8_t[RG][16][16];
  static __device__ __forceinline__ void stage_queries(const KvTreeArgs& a, const TreeUnit& u, int hk, int row0, int w,
                                                       int lane, Staging& to) {
    const int rr = 4 * w + (lane >> 4), piece = (lane & 15) ^ rr;
#pragma unroll
    for (int gi = 0; gi < RG; gi++) {
      const int r = min(row0 + 16 * gi + rr, u.nodes * a.G - 1), node = r / a.G;
      const _Float16* p = a.q + ((size_t)u.b * a.nodes + node) * a.ld_q + (hk * a.G + r - node * a.G) * kHeadDim + 8 * piece;
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)p,
                                       (__attribute__((address_space(3))) void*)to[gi][4 * w], 16, 0, 0);
    }
  }
  // ... in the order of the key fragments, each wave its own pieces
  static __device__ __forceinline__ void order_queries(int w, int lane, Staging& q) {
    if constexpr (BITS == 4) {
#pragma unroll
      for (int gi = 0; gi < RG; gi++) {
        half8_t& h = q[gi][4 * w + (lane >> 4)][lane & 15];
        h = in_key_order(h);
      }
    }
  }
  __device__ __forceinline__ void read_queries(const Staging& from, int n, int g) {
#pragma unroll
    for (int gi = 0; gi < RG; gi++)
#pragma unroll
      for (int c = 0; c < 4; c++) q[gi][c] = from[gi][n][(4 * g + c) ^ n];
  }
  __device__ __forceinline__ void start() {
#pragma unroll
    for (int gi = 0; gi < RG; gi++) {
      float part = 0.f;
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const kv_u32x4_t w = __builtin_bit_cast(kv_u32x4_t, q[gi][c]);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const uint32_t two = w[e];
          part = __builtin_amdgcn_fdot2(__builtin_bit_cast(half2_t, two), half2_t{(_Float16)1.f, (_Float16)1.f}, part, false);
        }
      }
      qsum[gi] = -kBias * sum_over_groups(part);
      m[gi] = 0.f, l[gi] = 0.f, bar[gi] = -INFINITY;
#pragma unroll
      for (int db = 0; db < 8; db++) o[gi][db] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
  }

  // fmaxf would first quiet each operand that it cannot prove to be no signalling NaN
  static __device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
  }

  // x: NS exponents per group, relative to the references.  Where a lane has one past its bar the references move to
  // kTreeHead below the largest: once a row has seen a key the bar is kTreeBar, before that any key passes it.
  template <int NS>
  __device__ __forceinline__ void raise(float (&x)[RG][NS]) {
    float top[RG];
    bool any = false;
#pragma unroll
    for (int gi = 0; gi < RG; gi++) {
      top[gi] = max3(x[gi][0], x[gi][1], x[gi][2]);
#pragma unroll
      for (int i = 3; i < NS; i += 2) top[gi] = max3(top[gi], x[gi][i], x[gi][i + 1 < NS ? i + 1 : i]);
      any |= top[gi] > bar[gi];
    }
    if (!__builtin_amdgcn_ballot_w64(any)) return;
#pragma unroll
    for (int gi = 0; gi < RG; gi++) {
      const float t = max_over_groups(top[gi]) - kTreeHead;
      const float d = fmaxf(t, bar[gi] == kTreeBar ? 0.f : kTreeLow);  // the first keys of a row lower it too
      if (t > -INFINITY || bar[gi] == kTreeBar) {
        bar[gi] = kTreeBar;
        // (an empty row's l and o are zeros: with logits of -128 and below exp2(-d) would make them 0 * inf)
        const float alpha = __builtin_amdgcn_exp2f(-fmaxf(d, 0.f));
        m[gi] += d;
        l[gi] *= alpha;
#pragma unroll
        for (int db = 0; db < 8; db++) o[gi][db] *= alpha;
#pragma unroll
        for (int i = 0; i < NS; i++) x[gi][i] -= d;
      }
    }
  }

  // P^T of NP pages from their unscaled logits.  k: the pages' key scales times qk_scale, lv: log2 of their value scales,
  // nv: 1 over those; hide(x) puts -inf in the place of keys that do not count, if `some`; odd: a value scale of zero or
  // below (then keep and flip apply, per page)
  template <int NP, typename Hide>
  __device__ __forceinline__ void softmax(const float4_t (&s)[NP][RG], const float (&k)[NP], const float (&lv)[NP],
                                          const float (&nv)[NP], bool some, Hide hide, bool odd, const uint32_t (&keep)[NP],
                                          const uint32_t (&flip)[NP], half8_t (&pf)[NP / 2][RG]) {
    float x[RG][4 * NP];
#pragma unroll
    for (int gi = 0; gi < RG; gi++)
#pragma unroll
      for (int j = 0; j < NP; j++) {
        const float off = __builtin_fmaf(qsum[gi], k[j], lv[j] - m[gi]);
#pragma unroll
        for (int i = 0; i < 4; i++) x[gi][4 * j + i] = __builtin_fmaf(s[j][gi][i], k[j], off);
      }
    if (some) hide(x);
    raise<4 * NP>(x);
    kv_u32x4_t packed[NP / 2][RG];
#pragma unroll
    for (int gi = 0; gi < RG; gi++)
#pragma unroll
      for (int h = 0; h < NP / 2; h++) {
        float p[8];
        half8_t r;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          p[i] = __builtin_amdgcn_exp2f(x[gi][8 * h + i]);
          r[i] = (_Float16)p[i];
        }
        l[gi] = __builtin_fmaf((p[0] + p[1]) + (p[2] + p[3]), nv[2 * h], l[gi]);
        l[gi] = __builtin_fmaf((p[4] + p[5]) + (p[6] + p[7]), nv[2 * h + 1], l[gi]);
        packed[h][gi] = __builtin_bit_cast(kv_u32x4_t, r);
        asm("" : "+v"(packed[h][gi]));  // converted in pairs here, whether or not the branch below is taken
      }
    if (odd) {
#pragma unroll
      for (int gi = 0; gi < RG; gi++)
#pragma unroll
        for (int h = 0; h < NP / 2; h++)
          packed[h][gi] = (packed[h][gi] & kv_u32x4_t{keep[2 * h], keep[2 * h], keep[2 * h + 1], keep[2 * h + 1]}) ^
                          kv_u32x4_t{flip[2 * h], flip[2 * h], flip[2 * h + 1], flip[2 * h + 1]};
    }
#pragma unroll
    for (int gi = 0; gi < RG; gi++)
#pragma unroll
      for (int h = 0; h < NP / 2; h++) pf[h][gi] = __builtin_bit_cast(half8_t, packed[h][gi]);
  }

  // The reference, below any other while the row has seen nothing
  __device__ __forceinline__ float reference(int gi) const { return bar[gi] == kTreeBar ? m[gi] : kTreeLow; }

  // The nodes 16 t .. 16 t + 15 as keys: their fragments, and what each row sees of them
  struct Nodes {
    half8_t k[4], v[4];
    unsigned long long mask[RG];
    __device__ __forceinline__ void load(const KvTreeArgs& a, const TreeUnit& u, int hk, int t, int row0, int n, int g) {
      const int last = u.nodes - 1;
      const size_t seq = (size_t)u.b * a.nodes;
      const _Float16* kp = a.k_new + (seq + min(16 * t + n, last)) * a.ld_k + hk * kHeadDim + 32 * g;
#pragma unroll
      for (int c = 0; c < 4; c++) k[c] = *reinterpret_cast<const half8_t*>(kp + 8 * c);
#pragma unroll
      for (int i = 0; i < 4; i++)
        v[i] = *reinterpret_cast<const half8_t*>(a.v_new + (seq + min(16 * t + 4 * g + i, last)) * a.ld_v + hk * kHeadDim +
                                                 8 * n);
#pragma unroll
      for (int gi = 0; gi < RG; gi++) {
        const int node = min((row0 + 16 * gi + n) / a.G, last);
        mask[gi] = a.mask ? a.mask[seq + node] : (2ull << node) - 1;
      }
    }
  };
  __device__ __forceinline__ void process_nodes(const KvTreeArgs& a, const TreeUnit& u, int hk, int t, const Nodes& in,
                                                int lane) {
    const int n = lane & 15, g = lane >> 4, last = u.nodes - 1;
    const size_t seq = (size_t)u.b * a.nodes;
    half8_t kf[4], vr[4];
#pragma unroll
    for (int c = 0; c < 4; c++) kf[c] = in_key_order(in.k[c]);
    unsigned long long odd[4], any_odd = 0;  // lanes whose 8 values of key 4g + i hold an infinity or NaN
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int key = 16 * t + 4 * g + i;
      vr[i] = in.v[i];
      const kv_u32x4_t w = __builtin_bit_cast(kv_u32x4_t, vr[i]);
      bool bad = false;
#pragma unroll
      for (int e = 0; e < 4; e++) bad |= (w[e] & 0x7C00u) == 0x7C00u || (w[e] & 0x7C000000u) == 0x7C000000u;
      odd[i] = __builtin_amdgcn_ballot_w64(bad && key <= last);
      any_odd |= odd[i];
      // such a key would reach the rows that do not see it as 0 * inf: it leaves the product and is added below
      if ((odd[i] >> (16 * g) & 0xFFFF) || key > last) vr[i] = half8_t{};
    }
    // values times 2^up: the largest in [64, 128), where the least step of P' costs what it costs a page of codes
    uint32_t pairs = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const kv_u32x4_t w = __builtin_bit_cast(kv_u32x4_t, vr[i]);
#pragma unroll
      for (int e = 0; e < 4; e++) pairs = max_u16x2(pairs, w[e] & 0x7FFF7FFFu);
    }
    const int up = min(max(21 - (int)(wave_max_u32(max(pairs & 0xFFFFu, pairs >> 16)) >> 10), 0), 15);
    const _Float16 vup = __builtin_bit_cast(_Float16, (uint16_t)((15 + up) << 10));
#pragma unroll
    for (int i = 0; i < 4; i++) vr[i] *= vup;
    float x[RG][4];
    unsigned seen[RG];  // bit j: this row sees node 16 t + j
#pragma unroll
    for (int gi = 0; gi < RG; gi++) {
      seen[gi] = (unsigned)(in.mask[gi] >> (16 * t)) & (16 * t + 15 <= last ? 0xFFFFu : (1u << (last + 1 - 16 * t)) - 1);
      float4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 4; c++)
        s = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[c], q[gi][c], s, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; i++)
        x[gi][i] = (seen[gi] >> (4 * g + i) & 1) ? __builtin_fmaf(s[i], a.qk_scale, -m[gi] - (float)up) : -INFINITY;
    }
    raise<4>(x);
#pragma unroll
    for (int gi = 0; gi < RG; gi++) {
      float p[4];
      half4_t pf;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        p[i] = __builtin_amdgcn_exp2f(x[gi][i]);
        pf[i] = (_Float16)p[i];
      }
      l[gi] = __builtin_fmaf((p[0] + p[1]) + (p[2] + p[3]), (float)vup, l[gi]);
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
          const float pk = __shfl(pj, n + 16 * (j >> 2)) * (float)vup;
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

// s_waitcnt vmcnt(n) for a uniform n of at most MOST
template <int MOST, int EACH = 1>
__device__ __forceinline__ void wait_loads(int n) {
  if constexpr (MOST == 0) {
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
  } else {
    if (n >= MOST)
      __builtin_amdgcn_s_waitcnt(waitcnt_vm(MOST * EACH));
    else
      wait_loads<MOST - 1, EACH>(n);
  }
}

// What softmax takes of a page's scales, per lane a page
struct PageScales {
  uint16_t kraw, vraw;
  float k, l, n;           // key scale times qk_scale; log2 |v| and 1 / |v| of the value scale
  unsigned long long odd;  // lanes whose value scale is 0 or below
  __device__ __forceinline__ void load(const KvTreeArgs& a, int page, int hk) {
    const size_t at = (size_t)page * a.Hkv + hk;
    kraw = a.ksc[at], vraw = a.vsc[at];
  }
  __device__ __forceinline__ void use(float qk_scale) {
    k = (float)__builtin_bit_cast(_Float16, kraw) * qk_scale;
    const float v = (float)__builtin_bit_cast(_Float16, vraw);
    const float av = v == 0.f ? 0x1p-24f : fabsf(v);  // a page of scale 0 counts as if it were 2^-24; its P' are dropped
    l = __builtin_amdgcn_logf(av);
    n = __builtin_amdgcn_rcpf(av);
    odd = __builtin_amdgcn_ballot_w64(v <= 0.f);
  }
  __device__ __forceinline__ uint32_t keep(int i) const {
    return (__builtin_amdgcn_readlane((int)vraw, i) & 0x7FFF) ? ~0u : 0u;
  }
  __device__ __forceinline__ uint32_t flip(int i) const {
    return (__builtin_amdgcn_readlane((int)vraw, i) & 0x8000) ? 0x80008000u : 0u;
  }
};
__device__ __forceinline__ float lane_of(float v, int i) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), i));
}
// softmax of NP pages, keys key0 on: pages of A from lane ia on; with B, those of lane ia of A and of lane ia of B
template <int BITS, int RG, int NP>
__device__ __forceinline__ void tree_softmax(TreeRows<BITS, RG>& x, const float4_t (&s)[NP][RG], const PageScales& A,
                                             const PageScales* B, int ia, int key0, int len, int g,
                                             half8_t (&pf)[NP / 2][RG]) {
  float k[NP], lv[NP], nv[NP];
  uint32_t keep[NP], flip[NP];
  bool odd = false;
#pragma unroll
  for (int j = 0; j < NP; j++) {
    const PageScales& S = B && j ? *B : A;
    const int i = B ? ia : ia + j;
    k[j] = lane_of(S.k, i), lv[j] = lane_of(S.l, i), nv[j] = lane_of(S.n, i);
    odd |= S.odd >> i & 1;
    keep[j] = ~0u, flip[j] = 0u;
  }
  if (odd) {
#pragma unroll
    for (int j = 0; j < NP; j++) {
      const PageScales& S = B && j ? *B : A;
      const int i = B ? ia : ia + j;
      keep[j] = S.keep(i), flip[j] = S.flip(i);
    }
  }
  auto past_the_end = [&](float (&v)[RG][4 * NP]) {
#pragma unroll
    for (int i = 0; i < 4 * NP; i++) {
      const bool in = key0 + kPage * (i >> 2) + 4 * g + (i & 3) < len;
#pragma unroll
      for (int gi = 0; gi < RG; gi++) v[gi][i] = in ? v[gi][i] : -INFINITY;
    }
  };
  x.template softmax<NP>(s, k, lv, nv, key0 + NP * kPage > len, past_the_end, odd, keep, flip, pf);
}

// The part of a unit that a run holds: steps t0 .. t1 - 1, of them the nodes (step 0) and cache steps c0 .. c1 - 1 (the last)
struct TreePart {
  int hk, row0, rows;  // kv head, the unit's first row, and its sequence's rows
  int t0, t1, c0, c1;
  bool whole;
  __device__ __forceinline__ TreePart(const KvTreeArgs& a, const TreeUnit& u, int extra, int s, int s_end) {
    rows = u.nodes * a.G;
    const int tiles = (rows + a.tile - 1) / a.tile, unit = (s - u.first) / u.steps;
    hk = unit / tiles, row0 = (unit - hk * tiles) * a.tile;
    t0 = s - u.first - unit * u.steps, t1 = min(u.steps, t0 + s_end - s);
    c0 = max(t0 - 1 - extra, 0), c1 = max(t1 - 1 - extra, 0);
    whole = t0 == 0 && t1 == u.steps;
  }
};

// The result of 8 consecutive dims of a row, or its part of a split unit: a run has at most two of those, the end of one
// unit (slot 0) and the beginning of another (slot 1).
__device__ __forceinline__ void tree_store(const KvTreeArgs& a, const TreeUnit& u, const TreePart& p, int wg, int row,
                                           int d, float m, float l, const float (&v)[8]) {
  if (row >= p.rows) return;
  if (p.whole) {
    const int node = row / a.G, h = p.hk * a.G + row - node * a.G;
    half8_t r;
#pragma unroll
    for (int e = 0; e < 8; e++) r[e] = (_Float16)(l == 0.f ? 0.f : v[e] / l);
    *reinterpret_cast<half8_t*>(a.out + (((size_t)u.b * a.nodes + node) * a.Hq + h) * kHeadDim + d) = r;
  } else {
    const size_t at = ((size_t)wg * 2 + (p.t0 == 0)) * a.tile + row - p.row0;
    float4_t* po = reinterpret_cast<float4_t*>(a.part_o + at * kHeadDim + d);
    po[0] = float4_t{v[0], v[1], v[2], v[3]};
    po[1] = float4_t{v[4], v[5], v[6], v[7]};
    if (d == 0) a.part_ml[at * 2] = m, a.part_ml[at * 2 + 1] = l;
  }
}

// ---- split: up to 96 rows, pages per wave ---------------------------------------------------------------------------------

// Codes of (page, kv head) blocks in LDS, brought there without passing through registers
template <int BITS>
struct Staged {
  static constexpr int ROW = KvRegs<BITS>::ROW;
  static constexpr int BLOCK = kPage * ROW;         // bytes of a (page, kv head)'s keys, or values
  static constexpr int LOADS = BLOCK / 1024;        // of a block, 1 KB each

  // Where 16-byte piece `piece` of row `row` of a block lies in its stage: pieces are permuted so that neither the key
  // fragments (one piece of 16 rows) nor the value rows (all pieces of rows 4 apart) meet in a bank.  8 bits: rows in
  // order, piece p at place p ^ row % 8; 4 bits (rows of 4 pieces): row r at place 4 (r % 4) + r / 4, piece p at p ^ r % 4.
  static __device__ __forceinline__ int place(int row, int piece) {
    if constexpr (BITS == 8)
      return row * ROW + 16 * (piece ^ (row & 7));
    else
      return (4 * (row & 3) + (row >> 2)) * ROW + 16 * (piece ^ (row & 3));
  }
  // ... and the byte of a block that lane l's 16 bytes of the stage's first KB come from (later KBs: 1 KB on)
  static __device__ __forceinline__ int source(int l) {
    if constexpr (BITS == 8) {
      return (l >> 3) * ROW + 16 * ((l & 7) ^ (l >> 3));
    } else {
      const int row = 4 * (l >> 2 & 3) + (l >> 4);
      return row * ROW + 16 * ((l & 3) ^ (row & 3));
    }
  }
  static __device__ __forceinline__ void load_block(const uint8_t* block, uint8_t* to, int source) {
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(block), (short)0, BLOCK, 0x00020000);
    // The stage's address is hidden from alias analysis: where that does not tell the stage being filled from the one being
    // read, the compiler puts a wait for all loads in flight before the read; the waits here are explicit (16 sequences up to
    // 32k tokens, 4 bits: 5 nodes 83 and 70 us, 9 nodes 133 and 105, 16 nodes 177 and 154).
    uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)to;
    asm("" : "+s"(at));
#pragma unroll
    for (int i = 0; i < BLOCK / 1024; i++)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(uintptr_t)(at + 1024 * i), 16,
                                               source, 1024 * i, 0, 0);
  }
  // this lane's codes of a staged block: key row n, dims 32 g ..; values of rows 4 g + i, dims 8 n ..
  static __device__ __forceinline__ void read_keys(const uint8_t* st, int n, int g, KvRegs<BITS>& r) {
#pragma unroll
    for (int j = 0; j < BITS / 4; j++) {
      const kv_u32x4_t a = *reinterpret_cast<const kv_u32x4_t*>(st + place(n, BITS / 4 * g + j));
      r.k[4 * j] = a.x, r.k[4 * j + 1] = a.y, r.k[4 * j + 2] = a.z, r.k[4 * j + 3] = a.w;
    }
  }
  static __device__ __forceinline__ void read_values(const uint8_t* st, int n, int g, KvRegs<BITS>& r) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (BITS == 8) {
        const kv_u32x2_t a = *reinterpret_cast<const kv_u32x2_t*>(st + place(4 * g + i, n >> 1) + 8 * (n & 1));
        r.v[i] = a.x, r.v[4 + i] = a.y;
      } else {
        r.v[i] = *reinterpret_cast<const uint32_t*>(st + place(4 * g + i, n >> 2) + 4 * (n & 3));
      }
    }
  }
  // of values of rows 4 g + i: the 4 bytes that hold dims 8 n + 4 half .. (4 bits: all of dims 8 n ..)
  static __device__ __forceinline__ void read_half_values(const uint8_t* st, int n, int g, int half, uint32_t (&r)[4]) {
#pragma unroll
    for (int i = 0; i < 4; i++)
      r[i] = *reinterpret_cast<const uint32_t*>(BITS == 8 ? st + place(4 * g + i, n >> 1) + 8 * (n & 1) + 4 * half
                                                          : st + place(4 * g + i, n >> 2) + 4 * (n & 3));
  }
};

template <int BITS, int RG>
__global__ __launch_bounds__(64 * kSplitWaves, RG <= kPairedGroups ? 2 : 1) void kv_tree_split_kernel(const KvTreeArgs a) {
  using Rows = TreeRows<BITS, RG>;
  using St = Staged<BITS>;
  // A stage holds a step of a wave: the keys of two pages, then their values.  Two workgroups share a CU's LDS up to 32 rows.
  constexpr int W = kSplitWaves, STAGES = (RG <= kPairedGroups ? 2 : 4) * (BITS == 8 ? 1 : 2), AHEAD = STAGES - 1;
  // Queries stay in registers, but for 6 groups: with the accumulators they take more than a SIMD has, and are read from LDS
  // a fragment ahead (19 nodes, 7 sequences up to 20000 tokens: 86 and 74 us; 16 nodes, 5 groups: 65 us either way)
  constexpr bool QREG = RG <= 5;
  constexpr int ROUND = RG <= kPairedGroups ? 1 : 3;  // groups of rows merged at a time
  __shared__ union {
    uint8_t stage[W][STAGES][4 * St::BLOCK];
    struct {
      float o[ROUND][W][16][kHeadDim + 4];
      float ml[ROUND][W][16][2];
    } red;
  } sh;
  __shared__ typename Rows::Staging sh_q;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wg = blockIdx.x;
  const TreeRuns runs(a);
  if (wg >= runs.count) return;
  const int s_end = runs.start(wg + 1);
  for (int s = runs.start(wg); s < s_end;) {
    const TreeUnit u = tree_at_step<true>(a, runs, s);
    const TreePart p(a, u, runs.extra, s, s_end);
    // Lane i holds, for cache step cb + i, the wave's two pages
    const int* ptab = a.page_table + (size_t)u.b * a.max_pages;
    int cb = p.c0, ida, idb;
    PageScales A, B;
    auto page_of = [&](int lp) { return min(max(ptab[min(lp, u.pages - 1)], 0), a.num_pages - 1); };
    auto load_ids = [&] {
      const int lp = ((cb + lane) * W + w) * 2;
      ida = page_of(lp), idb = page_of(lp + 1);
    };
    const int source = St::source(lane);
    // the pages of cache step c into its stage
    auto issue = [&](int c) {
      if (c >= p.c1) return;
      const int i = c - cb;
      const size_t ba = (size_t)__builtin_amdgcn_readlane(ida, i) * a.Hkv + p.hk;
      const size_t bb = (size_t)__builtin_amdgcn_readlane(idb, i) * a.Hkv + p.hk;
      uint8_t* st = sh.stage[w][(c - p.c0) % STAGES];
      St::load_block(a.kc + ba * St::BLOCK, st, source);
      St::load_block(a.kc + bb * St::BLOCK, st + St::BLOCK, source);
      St::load_block(a.vc + ba * St::BLOCK, st + 2 * St::BLOCK, source);
      St::load_block(a.vc + bb * St::BLOCK, st + 3 * St::BLOCK, source);
    };
    // Page ids, queries and nodes first, then the scales and the first pages; the queries' and nodes' work runs while
    // those come in.
    Rows x;
    const bool nodes_here = p.t0 == 0 && 16 * w < u.nodes;
    typename Rows::Nodes nodes;
    if (p.c0 < p.c1) load_ids();
    Rows::stage_queries(a, u, p.hk, p.row0, w, lane, sh_q);
    if (nodes_here) nodes.load(a, u, p.hk, w, p.row0, n, g);
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
    issue_fence();
    if (p.c0 < p.c1) {
      A.load(a, ida, p.hk), B.load(a, idb, p.hk);
      issue_fence();
#pragma unroll
      for (int i = 0; i < AHEAD; i++) issue(p.c0 + i);
    }
    Rows::order_queries(w, lane, sh_q);
    lds_barrier();  // all rows of the queries are in
    x.read_queries(sh_q, n, g);
    x.start();
    if (nodes_here) x.process_nodes(a, u, p.hk, w, nodes, lane);
    if (p.c0 < p.c1) A.use(a.qk_scale), B.use(a.qk_scale);

    for (int c = p.c0; c < p.c1; c++) {
      if (c + AHEAD - cb >= 64 && c + AHEAD < p.c1) {  // the next 64 steps' pages, from step c on
        cb = c;
        load_ids();
        A.load(a, ida, p.hk), B.load(a, idb, p.hk);
        A.use(a.qk_scale), B.use(a.qk_scale);
      }
      issue(c + AHEAD);
      // step c is in (younger steps may be in flight), and nothing that reads it moves above the wait
      wait_loads<AHEAD, 4 * St::LOADS>(min(p.c1 - 1 - c, AHEAD));
      issue_fence();
      const uint8_t* st = sh.stage[w][(c - p.c0) % STAGES];
      KvRegs<BITS> ra, rb;
      St::read_keys(st, n, g, ra);
      St::read_keys(st + St::BLOCK, n, g, rb);
      float4_t sc[2][RG];
      half8_t pf[1][RG];
#pragma unroll
      for (int gi = 0; gi < RG; gi++) sc[0][gi] = sc[1][gi] = float4_t{0.f, 0.f, 0.f, 0.f};
      half8_t q[2][RG];  // QREG: not used
      auto read_q = [&](int f) {
#pragma unroll
        for (int gi = 0; gi < RG; gi++) q[f & 1][gi] = sh_q[gi][n][(4 * g + f) ^ n];
      };
      if constexpr (!QREG) read_q(0);
#pragma unroll
      for (int f = 0; f < 4; f++) {
        if constexpr (!QREG) {  // a fragment ahead, and not where it is used
          if (f < 3) read_q(f + 1);
          issue_fence();
        }
        const half8_t ka = ra.kfrag(f), kb = rb.kfrag(f);
#pragma unroll
        for (int gi = 0; gi < RG; gi++) {
          const half8_t qf = QREG ? x.q[gi][f] : q[f & 1][gi];
          sc[0][gi] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qf, sc[0][gi], 0, 0, 0);
          sc[1][gi] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb, qf, sc[1][gi], 0, 0, 0);
        }
      }
      if constexpr (!QREG) issue_fence();
      St::read_values(st + 2 * St::BLOCK, n, g, ra);
      St::read_values(st + 3 * St::BLOCK, n, g, rb);
      tree_softmax<BITS, RG, 2>(x, sc, A, &B, c - cb, (c * W + w) * 2 * kPage, u.len, g, pf);
      uint32_t ta[8], tb[8];
      ra.vtrans(ta);
      rb.vtrans(tb);
#pragma unroll
      for (int db = 0; db < 8; db++) {
        const half4_t xa = codes_f16(ta[db], (_Float16)Rows::kBias), xb = codes_f16(tb[db], (_Float16)Rows::kBias);
        const half8_t v = __builtin_shufflevector(xa, xb, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
        for (int gi = 0; gi < RG; gi++)
          x.o[gi][db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pf[0][gi], x.o[gi][db], 0, 0, 0);
      }
      issue_fence();  // the stage's reads are done before the next loads into it
    }

    // merge the waves, up to ROUND groups of rows at a time; lane (n, g) holds dims 32g + 8i + db of row n
    lds_barrier();  // the merge takes the stages' place
    const int tq = threadIdx.x >> 4, td = (threadIdx.x & 15) * 8;
#pragma unroll
    for (int base = 0; base < RG; base += ROUND) {
      if (base > 0) lds_barrier();  // (no wait for the stores of the rows before)
#pragma unroll
      for (int r = 0; r < ROUND; r++) {
        const int gi = base + r;
        if (gi >= RG) continue;
        const float lsum = sum_over_groups(x.l[gi]);
        float* mine = sh.red.o[r][w][n] + 32 * g;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int j = 0; j < 2; j++)
            *reinterpret_cast<float4_t*>(mine + 8 * i + 4 * j) =
                float4_t{x.o[gi][4 * j][i], x.o[gi][4 * j + 1][i], x.o[gi][4 * j + 2][i], x.o[gi][4 * j + 3][i]};
        if (g == 0) sh.red.ml[r][w][n][0] = x.reference(gi), sh.red.ml[r][w][n][1] = lsum;
      }
      lds_barrier();
#pragma unroll
      for (int r = 0; r < ROUND; r++) {
        const int gi = base + r;
        if (gi >= RG) continue;
        float mx = kTreeLow;
#pragma unroll
        for (int i = 0; i < W; i++) mx = fmaxf(mx, sh.red.ml[r][i][tq][0]);
        float sum = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < W; i++) {
          const float f = __builtin_amdgcn_exp2f(sh.red.ml[r][i][tq][0] - mx);
          sum += sh.red.ml[r][i][tq][1] * f;
          const float4_t* from = reinterpret_cast<const float4_t*>(sh.red.o[r][i][tq] + td);
          const float4_t y = from[0], z = from[1];
#pragma unroll
          for (int e = 0; e < 4; e++) acc[e] += y[e] * f, acc[4 + e] += z[e] * f;
        }
        tree_store(a, u, p, wg, p.row0 + 16 * gi + tq, td, mx, sum, acc);
      }
    }
    lds_barrier();
    s += p.t1 - p.t0;
  }
}

// ---- shared: rows per wave, pages decoded by all ---------------------------------------------------------------------------

// A step's 4 pages as MFMA fragments, 1 KB each, a lane's 16 bytes in lane order: keys [page][4], values [pair of pages][8]
struct SharedTile {
  half8_t k[kSharedPages][4][64];
  half8_t v[kSharedPages / 2][8][64];
};

template <int BITS>
struct SharedMem {
  // Steps whose codes are staged, one of them being decoded: blocks of random pages take 2 to 3 us to come, so 3 steps kept
  // the memory at 3.4 TB/s (8 bits) and 1.7 (4 bits)
  static constexpr int RING = BITS == 8 ? 6 : 10;
  SharedTile tile[2];
  uint8_t codes[RING][2 * kSharedPages][Staged<BITS>::BLOCK];  // keys of each page, then values
};

// A wave's share of decoding a step: waves 0-3 the keys of a page each, waves 4-7 half the dims of a pair's values (4 of
// every 8)
template <int BITS>
__device__ __forceinline__ void shared_decode(const uint8_t (*codes)[Staged<BITS>::BLOCK], SharedTile& to, int w, int lane) {
  constexpr _Float16 kBias = BITS == 8 ? (_Float16)1152.0f : (_Float16)1032.0f;
  asm volatile("" : "+v"(lane));  // the LDS addresses are made here, not kept in registers over the steps
  const int n = lane & 15, g = lane >> 4;
  if (w < 4) {
    KvRegs<BITS> r;
    Staged<BITS>::read_keys(codes[w], n, g, r);
#pragma unroll
    for (int f = 0; f < 4; f++) to.k[w][f][lane] = r.kfrag(f);
  } else {
    const int pair = (w - 4) >> 1, half = w & 1;
    // 4 dims 8n + 4 half + e of the 4 keys 4g .. 4g + 3 of either page, as biased bytes
    uint32_t t[2][4];
#pragma unroll
    for (int page = 0; page < 2; page++) {
      uint32_t b[4];
      Staged<BITS>::read_half_values(codes[4 + 2 * pair + page], n, g, half, b);
      if constexpr (BITS == 8) {
#pragma unroll
        for (int i = 0; i < 4; i++) b[i] ^= 0x80808080u;
        transpose4x4(b, t[page]);
      } else {
        uint32_t two[4];  // two[j], j < 2: byte j of the 4 rows, two dims each
#pragma unroll
        for (int i = 0; i < 4; i++) b[i] >>= 16 * half;
        transpose4x4(b, two);
#pragma unroll
        for (int j = 0; j < 2; j++) {
          t[page][2 * j] = (two[j] & 0x0F0F0F0Fu) ^ 0x08080808u;
          t[page][2 * j + 1] = ((two[j] >> 4) & 0x0F0F0F0Fu) ^ 0x08080808u;
        }
      }
    }
    half8_t(*out)[64] = to.v[pair] + 4 * half;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const half4_t xa = codes_f16(t[0][e], kBias), xb = codes_f16(t[1][e], kBias);
      out[e][lane] = __builtin_shufflevector(xa, xb, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
}

// A part with GN groups of rows in this wave (0: it only decodes)
template <int BITS, int GN>
__device__ __forceinline__ void shared_part(const KvTreeArgs& a, SharedMem<BITS>& sh, const TreeUnit& u,
                                            const TreePart& p, int row0, int w, int lane, int wg) {
  constexpr int PAGES = kSharedPages, BATCH = 64 / PAGES;  // steps whose pages the lanes hold
  constexpr int RG = GN > 0 ? GN : 1;
  using Rows = TreeRows<BITS, RG>;
  using St = Staged<BITS>;
  constexpr int RING = SharedMem<BITS>::RING;
  const int n = lane & 15, g = lane >> 4;
  const int* ptab = a.page_table + (size_t)u.b * a.max_pages;
  // Lane i holds page PAGES cb + i of the sequence (id0, with what softmax takes of its scales) and page
  // PAGES (cb + BATCH) + i (id1): the next batch's ids and scales are loaded one batch and half a batch ahead.
  int cb = p.c0, id0 = 0, id1 = 0;
  PageScales S, next;
  auto load_ids = [&](int c) {
    int i = lane;
    asm volatile("" : "+v"(i));  // addresses of the rare loads are made where they are used, not kept in registers
    return min(max(ptab[min(PAGES * c + i, u.pages - 1)], 0), a.num_pages - 1);
  };
  auto block_of = [&](int c, int j) {
    const int i = PAGES * (c - cb) + j;
    return (size_t)__builtin_amdgcn_readlane(i < 64 ? id0 : id1, i & 63) * a.Hkv + p.hk;
  };
  // this wave's block of cache step c: page w % 4, keys or values
  const int source = St::source(lane);
  const uint8_t* cache = w < 4 ? a.kc : a.vc;
  auto issue = [&](int c) {
    if (c < p.c1) St::load_block(cache + block_of(c, w & 3) * St::BLOCK, sh.codes[(unsigned)(c - p.c0) % RING][w], source);
  };

  Rows x;
  const bool pages = p.c0 < p.c1;
  if (pages) id0 = load_ids(cb), id1 = load_ids(cb + BATCH);
  if constexpr (GN > 0) x.load_queries(a, u, p.hk, row0, n, g);
  issue_fence();
  if (pages) {
#pragma unroll
    for (int i = 0; i < RING; i++) issue(p.c0 + i);
    S.load(a, id0, p.hk);
  }
  issue_fence();
  if constexpr (GN > 0) {
    x.start();
    if (p.t0 == 0) {
#pragma unroll 1
      for (int t = 0; 16 * t < u.nodes; t++) {
        typename Rows::Nodes nodes;
        nodes.load(a, u, p.hk, t, row0, n, g);
        x.process_nodes(a, u, p.hk, t, nodes, lane);
      }
    }
  }
  if (pages) S.use(a.qk_scale);  // (its loads are younger than the first steps': those are in)
  __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
  lds_barrier();
  if (pages) shared_decode<BITS>(sh.codes[0], sh.tile[0], w, lane);
  lds_barrier();
  for (int c = p.c0; c < p.c1;) {
#pragma unroll
    for (int j = 0; j < 2; j++) {
      if (c < p.c1) {  // tile j holds cache step c; the codes of step c + 1 are in, those of the next ones come
        issue(c + RING);
        if constexpr (GN > 0) {
          // Few rows leave registers for all four pages at once, and for reading further ahead: their products are short.
          // A pass's fragments in the order of their use, keys (f, page), then values (page pair, dims), are read AHEAD before
          // the products that take them and pinned by fences: left to itself the compiler reads each right before its use.
          constexpr int NP = RG == 1 ? 4 : 2, PER = 8 * NP, AHEAD = RG == 1 ? 8 : RG == 2 ? 3 : 2, FR = AHEAD + 1;
          const SharedTile& tile = sh.tile[j];
          half8_t fr[FR];
          auto read = [&](int k) {  // fragment k % PER of pass k / PER
            const int page0 = NP * (k / PER), f = k % PER;
            return f < 4 * NP ? tile.k[page0 + f % NP][f / NP][lane]
                              : tile.v[page0 / 2 + (f - 4 * NP) / 8][f % 8][lane];
          };
#pragma unroll
          for (int k = 0; k < AHEAD; k++) fr[k] = read(k);
#pragma unroll
          for (int pass = 0; pass < PAGES / NP; pass++) {
            float4_t sc[NP][RG];
            half8_t pf[NP / 2][RG];
#pragma unroll
            for (int i = 0; i < NP; i++)
#pragma unroll
              for (int gi = 0; gi < RG; gi++) sc[i][gi] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int f = 0; f < PER; f++) {
              // The wave of a SIMD that is at its products goes first, the other's softmax fills in (40 sequences up to 2000
              // tokens, 64 nodes: 136 -> 132 us; 24 nodes 75 -> 74; with two groups it costs 1 %)
              if (RG != 2 && (f == 0 || f == 4 * NP)) __builtin_amdgcn_s_setprio(1);
              if (RG != 2 && (f == 4 * NP - 1 || f == PER - 1)) __builtin_amdgcn_s_setprio(0);
              const int k = PER * pass + f;
              if (k + AHEAD < 8 * PAGES) fr[(k + AHEAD) % FR] = read(k + AHEAD);
              issue_fence();
#pragma unroll
              for (int gi = 0; gi < RG; gi++) {
                if (f < 4 * NP)
                  sc[f % NP][gi] =
                      __builtin_amdgcn_mfma_f32_16x16x32_f16(fr[k % FR], x.q[gi][f / NP], sc[f % NP][gi], 0, 0, 0);
                else
                  x.o[gi][f % 8] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fr[k % FR], pf[(f - 4 * NP) / 8][gi],
                                                                          x.o[gi][f % 8], 0, 0, 0);
              }
              if (f == 4 * NP - 1)
                tree_softmax<BITS, RG, NP>(x, sc, S, nullptr, PAGES * (c - cb) + NP * pass,
                                           (PAGES * c + NP * pass) * kPage, u.len, g, pf);
            }
          }
        }
        if (c + 1 < p.c1)  // into the tile that step c - 1 was read from
          shared_decode<BITS>(sh.codes[(unsigned)(c + 1 - p.c0) % RING], sh.tile[j ^ 1], w, lane);
        c++;
        if (c == cb + BATCH / 2) {
          next.load(a, id1, p.hk);
        } else if (c == cb + BATCH) {
          cb = c;
          id0 = id1;
          S.kraw = next.kraw, S.vraw = next.vraw;
          S.use(a.qk_scale);
          id1 = load_ids(cb + BATCH);
        }
        wait_loads<RING - 2, St::LOADS>(min(p.c1 - 2 - c, RING - 2));  // the codes of step c + 1 are in before the barrier
        lds_barrier();
      }
    }
  }
  if constexpr (GN > 0) {
#pragma unroll
    for (int gi = 0; gi < RG; gi++) {
      const float l = sum_over_groups(x.l[gi]);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        float v[8];
#pragma unroll
        for (int db = 0; db < 8; db++) v[db] = x.o[gi][db][i];
        tree_store(a, u, p, wg, row0 + 16 * gi + n, 32 * g + 8 * i, x.reference(gi), l, v);
      }
    }
  }
}

template <int BITS, int RG>
__global__ __launch_bounds__(64 * kSharedSlots, 2) void kv_tree_shared_kernel(const KvTreeArgs a) {
  __shared__ SharedMem<BITS> sh;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wg = blockIdx.x;
  const TreeRuns runs(a);
  if (wg >= runs.count) return;
  const int s_end = runs.start(wg + 1);
  for (int s = runs.start(wg); s < s_end;) {
    const TreeUnit u = tree_at_step<false>(a, runs, s);
    const TreePart p(a, u, runs.extra, s, s_end);
    // The unit's groups of rows, dealt evenly (wave w and wave w + 4 share a SIMD), but RG - 1 to a wave at least while they
    // last: a wave has code for RG and RG - 1 groups, and where a sequence has fewer live nodes than the launch has room for,
    // the group that a share of one would be rounded up by is the next wave's.  (Code for RG - 2 too: 35 spilled registers
    // instead of 22.)  The last share may be short of one, past the unit's rows.
    constexpr int LEAST = RG > 1 ? RG - 1 : 1;
    const int groups = (min(p.rows - p.row0, a.tile) + 15) / 16;
    const int each = groups / kSharedSlots, more = groups - each * kSharedSlots;
    const bool even = each >= LEAST;
    const int first = even ? w * each + min(w, more) : min(w * LEAST, groups);
    const int mine = even ? each + (w < more) : min(groups - first, LEAST), row0 = p.row0 + 16 * first;
    if (mine == RG)
      shared_part<BITS, RG>(a, sh, u, p, row0, w, lane, wg);
    else if (RG > 1 && mine > 0)
      shared_part<BITS, RG - 1>(a, sh, u, p, row0, w, lane, wg);
    else
      shared_part<BITS, 0>(a, sh, u, p, row0, w, lane, wg);
    s += p.t1 - p.t0;
  }
}

// Joins the parts of split units: one workgroup of 4 waves per (16 / SPLIT rows, unit of the sequence, sequence), SPLIT waves
// share the parts of 4 rows.  One wave per 4 rows has fewer workgroups derive the split; few rows have many parts each (one
// sequence of 8000 tokens, 1 node: 63; both launches 21.3 us with SPLIT = 1, 15.0 with 4; 16 nodes of 16 sequences up to 4k,
// this launch: 6.2 and 9.2 us).
constexpr int kTreeMergeWaves = 4;
template <int SPLIT>
__global__ __launch_bounds__(64 * kTreeMergeWaves) void kv_tree_merge_kernel(const KvTreeArgs a) {
  __shared__ float sh_o[kTreeMergeWaves][4][kHeadDim];
  __shared__ float sh_ml[kTreeMergeWaves][4][2];
  const TreeRuns runs(a);
  const int b = blockIdx.z, unit = blockIdx.y;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const TreeUnit u = tree_find<true>(a, runs, [&](int at, int) { return at == b; });
  const int rows = u.nodes * a.G, tiles = (rows + a.tile - 1) / a.tile;
  if (unit >= a.Hkv * tiles) return;
  const int first = w % SPLIT, group = w / SPLIT;  // of the parts, and the wave's 4 rows
  const int hk = unit / tiles, in_tile = 16 / SPLIT * blockIdx.x + 4 * group + (lane >> 4), row = (unit - hk * tiles) * a.tile + in_tile;
  const int td = (lane & 15) * 8;
  const int s0 = u.first + unit * u.steps, w0 = runs.of(s0), w1 = runs.of(s0 + u.steps - 1);
  if (w0 == w1) return;
  float mx = kTreeLow, sum = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  auto join = [&](float m, float l, const float4_t& x, const float4_t& y) {
    const float mn = fmaxf(mx, m);
    const float fa = __builtin_amdgcn_exp2f(mx - mn), fw = __builtin_amdgcn_exp2f(m - mn);
    sum = sum * fa + l * fw;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      acc[e] = acc[e] * fa + x[e] * fw;
      acc[4 + e] = acc[4 + e] * fa + y[e] * fw;
    }
    mx = mn;
  };
#pragma unroll 4
  for (int part = w0 + first; part <= w1; part += SPLIT) {
    const size_t at = ((size_t)part * 2 + (part == w0)) * a.tile + in_tile;
    const float4_t* po = reinterpret_cast<const float4_t*>(a.part_o + at * kHeadDim + td);
    join(a.part_ml[at * 2], a.part_ml[at * 2 + 1], po[0], po[1]);
  }
  if constexpr (SPLIT > 1) {
    if (first > 0) {
      float4_t* o = reinterpret_cast<float4_t*>(sh_o[w][lane >> 4] + td);
      o[0] = float4_t{acc[0], acc[1], acc[2], acc[3]}, o[1] = float4_t{acc[4], acc[5], acc[6], acc[7]};
      if (td == 0) sh_ml[w][lane >> 4][0] = mx, sh_ml[w][lane >> 4][1] = sum;
    }
    __syncthreads();
    if (first > 0) return;
#pragma unroll
    for (int i = 1; i < SPLIT; i++) {
      const float4_t* o = reinterpret_cast<const float4_t*>(sh_o[w + i][lane >> 4] + td);
      join(sh_ml[w + i][lane >> 4][0], sh_ml[w + i][lane >> 4][1], o[0], o[1]);
    }
  }
  if (row >= rows) return;
  const int node = row / a.G, h = hk * a.G + row - node * a.G;
  half8_t r;
#pragma unroll
  for (int e = 0; e < 8; e++) r[e] = (_Float16)(sum == 0.f ? 0.f : acc[e] / sum);
  *reinterpret_cast<half8_t*>(a.out + (((size_t)b * a.nodes + node) * a.Hq + h) * kHeadDim + td) = r;
}

// The kernel's form (rg: most groups of 16 rows per wave), rows of a unit, pages of a step, and the most workgroups of the
// launch (a run each)
struct TreePlan {
  bool shared;
  int rg, tile, tiles, step, wgs;
  long long steps;  // of a batch that fills its tables
};
static TreePlan tree_plan(int batch, int nodes, int num_q_heads, int num_kv_heads, int max_pages) {
  const int groups = (nodes * (num_q_heads / num_kv_heads) + 15) / 16;
  TreePlan p;
  p.shared = groups > kSplitGroups;
  const int most = p.shared ? kSharedSlots * kSharedGroups : kSplitGroups;
  p.tiles = (groups + most - 1) / most;
  const int per_tile = (groups + p.tiles - 1) / p.tiles;
  p.rg = p.shared ? (per_tile + kSharedSlots - 1) / kSharedSlots : per_tile;
  p.tile = 16 * per_tile;
  p.step = p.shared ? kSharedPages : 2 * kSplitWaves;
  p.steps = (long long)batch * num_kv_heads * p.tiles * ((max_pages + p.step - 1) / p.step + 1 + kTreeExtra);
  p.wgs = (int)std::min<long long>(!p.shared && p.rg <= kPairedGroups ? 512 : 256, p.steps);
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
                     sm_scale * 1.4426950408889634f, p.wgs, p.tile, p.step, part_o, part_o + slots * kHeadDim,
                     static_cast<_Float16*>(out)};
  hipStream_t st = as_stream(stream);
  using Kern = decltype(&kv_tree_split_kernel<8, 1>);
#define EXL3_TREE_SPLIT(RG) {kv_tree_split_kernel<4, RG>, kv_tree_split_kernel<8, RG>}
  static const Kern split[kSplitGroups][2] = {EXL3_TREE_SPLIT(1), EXL3_TREE_SPLIT(2), EXL3_TREE_SPLIT(3),
                                              EXL3_TREE_SPLIT(4), EXL3_TREE_SPLIT(5), EXL3_TREE_SPLIT(6)};
#undef EXL3_TREE_SPLIT
  static const Kern shared[kSharedGroups][2] = {{kv_tree_shared_kernel<4, 1>, kv_tree_shared_kernel<8, 1>},
                                                {kv_tree_shared_kernel<4, 2>, kv_tree_shared_kernel<8, 2>},
                                                {kv_tree_shared_kernel<4, 3>, kv_tree_shared_kernel<8, 3>}};
  (p.shared ? shared[p.rg - 1] : split[p.rg - 1])[bits == 8]<<<p.wgs, 64 * (p.shared ? kSharedSlots : kSplitWaves), 0, st>>>(a);
  EXL3_CHECK_LAUNCH();
  const bool few = (long long)batch * nodes * num_q_heads <= 4096;
  (few ? kv_tree_merge_kernel<4> : kv_tree_merge_kernel<1>)<<<dim3(few ? p.tile / 4 : p.tile / 16, num_kv_heads * p.tiles,
                                                                  batch), 64 * kTreeMergeWaves, 0, st>>>(a);
  EXL3_CHECK_LAUNCH();
  return EXL3_OK;
}
