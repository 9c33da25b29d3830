// Verification of drafted tokens against the target's probabilities, from given random numbers (gfx950).
//
// Node 0 of a sequence is its last committed token, nodes 1 .. n-1 are drafts (parents come before children); row i of
// the target is its distribution after node i, u_i a uniform number.
//   Chain with the draft's distributions q (node i drawn from q after node i-1): node i is accepted while p(t_i) > 0 and
//     u_i q(t_i) < p(t_i); at the first refusal the next token comes from w = max(p - q, 0), after the last node from p.
//   Tree (or chain) of candidates: at the current node its children in index order, m = 1: child j is accepted when
//     p(t_j) > 0 and u_j m < p(t_j); a refused one takes m -= p(t_j) and its token is struck from p (p = 0 for a brother
//     with the same token).  The next token comes from p without the struck tokens.
//   Next token: the smallest v with w(0) + .. + w(v) > u_0 * (the sum of w).
// Given its drafts, either rule leaves every emitted token distributed as the target's.  Products and sums are in 64 bits.
// The product of two floats is exact there, so a chain's decisions are; m is rounded once per refused child.  A running sum
// over 10^5 terms goes through some tens of additions (16 a lane, a scan over the wave, the parts), each off by at most
// 2^-53 of the row's total.  So another order of summation picks another token only where u * total lies within some 10^-14
// of the total from the edge between the two; the floats u themselves are 6 * 10^-8 apart.
//
// The walk reads one probability per node (lane i: node i) and is wave-uniform afterwards.  Only the row that the next
// token comes from is read whole.  verify_mass_kernel: (chunks of the row, sequences) workgroups, each repeats the walk
// and sums its chunk; verify_pick_kernel: one workgroup per sequence scans the chunks' sums, then the chunk that the
// threshold falls in.  Two launches instead of one with a counter: nothing has to be zero beforehand and nobody waits.
// Bound by latency at few sequences (gathers behind gathers), by memory at many.
#include <algorithm>

#include "exl3_api.hpp"
#include "exl3_device.hpp"

namespace exl3 {

typedef float verify_f4_t __attribute__((ext_vector_type(4), aligned(4)));  // rows start at any multiple of 4 bytes

constexpr int kVerifyNodes = 64;     // a node per lane
constexpr int kVerifyPart = 1024;    // consecutive elements that one wave sums: 16 a lane
constexpr int kMassWaves = 4;
constexpr int kMassThreads = 64 * kMassWaves;

struct VerifyEnd {
  unsigned long long struck;  // refused children of the last accepted node
  int node, count;            // the last accepted node; accepted nodes with the root (0: no sequence)
  int residual;               // w = max(p - q, 0)
  int pad;
};

struct VerifyArgs {
  const float *p, *q;
  const int *tokens, *parents;
  const float* uniform;
  const int* num_nodes;
  int nodes, vocab, parts;
  int *accepted, *counts, *out_tokens;
  double* mass;      // [batch][parts][2]: the part's sum of w, and of p
  VerifyEnd* end;    // [batch]
};

struct VerifyWalk {
  VerifyEnd end;
  unsigned long long path;
  int token;  // the lane's node's
};

// One wave; lane i holds node i.
__device__ __forceinline__ VerifyWalk verify_walk(const VerifyArgs& a, int b) {
  const int lane = threadIdx.x & 63;
  const int n = a.num_nodes ? min(max(a.num_nodes[b], 0), a.nodes) : a.nodes;
  const size_t at = (size_t)b * a.nodes + min(lane, a.nodes - 1);
  const int token = a.tokens[at];
  const int parent = a.parents ? a.parents[at] : lane - 1;
  const float u = a.uniform[at];
  const bool node = lane >= 1 && lane < n && parent >= 0 && parent < lane;
  float pt = 0.f, qt = 0.f;
  if (node && token >= 0 && token < a.vocab) {
    const size_t i = ((size_t)b * a.nodes + parent) * a.vocab + token;
    pt = a.p[i];
    pt = pt < __builtin_inff() ? pt : 0.f;
    if (a.q) qt = a.q[i];
  }
  VerifyWalk w;
  w.token = token;
  w.end = VerifyEnd{0, 0, n > 0, 0, 0};
  w.path = n > 0;
  if (a.q) {
    const unsigned long long fits = __builtin_amdgcn_ballot_w64(node && pt > 0.f && (double)u * qt < (double)pt);
    const int taken = __builtin_ctzll(~(fits >> 1));  // at most 63: the shift leaves bit 63 clear
    if (n > 0) {
      w.end.node = taken;
      w.end.count = taken + 1;
      w.end.residual = taken + 1 < n;
      w.path = taken == 63 ? ~0ull : (2ull << taken) - 1;
    }
    return w;
  }
  double left = 1.0;
  unsigned long long children = __builtin_amdgcn_ballot_w64(node && parent == 0);
  while (children) {  // every child once; an accepted one has a larger index than its parent
    const int i = __builtin_ctzll(children);
    children &= children - 1;
    const int ti = __builtin_amdgcn_readlane(token, i);
    const bool again = (__builtin_amdgcn_ballot_w64(token == ti) & w.end.struck) != 0;
    const float pi = again ? 0.f : __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, pt), i));
    const float ui = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, u), i));
    if (pi > 0.f && (double)ui * left < (double)pi) {
      w.end.node = i;
      w.end.count++;
      w.path |= 1ull << i;
      w.end.struck = 0;
      left = 1.0;
      children = __builtin_amdgcn_ballot_w64(node && parent == i);
    } else {
      left -= pi > 0.f ? (double)pi : 0.0;
      w.end.struck |= 1ull << i;
    }
  }
  return w;
}

// The struck tokens in [first, last), compacted into list by one wave; their number
__device__ __forceinline__ int struck_in(unsigned long long struck, int token, int first, int last, int* list) {
  const int lane = threadIdx.x & 63;
  const bool in = (struck >> lane & 1) && token >= first && token < last;
  const unsigned long long mask = __builtin_amdgcn_ballot_w64(in);
  if (in) list[__builtin_popcountll(mask & ((1ull << lane) - 1))] = token;
  return __builtin_popcountll(mask);
}

// A lane's 16 elements of a part of the row: v + STEP j + e (j, e < 4), 0 past `last`.  All loads are issued before
// any of them is used; weights that are no finite positive number are 0.
template <int STEP>
struct VerifyRow {
  float p[16], q[16];

  __device__ __forceinline__ void load(const float* prow, const float* qrow, int v, bool whole, int last) {
    get(prow, v, whole, last, p);
    if (qrow) get(qrow, v, whole, last, q);
#pragma unroll
    for (int i = 0; i < 16; i++) {
      p[i] = p[i] > 0.f && p[i] < __builtin_inff() ? p[i] : 0.f;
      q[i] = qrow && q[i] > 0.f ? q[i] : 0.f;
    }
  }
  __device__ __forceinline__ void strike(int v, int n, const int* list) {
    for (int i = 0; i < n; i++) {
      const int t = list[i] - v;
#pragma unroll
      for (int j = 0; j < 16; j++) p[j] = t == STEP * (j / 4) + (j & 3) ? 0.f : p[j];
    }
  }
  __device__ __forceinline__ double rest(int i) const {
    const double d = (double)p[i] - (double)q[i];
    return d > 0.0 ? d : 0.0;
  }

 private:
  __device__ __forceinline__ static void get(const float* row, int v, bool whole, int last, float x[16]) {
    if (whole) {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const verify_f4_t r = *reinterpret_cast<const verify_f4_t*>(row + v + STEP * j);
#pragma unroll
        for (int e = 0; e < 4; e++) x[4 * j + e] = r[e];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; j++) {
        const int i = v + STEP * (j / 4) + (j & 3);
        x[j] = i < last ? row[i] : 0.f;
      }
    }
  }
};

template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_f64(double v) {  // 0 where no lane feeds
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)(unsigned)u, CTRL, ROWS, 0xF, ROWS == 0xF);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(unsigned)(u >> 32), CTRL, ROWS, 0xF, ROWS == 0xF);
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ double wave_scan_f64(double v) {  // inclusive
  v += dpp_f64<0x111, 0xF>(v);  // row_shr:1, 2, 4, 8: inside each row of 16
  v += dpp_f64<0x112, 0xF>(v);
  v += dpp_f64<0x114, 0xF>(v);
  v += dpp_f64<0x118, 0xF>(v);
  v += dpp_f64<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
  v += dpp_f64<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ double lane_f64(double v, int from) {  // from: wave-uniform
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
  const unsigned lo = __builtin_amdgcn_readlane((int)(unsigned)u, from);
  const unsigned hi = __builtin_amdgcn_readlane((int)(unsigned)(u >> 32), from);
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}

__global__ __launch_bounds__(kMassThreads) void verify_mass_kernel(const VerifyArgs a, int each) {
  __shared__ VerifyEnd end;
  __shared__ int list[kVerifyNodes], nlist;
  const int b = blockIdx.y, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part0 = blockIdx.x * kMassWaves * each, part1 = min(part0 + kMassWaves * each, a.parts);
  if (wave == 0) {
    const VerifyWalk w = verify_walk(a, b);
    const int n = struck_in(w.end.struck, w.token, part0 * kVerifyPart, min(part1 * kVerifyPart, a.vocab), list);
    if (lane == 0) end = w.end, nlist = n;
    if (blockIdx.x == 0) {
      const size_t at = (size_t)b * a.nodes;
      if (w.path >> lane & 1) {
        const int place = __builtin_popcountll(w.path & ((1ull << lane) - 1));
        a.accepted[at + place] = lane;
        if (place > 0) a.out_tokens[at + place - 1] = w.token;
      }
      if (lane >= w.end.count && lane < a.nodes) {
        a.accepted[at + lane] = -1;
        a.out_tokens[at + lane] = -1;
      }
      if (lane == 0) {
        a.counts[b] = w.end.count;
        a.end[b] = w.end;
      }
    }
  }
  __syncthreads();
  const VerifyEnd e = end;
  if (e.count == 0) return;
  const size_t row = ((size_t)b * a.nodes + e.node) * a.vocab;
  const float *p = a.p + row, *q = e.residual ? a.q + row : nullptr;
  for (int part = part0 + wave; part < part1; part += kMassWaves) {
    const int first = part * kVerifyPart, last = min(first + kVerifyPart, a.vocab);
    VerifyRow<256> r;
    r.load(p, q, first + 4 * lane, first + kVerifyPart <= last, last);
    double sw = 0.0, sp = 0.0;
#pragma unroll
    for (int i = 0; i < 16; i++) sp += (double)r.p[i];
    if (q) {
#pragma unroll
      for (int i = 0; i < 16; i++) sw += r.rest(i);
    } else if (nlist) {
      r.strike(first + 4 * lane, nlist, list);
#pragma unroll
      for (int i = 0; i < 16; i++) sw += (double)r.p[i];
    } else {
      sw = sp;
    }
    sw = wave_scan_f64(sw), sp = wave_scan_f64(sp);
    if (lane == 63) {
      double* to = a.mass + ((size_t)b * a.parts + part) * 2;
      to[0] = sw, to[1] = sp;
    }
  }
}

// One wave per sequence: from the parts' sums, a run of parts per lane, to a run, to its part, to its element
__global__ __launch_bounds__(64) void verify_pick_kernel(const VerifyArgs a) {
  __shared__ int list[kVerifyNodes];
  const int b = blockIdx.x, lane = threadIdx.x;
  const VerifyEnd e = a.end[b];
  const float u = a.uniform[(size_t)b * a.nodes];
  const int token = a.tokens[(size_t)b * a.nodes + min(lane, a.nodes - 1)];
  if (e.count == 0) return;
  const double* mass = a.mass + (size_t)b * a.parts * 2;
  const int run = (a.parts + 63) / 64, run0 = lane * run, run1 = min(run0 + run, a.parts);
  double mw = 0.0, mp = 0.0;
  for (int i = run0; i < run1; i++) mw += mass[2 * i], mp += mass[2 * i + 1];
  double scan = wave_scan_f64(mw);
  const bool plain = !(lane_f64(scan, 63) > 0.0);  // nothing left of w: the target's row as it is
  double mine = plain ? mp : mw;
  if (plain) scan = wave_scan_f64(mp);
  const double total = lane_f64(scan, 63);
  int next = -1;
  if (total > 0.0) {
    const double bar = (u > 0.f ? (double)fminf(u, 1.f) : 0.0) * total;
    // where the scan first passes the threshold; rounding may leave that to nobody, then it is the last with any weight
    auto passes = [&](double scan, double mine) {
      const unsigned long long over = __builtin_amdgcn_ballot_w64(scan > bar && mine > 0.0);
      return over ? __builtin_ctzll(over) : 63 - __builtin_clzll(__builtin_amdgcn_ballot_w64(mine > 0.0) | 1);
    };
    int at = passes(scan, mine);
    double base = at > 0 ? lane_f64(scan, at - 1) : 0.0;
    const int from = at * run, to = min(from + run, a.parts);
    int part = from;
    for (int i0 = from; i0 < to; i0 += 64) {
      const int i = i0 + lane;
      mine = i < to ? mass[2 * i + plain] : 0.0;
      if (!__builtin_amdgcn_ballot_w64(mine > 0.0)) continue;
      scan = base + wave_scan_f64(mine);
      const int l = passes(scan, mine);
      part = i0 + l;
      if (lane_f64(scan, l) > bar || i0 + 64 >= to) {
        base = l > 0 ? lane_f64(scan, l - 1) : base;
        break;
      }
      base = lane_f64(scan, 63);
    }
    const int first = part * kVerifyPart, last = min(first + kVerifyPart, a.vocab);
    const int n = struck_in(plain ? 0 : e.struck, token, first, last, list);
    __syncthreads();
    const size_t row = ((size_t)b * a.nodes + e.node) * a.vocab;
    const float *p = a.p + row, *q = e.residual && !plain ? a.q + row : nullptr;
    const int v = first + 16 * lane;
    VerifyRow<4> r;
    r.load(p, q, v, first + kVerifyPart <= last, last);
    r.strike(v, n, list);
    double w[16], sum = 0.0;
#pragma unroll
    for (int i = 0; i < 16; i++) w[i] = r.rest(i), sum += w[i];
    scan = base + wave_scan_f64(sum);
    double c = scan - sum;
    int found = -1, positive = -1;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      c += w[i];
      if (w[i] > 0.0) {
        positive = v + i;
        if (c > bar && found < 0) found = v + i;
      }
    }
    const unsigned long long hit = __builtin_amdgcn_ballot_w64(found >= 0);
    const unsigned long long any = __builtin_amdgcn_ballot_w64(positive >= 0);
    if (hit)
      next = __builtin_amdgcn_readlane(found, __builtin_ctzll(hit));
    else if (any)
      next = __builtin_amdgcn_readlane(positive, 63 - __builtin_clzll(any));
  }
  if (lane == 0) a.out_tokens[(size_t)b * a.nodes + e.count - 1] = next;
}

static int verify_parts(int vocab) { return (vocab + kVerifyPart - 1) / kVerifyPart; }
static size_t verify_bytes(int batch, int vocab) {
  return (size_t)batch * (verify_parts(vocab) * 2 * sizeof(double) + sizeof(VerifyEnd));
}

}  // namespace exl3

using namespace exl3;

extern "C" size_t exl3_verify_workspace_bytes(int batch, int vocab) {
  if (batch <= 0 || vocab <= 0 || vocab > (1 << 28)) return 0;
  return verify_bytes(batch, vocab);
}

extern "C" int exl3_verify_drafts(const float* target_probs, const float* draft_probs, const int* tokens,
                                  const int* parents, const float* uniform, const int* num_nodes, int batch, int nodes,
                                  int vocab, int* accepted_nodes, int* counts, int* out_tokens, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  EXL3_CHECK_ARG(batch >= 0 && batch <= 65535 && nodes >= 1 && nodes <= kVerifyNodes && vocab >= 1 && vocab <= (1 << 28),
                 "exl3_verify_drafts: batch = %d, nodes = %d (1 to 64), vocab = %d", batch, nodes, vocab);
  EXL3_CHECK_ARG(!(draft_probs && parents),
                 "exl3_verify_drafts: the draft's probabilities come with a chain (parents = NULL)");
  if (batch == 0) return EXL3_OK;
  EXL3_CHECK_ARG(target_probs && tokens && uniform && accepted_nodes && counts && out_tokens,
                 "exl3_verify_drafts: null pointer");
  const size_t need = verify_bytes(batch, vocab);
  EXL3_CHECK_ARG(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 7) == 0,
                 "exl3_verify_drafts: workspace %zu bytes, need %zu (8-byte aligned)", workspace_bytes, need);
  double* mass = static_cast<double*>(workspace);
  const int parts = verify_parts(vocab);
  const VerifyArgs a{target_probs, draft_probs, tokens, parents, uniform, num_nodes, nodes, vocab, parts,
                     accepted_nodes, counts, out_tokens, mass,
                     reinterpret_cast<VerifyEnd*>(mass + (size_t)batch * parts * 2)};
  // parts per wave: at 64 rows of 131072 the sums take 9.7 / 8.8 / 9.6 us at 1 / 2 / 4, at one row of 32003
  // 4.2 / 5.0 / 6.9 us
  const int each = (long long)batch * parts > 4096 ? 2 : 1;
  verify_mass_kernel<<<dim3((parts + kMassWaves * each - 1) / (kMassWaves * each), batch), kMassThreads, 0,
                       as_stream(stream)>>>(a, each);
  EXL3_CHECK_LAUNCH();
  verify_pick_kernel<<<batch, 64, 0, as_stream(stream)>>>(a);
  EXL3_CHECK_LAUNCH();
  return EXL3_OK;
}
