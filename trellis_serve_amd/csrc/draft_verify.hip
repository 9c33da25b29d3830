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
// Given its drafts, either rule leaves every emitted token distributed as the target's.  Products and sums are in 64 bits:
// the products of two floats are exact there, and the running sums of 10^5 terms are off by 10^-12 of a term at most, so
// decisions do not depend on the order of the sums.
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
constexpr int kVerifyChunks = 64;    // most chunks of a row: a lane each in the pick
constexpr int kMassThreads = 256;
constexpr int kPickThreads = 1024;
constexpr int kVerifyBlock = 4 * kPickThreads;  // chunk lengths are multiples of it

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
  int nodes, vocab, chunks, chunk_len;
  int *accepted, *counts, *out_tokens;
  double* mass;      // [batch][chunks][2]: the chunk's sum of w, and of p
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

// p as a weight: finite positive values, anything else is 0
__device__ __forceinline__ double verify_weight(float p) { return p > 0.f && p < __builtin_inff() ? (double)p : 0.0; }
__device__ __forceinline__ double verify_rest(float p, float q) {
  const double d = verify_weight(p) - (q > 0.f ? (double)q : 0.0);
  return d > 0.0 ? d : 0.0;
}

// The struck tokens in [first, last), compacted into list by one wave; their number
__device__ __forceinline__ int struck_in(unsigned long long struck, int token, int first, int last, int* list) {
  const int lane = threadIdx.x & 63;
  const bool in = (struck >> lane & 1) && token >= first && token < last;
  const unsigned long long mask = __builtin_amdgcn_ballot_w64(in);
  if (in) list[__builtin_popcountll(mask & ((1ull << lane) - 1))] = token;
  return __builtin_popcountll(mask);
}

// Weights w[0..3] of elements v .. v+3 (0 past `last`), and their p
__device__ __forceinline__ void verify_load(const float* p, const float* q, int v, int last, int nstruck,
                                            const int* list, double w[4], double pw[4]) {
  float pv[4] = {0.f, 0.f, 0.f, 0.f}, qv[4] = {0.f, 0.f, 0.f, 0.f};
  if (v + 4 <= last) {
    const verify_f4_t x = *reinterpret_cast<const verify_f4_t*>(p + v);
#pragma unroll
    for (int e = 0; e < 4; e++) pv[e] = x[e];
    if (q) {
      const verify_f4_t y = *reinterpret_cast<const verify_f4_t*>(q + v);
#pragma unroll
      for (int e = 0; e < 4; e++) qv[e] = y[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (v + e < last) {
        pv[e] = p[v + e];
        if (q) qv[e] = q[v + e];
      }
  }
#pragma unroll
  for (int e = 0; e < 4; e++) {
    pw[e] = verify_weight(pv[e]);
    w[e] = q ? verify_rest(pv[e], qv[e]) : pw[e];
  }
  for (int i = 0; i < nstruck; i++) {
    const int t = list[i] - v;
#pragma unroll
    for (int e = 0; e < 4; e++) w[e] = t == e ? 0.0 : w[e];
  }
}

__device__ __forceinline__ double shfl_up_f64(double v, int by) {
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
  const unsigned lo = __shfl_up((unsigned)u, by), hi = __shfl_up((unsigned)(u >> 32), by);
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ double shfl_f64(double v, int from) {
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
  const unsigned lo = __shfl((unsigned)u, from), hi = __shfl((unsigned)(u >> 32), from);
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ double wave_scan_f64(double v) {  // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const double o = shfl_up_f64(v, m);
    v += lane >= m ? o : 0.0;
  }
  return v;
}

__global__ __launch_bounds__(kMassThreads) void verify_mass_kernel(const VerifyArgs a) {
  __shared__ VerifyEnd end;
  __shared__ int list[kVerifyNodes], nlist;
  __shared__ double sums[kMassThreads / 64][2];
  const int b = blockIdx.y, chunk = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int first = chunk * a.chunk_len, last = min(first + a.chunk_len, a.vocab);
  if (wave == 0) {
    const VerifyWalk w = verify_walk(a, b);
    const int n = struck_in(w.end.struck, w.token, first, last, list);
    if (lane == 0) end = w.end, nlist = n;
    if (chunk == 0) {
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
  double sw = 0.0, sp = 0.0;
#pragma unroll 4
  for (int v = first + 4 * threadIdx.x; v < last; v += 4 * kMassThreads) {
    double w[4], pw[4];
    verify_load(p, q, v, last, nlist, list, w, pw);
    sw += (w[0] + w[1]) + (w[2] + w[3]);
    sp += (pw[0] + pw[1]) + (pw[2] + pw[3]);
  }
  sw = wave_scan_f64(sw), sp = wave_scan_f64(sp);
  if (lane == 63) sums[wave][0] = sw, sums[wave][1] = sp;
  __syncthreads();
  if (threadIdx.x < 2) {
    double t = 0.0;
#pragma unroll
    for (int i = 0; i < kMassThreads / 64; i++) t += sums[i][threadIdx.x];
    a.mass[((size_t)b * a.chunks + chunk) * 2 + threadIdx.x] = t;
  }
}

__global__ __launch_bounds__(kPickThreads) void verify_pick_kernel(const VerifyArgs a) {
  constexpr int WAVES = kPickThreads / 64;
  __shared__ int list[kVerifyNodes], nlist, picked, fallback;
  __shared__ double wave_sum[WAVES];
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const VerifyEnd e = a.end[b];
  if (e.count == 0) return;
  // every wave: the chunk that the threshold falls in
  const double* mass = a.mass + (size_t)b * a.chunks * 2;
  const double mw = lane < a.chunks ? mass[2 * lane] : 0.0, mp = lane < a.chunks ? mass[2 * lane + 1] : 0.0;
  double run = wave_scan_f64(mw);
  const bool plain = !(shfl_f64(run, 63) > 0.0);  // nothing left of w: the target's row as it is
  const double mine = plain ? mp : mw;
  if (plain) run = wave_scan_f64(mp);
  const double total = shfl_f64(run, 63);
  int next = -1;
  if (total > 0.0) {
    const float u = a.uniform[(size_t)b * a.nodes];
    const double bar = (u > 0.f ? (double)fminf(u, 1.f) : 0.0) * total;
    unsigned long long over = __builtin_amdgcn_ballot_w64(run > bar);
    if (!over) over = 1ull << (63 - __builtin_clzll(__builtin_amdgcn_ballot_w64(mine > 0.0)));  // u = 1: the last
    const int chunk = __builtin_ctzll(over);
    double base = shfl_f64(run, max(chunk - 1, 0));
    base = chunk > 0 ? base : 0.0;
    const int first = chunk * a.chunk_len, last = min(first + a.chunk_len, a.vocab);
    if (wave == 0) {
      const int token = a.tokens[(size_t)b * a.nodes + min(lane, a.nodes - 1)];
      const int n = struck_in(plain ? 0 : e.struck, token, first, last, list);
      if (lane == 0) nlist = n, picked = 0x7FFFFFFF, fallback = -1;
    }
    __syncthreads();
    const size_t row = ((size_t)b * a.nodes + e.node) * a.vocab;
    const float *p = a.p + row, *q = e.residual && !plain ? a.q + row : nullptr;
    for (int at = first; at < last; at += kVerifyBlock) {
      const int v = at + 4 * threadIdx.x;
      double w[4] = {0.0, 0.0, 0.0, 0.0}, pw[4];
      if (v < last) verify_load(p, q, v, last, nlist, list, w, pw);
      const double sum = (w[0] + w[1]) + (w[2] + w[3]);
      const double scan = wave_scan_f64(sum);
      if (lane == 63) wave_sum[wave] = scan;
      __syncthreads();
      double before = base;
#pragma unroll
      for (int i = 0; i < WAVES; i++) {
        before += i < wave ? wave_sum[i] : 0.0;
        base += wave_sum[i];
      }
      double c = before + (scan - sum);
      int found = 0x7FFFFFFF, positive = -1;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        c += w[i];
        if (w[i] > 0.0) {
          positive = v + i;
          if (c > bar) found = min(found, v + i);
        }
      }
      if (found != 0x7FFFFFFF) atomicMin(&picked, found);
      if (positive >= 0) atomicMax(&fallback, positive);
      __syncthreads();
      if (picked != 0x7FFFFFFF) break;
    }
    next = picked != 0x7FFFFFFF ? picked : fallback;
  }
  if (threadIdx.x == 0) a.out_tokens[(size_t)b * a.nodes + e.count - 1] = next;
}

struct VerifyPlan {
  int chunks, chunk_len;
  size_t bytes;
};
static VerifyPlan verify_plan(int batch, int vocab) {
  const int blocks = (vocab + kVerifyBlock - 1) / kVerifyBlock;
  const int each = (blocks + kVerifyChunks - 1) / kVerifyChunks;
  const int chunks = (blocks + each - 1) / each;
  return VerifyPlan{chunks, each * kVerifyBlock,
                    (size_t)batch * (chunks * 2 * sizeof(double) + sizeof(VerifyEnd))};
}

}  // namespace exl3

using namespace exl3;

extern "C" size_t exl3_verify_workspace_bytes(int batch, int vocab) {
  if (batch <= 0 || vocab <= 0 || vocab > (1 << 28)) return 0;
  return verify_plan(batch, vocab).bytes;
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
  const VerifyPlan plan = verify_plan(batch, vocab);
  EXL3_CHECK_ARG(workspace && workspace_bytes >= plan.bytes && ((uintptr_t)workspace & 7) == 0,
                 "exl3_verify_drafts: workspace %zu bytes, need %zu (8-byte aligned)", workspace_bytes, plan.bytes);
  double* mass = static_cast<double*>(workspace);
  const VerifyArgs a{target_probs, draft_probs, tokens, parents, uniform, num_nodes, nodes, vocab, plan.chunks,
                     plan.chunk_len, accepted_nodes, counts, out_tokens, mass,
                     reinterpret_cast<VerifyEnd*>(mass + (size_t)batch * plan.chunks * 2)};
  verify_mass_kernel<<<dim3(plan.chunks, batch), kMassThreads, 0, as_stream(stream)>>>(a);
  EXL3_CHECK_LAUNCH();
  verify_pick_kernel<<<batch, kPickThreads, 0, as_stream(stream)>>>(a);
  EXL3_CHECK_LAUNCH();
  return EXL3_OK;
}
