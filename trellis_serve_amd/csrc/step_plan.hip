// A serving step's pages, rows and slots from the requests' lengths (gfx950).
//
// Sequence b holds len_b tokens and asks for new_b more, or gives its last -new_b up.  Pages hold 16 tokens:
//   have = ceil(len / 16);  need = ceil((len + new) / 16) - have  of a sequence that grows, taken from a ring of free pages
//   in order of b: b's first is entry (need_0 + .. + need_b-1) of the ring's live part;  give = have - ceil((len + new) /
//   16) of one that shrinks, put behind the live part in order of b.
// A sequence is refused (it gets no token, its rows are -1) when its table row or the step's rows end before its tokens, or
// when the running sum of need passes the live part: what one sequence gets depends on those before it only through sums, so
// the whole is two prefix sums and a copy.  Saturating sums of numbers >= 0 are associative, which keeps them in 32 bits.
//
// Latency bounds it: 4.8 us of kernel for 8 sequences of one row each, 4.6 + 3.6 us for 1024 sequences of up to 127 rows.  Both scans
// of a turn take one barrier each, waves inside by DPP (four scans of two barriers, waves by LDS shuffles: 6.0 and 5.2 us).
//
// step_plan_kernel: one workgroup scans the sequences, 1024 at a time, and, where the step is small, fills the rows too.
// Otherwise step_fill_kernel does: waves of one sequence write its rows, its new table entries and its returned pages.  The
// ring's state may be updated in place, since only the first kernel reads it.
// A returned page may go to the place of one that is taken in the same step, where the ring has fewer places than there are pages
// (live + given back > ring_pages): then all that is taken is read before anything is put back.  step_plan_kernel has a barrier
// between the two; before step_fill_kernel it writes the taken pages into the table, and the fill reads them there (1024 sequences
// of up to 127 rows: 35 us, else 7.6).
#include <algorithm>

#include "exl3_api.hpp"
#include "kv_device.hpp"

namespace exl3 {

constexpr int kPlanThreads = 1024;

struct StepPlanArgs {
  int* table;
  int max_pages;
  const int *lens, *new_lens;
  int batch;
  int* ring;
  int ring_pages;
  const int* state;
  int* state_out;
  int rows;
  int *row_start, *counts, *lens_after, *positions, *row_lens, *row_seq;
  long long* slots;
  int* base;  // [batch]: a sequence's first taken (or returned) page; then PlanRing
  int slices; // waves per sequence of the fill
};

// The step's view of the ring, behind `base`
struct PlanRing {
  int head, live;  // before the step
  int places;      // for returned pages: those of no live entry after the step's pages are taken; pages past them are left out
  int early;       // the table has the taken pages before the fill
};
constexpr int kPlanRingInts = sizeof(PlanRing) / sizeof(int);
__device__ __forceinline__ PlanRing& plan_ring(const StepPlanArgs& a) { return *reinterpret_cast<PlanRing*>(a.base + a.batch); }

// sums stop at kMost, which leaves room for one more number in 32 bits
constexpr int kMost = (1 << 30) - 1;

template <int CTRL, int ROWS>
__device__ __forceinline__ int plan_add(int v) {
  return min(v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, ROWS == 0xF), kMost);
}

// inclusive scans over the workgroup of N kinds of numbers in 0 .. kMost; carry: what came before, becomes the total.  part: LDS,
// of this call alone, so that the barrier of the one between two of its turns keeps it
template <int N>
__device__ __forceinline__ void plan_scan(int (&v)[N], int (&carry)[N], int (&part)[N][kPlanThreads / 64]) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
  for (int i = 0; i < N; i++) {
    v[i] = plan_add<0x111, 0xF>(v[i]);  // row_shr:1, 2, 4, 8: inside each row of 16
    v[i] = plan_add<0x112, 0xF>(v[i]);
    v[i] = plan_add<0x114, 0xF>(v[i]);
    v[i] = plan_add<0x118, 0xF>(v[i]);
    v[i] = plan_add<0x142, 0xA>(v[i]);  // row_bcast:15 into rows 1 and 3
    v[i] = plan_add<0x143, 0xC>(v[i]);  // row_bcast:31 into rows 2 and 3
    if (lane == 63) part[i][wave] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; i++) {
    int before = carry[i], total = carry[i];
#pragma unroll
    for (int w = 0; w < kPlanThreads / 64; w++) {
      before = w == wave ? total : before;
      total = min(total + part[i][w], kMost);
    }
    carry[i] = total;
    v[i] = min(before + v[i], kMost);
  }
}

__device__ __forceinline__ int plan_pages(int tokens) { return (int)(((unsigned)tokens + kPage - 1) / kPage); }

// What the scans say of sequence b, all asked for at once
struct PlanSequence {
  int len, asked, have, base, count, after, r0, r1;
  int* row;
};
__device__ __forceinline__ PlanSequence plan_sequence(const StepPlanArgs& a, int b) {
  const int len = min(max(a.lens[b], 0), a.max_pages * kPage);
  return PlanSequence{len, a.new_lens[b], plan_pages(len), a.base[b], a.counts[b], a.lens_after[b], a.row_start[b],
                      a.row_start[b + 1], a.table + (size_t)b * a.max_pages};
}

// A page that a sequence takes: base + j is below the live pages
__device__ __forceinline__ int plan_taken(const StepPlanArgs& a, const PlanRing& ring, const PlanSequence& s, int j) {
  const unsigned at = (unsigned)ring.head + s.base + j, P = a.ring_pages;
  return a.ring[at < P ? at : at - P];
}

// The pages that a sequence takes, into its table row
__device__ __forceinline__ void plan_take(const StepPlanArgs& a, const PlanRing& ring, const PlanSequence& s, int first, int step) {
  const int need = s.asked < 0 ? 0 : plan_pages(s.len + s.count) - s.have;
  for (int j = first; j < need; j += step) s.row[s.have + j] = plan_taken(a, ring, s, j);
}

// Sequence b's rows.  in_table: the pages that it takes are there
__device__ __forceinline__ void plan_rows(const StepPlanArgs& a, const PlanRing& ring, const PlanSequence& s, int b, int first,
                                          int step, bool in_table) {
  for (int i = first; i < s.r1 - s.r0; i += step) {
    const int r = s.r0 + i, pos = s.len + i, lp = pos / kPage;
    const bool live = i < s.count;
    int page = 0;
    if (live) page = in_table || lp < s.have ? s.row[lp] : plan_taken(a, ring, s, lp - s.have);
    a.positions[r] = live ? pos : -1;
    a.row_lens[r] = live ? pos + 1 : 0;
    a.row_seq[r] = live ? b : -1;
    a.slots[r] = live ? (long long)page * kPage + pos % kPage : -1;
  }
}

// The rows behind the last sequence
__device__ __forceinline__ void plan_no_rows(const StepPlanArgs& a, int first, int step) {
  for (int r = a.row_start[a.batch] + first; r < a.rows; r += step)
    a.positions[r] = -1, a.row_lens[r] = 0, a.row_seq[r] = -1, a.slots[r] = -1;
}

// The pages that a sequence gives up, to the ring's end
__device__ __forceinline__ void plan_give(const StepPlanArgs& a, const PlanRing& ring, const PlanSequence& s, int first, int step) {
  const int keep = plan_pages(s.after), give = s.asked < 0 ? min(s.have - keep, ring.places - s.base) : 0;
  const unsigned to = (unsigned)ring.head + (unsigned)ring.live + (unsigned)s.base;
  for (int j = first; j < give; j += step) a.ring[(to + j) % (unsigned)a.ring_pages] = s.row[keep + j];
}

template <bool FILL>
__global__ __launch_bounds__(kPlanThreads) void step_plan_kernel(const StepPlanArgs a) {
  __shared__ int part1[2][kPlanThreads / 64], part2[1][kPlanThreads / 64], popped;
  const int head = (int)((unsigned)a.state[0] % (unsigned)a.ring_pages);
  const int live = min(max(a.state[1], 0), a.ring_pages);
  const int room = a.max_pages * kPage, lane = threadIdx.x & 63;
  int ends[2] = {0, 0}, pages[1] = {0};  // rows asked for and pages given back; pages asked for
  if (threadIdx.x == 0) popped = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kPlanThreads) {
    const int b = b0 + threadIdx.x;
    const bool in = b < a.batch;
    const int len = in ? min(max(a.lens[b], 0), room) : 0, asked = in ? a.new_lens[b] : 0;
    const int grow = max(asked, 0), have = plan_pages(len);
    const int left = asked < 0 ? (asked < -len ? 0 : len + asked) : len;
    const int give = have - plan_pages(left);
    int v[2] = {min(grow, kMost), give}, sum[1];
    plan_scan(v, ends, part1);
    const bool fits = grow <= room - len && v[0] <= a.rows;
    const int need = fits ? plan_pages(len + grow) - have : 0;
    sum[0] = need;
    plan_scan(sum, pages, part2);
    const bool ok = fits && (need == 0 || sum[0] <= live);
    // the sums rise, so what is taken is the largest that passes
    const unsigned long long served = __builtin_amdgcn_ballot_w64(sum[0] <= live);
    if (served != 0 && lane == 63 - __builtin_clzll(served)) atomicMax(&popped, sum[0]);
    if (in) {
      a.row_start[b + 1] = min(v[0], a.rows);
      a.counts[b] = ok ? grow : 0;
      a.lens_after[b] = asked < 0 ? left : ok ? len + grow : len;
      a.base[b] = asked < 0 ? v[1] - give : sum[0] - need;
    }
  }
  __syncthreads();
  const bool early = live + ends[1] > a.ring_pages;
  const PlanRing ring{head, live, a.ring_pages - (live - popped), early};
  if (threadIdx.x == 0) {
    a.row_start[0] = 0;
    plan_ring(a) = ring;
    const unsigned at = (unsigned)head + (unsigned)popped;
    a.state_out[0] = (int)(at % (unsigned)a.ring_pages);
    a.state_out[1] = min(live - popped + ends[1], a.ring_pages);
  }
  if (!FILL && !early) return;
  __syncthreads();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int b = wave; b < a.batch; b += kPlanThreads / 64) {
    const PlanSequence s = plan_sequence(a, b);
    plan_take(a, ring, s, lane, 64);
    if (FILL) plan_rows(a, ring, s, b, lane, 64, false);
    if (FILL && !early) plan_give(a, ring, s, lane, 64);
  }
  if (!FILL) return;
  if (wave == a.batch % (kPlanThreads / 64)) plan_no_rows(a, lane, 64);
  if (!early) return;
  __syncthreads();
  for (int b = wave; b < a.batch; b += kPlanThreads / 64) plan_give(a, ring, plan_sequence(a, b), lane, 64);
}

__global__ __launch_bounds__(256) void step_fill_kernel(const StepPlanArgs a) {
  const long long i = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (i >= (long long)(a.batch + 1) * a.slices) return;
  const int b = (int)(i / a.slices), first = (int)(i % a.slices) * 64 + (threadIdx.x & 63), step = a.slices * 64;
  if (b == a.batch) return plan_no_rows(a, first, step);
  const PlanRing ring = plan_ring(a);
  const PlanSequence s = plan_sequence(a, b);
  if (!ring.early) plan_take(a, ring, s, first, step);
  plan_rows(a, ring, s, b, first, step, ring.early);
  plan_give(a, ring, s, first, step);
}

}  // namespace exl3

using namespace exl3;

extern "C" size_t exl3_kv_step_plan_workspace_bytes(int batch) {
  return batch <= 0 ? 0 : ((size_t)batch + kPlanRingInts) * sizeof(int);
}

extern "C" int exl3_kv_step_plan(int* page_table, int max_pages, const int* seq_lens, const int* new_lens, int batch,
                                 int page_size, int* free_pages, int num_free, const int* free_state, int* free_state_out,
                                 int rows, int* row_start, int* counts, int* lens_after, int* positions, int* row_lens,
                                 int* row_seq, long long* slots, void* workspace, size_t workspace_bytes, void* stream) {
  EXL3_CHECK_ARG(page_size == kPage, "exl3_kv_step_plan: page_size = %d (supported: 16)", page_size);
  EXL3_CHECK_ARG(batch >= 0 && max_pages >= 1 && max_pages <= (1 << 26) && (long long)batch * max_pages < (1LL << 30) &&
                     num_free >= 1 && num_free <= (1 << 28) && rows >= 0 && rows < (1 << 28),
                 "exl3_kv_step_plan: batch = %d, max_pages = %d, free pages = %d, rows = %d", batch, max_pages, num_free,
                 rows);
  if (batch == 0 && rows == 0) return EXL3_OK;
  EXL3_CHECK_ARG(batch >= 1, "exl3_kv_step_plan: %d rows of no sequence", rows);
  EXL3_CHECK_ARG(page_table && seq_lens && new_lens && free_pages && free_state && free_state_out && row_start && counts &&
                     lens_after && (rows == 0 || (positions && row_lens && row_seq && slots)),
                 "exl3_kv_step_plan: null pointer");
  const size_t need = exl3_kv_step_plan_workspace_bytes(batch);
  EXL3_CHECK_ARG(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 3) == 0,
                 "exl3_kv_step_plan: workspace %zu bytes, need %zu (4-byte aligned)", workspace_bytes, need);
  const size_t n = (size_t)batch * sizeof(int), r = (size_t)rows * sizeof(int);
  const Span all[] = {{page_table, n * max_pages}, {free_pages, num_free * sizeof(int)}, {free_state_out, 2 * sizeof(int)},
                      {row_start, n + sizeof(int)}, {counts, n}, {lens_after, n}, {positions, r}, {row_lens, r},
                      {row_seq, r}, {slots, 2 * r}, {workspace, need}, {seq_lens, n}, {new_lens, n},
                      {free_state == free_state_out ? nullptr : free_state, 2 * sizeof(int)}};
  EXL3_CHECK_ARG(apart(all, 11), "exl3_kv_step_plan: what the call writes overlaps another tensor of it");
  StepPlanArgs a{page_table, max_pages, seq_lens, new_lens, batch, free_pages, num_free, free_state, free_state_out, rows,
                 row_start, counts, lens_after, positions, row_lens, row_seq, slots, static_cast<int*>(workspace), 1};
  if (batch <= 256 && rows <= 2048) {
    step_plan_kernel<true><<<1, kPlanThreads, 0, as_stream(stream)>>>(a);
    EXL3_CHECK_LAUNCH();
    return EXL3_OK;
  }
  // waves per sequence: one while the sequences fill the card, then enough for about 256 rows a wave on average
  a.slices = (int)std::max<long long>(1, std::min<long long>(64, rows / (256LL * batch)));
  step_plan_kernel<false><<<1, kPlanThreads, 0, as_stream(stream)>>>(a);
  EXL3_CHECK_LAUNCH();
  const long long waves = (long long)(batch + 1) * a.slices;
  step_fill_kernel<<<(unsigned)((waves + 3) / 4), 256, 0, as_stream(stream)>>>(a);
  EXL3_CHECK_LAUNCH();
  return EXL3_OK;
}
