// The pages of a paged key-value cache when sequences change: forked, freed,
// copied, and compacted (no counterpart in the reference, whose cache holds one
// sequence: model lib.rs:36-50).
//
// `shared` [pages] counts the holders of a page beyond its first: a page that
// one table row names has 0 and needs no entry when the plan hands it out.  All
// state is written to arrays of its own, so that a void step leaves what was.
#include "lanes.h"

using namespace sj;

namespace {

// The workgroups of a launch over n entries: chunks of whole rounds, a round
// four consecutive entries a thread.  Every workgroup adds up the counts of
// those before it, so there are at most 4096.
constexpr int NT = 256, PER = 4, ROUND = NT * PER;
struct Chunks {
  long chunk, count;
};
Chunks chunks_of(long n) {
  const long rounds = n > ROUND * 4096L ? (n + ROUND * 4096L - 1) / (ROUND * 4096L) : 1;
  return {rounds * ROUND, (n + rounds * ROUND - 1) / (rounds * ROUND)};
}
constexpr int ALONE = 16384;  // entries, at most, that one workgroup takes by itself: 16 a thread

struct __attribute__((packed, aligned(4))) Int4 {
  u32x4 v;
};
// N entries from i0 on; `fill` behind the last
template <int N>
__device__ __forceinline__ void entries(const int32_t* x, long i0, long n, int fill, int32_t (&v)[N]) {
  if (i0 + N <= n) {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const u32x4 u = ((const Int4*)(x + i0 + j))->v;
#pragma unroll
      for (int k = 0; k < 4; k++) v[j + k] = (int32_t)u[k];
    }
  } else {
#pragma unroll
    for (int k = 0; k < N; k++) v[k] = i0 + k < n ? x[i0 + k] : fill;
  }
}
// the flags of a thread's entries, bit k that of entry k
template <int N, class F>
__device__ __forceinline__ uint32_t flags_of(const int32_t (&v)[N], F f) {
  uint32_t m = 0;
#pragma unroll
  for (int k = 0; k < N; k++) m |= (f(v[k], k) ? 1u : 0u) << k;
  return m;
}
// y = x, by thread `at` of `step`
__device__ __forceinline__ void copy_ints(int32_t* y, const int32_t* x, long n, long at, long step) {
  for (long i = 4 * at; i < n; i += 4 * step) {
    if (i + 4 <= n) {
      ((Int4*)(y + i))->v = ((const Int4*)(x + i))->v;
    } else {
      for (long j = i; j < n; j++) y[j] = x[j];
    }
  }
}
// sum over the workgroup's N threads, and of those before this one
template <int N>
__device__ __forceinline__ int block_scan(int v, int* ws, int& before) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int upto = (int)scan_add((uint32_t)v);
  __syncthreads();
  if (lane == 63) ws[w] = upto;
  __syncthreads();
  int all = 0;
  before = upto - v;
#pragma unroll
  for (int k = 0; k < N / 64; k++) {
    if (k < w) before += ws[k];
    all += ws[k];
  }
  return all;
}
// the first n of the workgroups' counts
template <int N>
__device__ __forceinline__ int sum_counts(const int32_t* counts, long n, int* ws) {
  int v = 0, before;
  for (long i = threadIdx.x; i < n; i += N) v += counts[i];
  return block_scan<N>(v, ws, before);
}

// ------------------------------------------------------------------- fork
//
// Request i after the step is the request parents[i] before it.  With c_r
// children of row r, a full page of the row has c_r - 1 holders more; its last
// page, if not full, stays with the first child (if nobody else holds it), the
// others take a page of their own to copy into; what has no holder left goes
// back to the list.  Three launches, because the holders of a page are added up
// between them (integers: the order does not matter): children and copies;
// tables and holders; the pages to free, by their number.
//
// Launches and the loads that wait for each other bound it, not bytes: 64
// requests take 10.8 us (2.7 + 4.3 + 3.8), a pool of 170000 pages with 2000
// requests 20.3 us (5.5 + 9.0 + 2.5 + 3.4; its 8 MB are 2 us at a copy's rate).
// Sixteen entries a thread by loads of 4 bytes, on the few workgroups that this
// leaves, took 9.0 + 12.1 for the last two.

constexpr int FORK_ROWS = 16384;  // requests, at most: the children are counted in LDS

struct ForkArgs {
  const int32_t *parents, *table, *lengths, *shared, *free_pages, *head;
  int32_t *table_after, *lengths_after, *shared_after, *free_after, *copies, *summary;
  // workspace: the plan's status; the children of each row before; of each row
  // after, the place of its fresh page in the list (-1: none); the pages to free
  // of each workgroup
  int32_t *status, *children, *place, *counts;
  long ldt, nfree, chunk;
  int requests, before, P, pages;
  Div d_page;
};

__device__ __forceinline__ bool bad_length(int n, long ldt, int P) { return n < 0 || ((long)n + P - 1) / P > ldt; }

// the last page of a row that is not full: its number, or -1; alone: nobody
// else holds it
__device__ __forceinline__ int open_page(const ForkArgs& a, int r, int n, bool& alone) {
  const int full = div(n, a.d_page);
  alone = true;
  if (n == full * a.P) return -1;
  const int p = a.table[(long)r * a.ldt + full];
  if (p < 0 || p >= a.pages) return -1;
  alone = a.shared[p] <= 0;
  return p;
}

__global__ __launch_bounds__(1024) void k_fork_plan(ForkArgs a) {
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  if (blockIdx.x) {  // the others copy the holders and the list
    const long at = (long)(blockIdx.x - 1) * 1024 + t, step = (long)(gridDim.x - 1) * 1024;
    copy_ints(a.shared_after, a.shared, a.pages, at, step);
    copy_ints(a.free_after, a.free_pages, a.nfree, at, step);
    return;
  }
  extern __shared__ int lds[];
  int *count = lds, *first = lds + a.before;
  __shared__ int ws[16], wrong;
  for (int r = t; r < a.before; r += 1024) count[r] = 0, first[r] = a.requests;
  if (t == 0) wrong = 0;
  __syncthreads();
  for (int i = t; i < a.requests; i += 1024) {
    const int p = a.parents[i];
    if (p >= a.before) wrong = 1;
    if (p < 0 || p >= a.before) continue;
    atomicAdd(&count[p], 1);
    atomicMin(&first[p], i);
  }
  for (int r = t; r < a.before; r += 1024)
    if (bad_length(a.lengths[r], a.ldt, a.P)) wrong = 1;
  __syncthreads();
  const bool bad = wrong;
  int taken = 0;
  const int head = a.head ? a.head[0] : 0;
  for (int i0 = 0; i0 < a.requests; i0 += 1024) {
    const int i = i0 + t;
    bool takes = false;
    if (i < a.requests && !bad) {
      const int p = a.parents[i];
      bool alone;
      if (p >= 0 && open_page(a, p, a.lengths[p], alone) >= 0) takes = first[p] != i || !alone;
    }
    const uint64_t mask = __ballot(takes);
    if (lane == 0) ws[w] = __popcll(mask);
    __syncthreads();
    int at = taken + __popcll(mask & ((1ull << lane) - 1)), all = 0;
    for (int k = 0; k < 16; k++) {
      if (k < w) at += ws[k];
      all += ws[k];
    }
    if (i < a.requests) a.place[i] = takes ? at : -1;
    taken += all;
    __syncthreads();
  }
  int status = bad ? SJ_PLAN_LENGTHS : 0;
  if (head < 0 || (long)head + taken > a.nfree) status |= SJ_PLAN_NO_PAGES;
  for (int r = t; r < a.before; r += 1024) a.children[r] = count[r];
  if (t == 0) {
    a.summary[0] = status ? 0 : taken;
    a.summary[1] = head + (status ? 0 : taken);
    a.summary[2] = *a.status = status;
    a.summary[3] = 0;
  }
}

// a workgroup per row: the row after of that number, and the holders of the row
// before of that number
__global__ __launch_bounds__(256) void k_fork_rows(ForkArgs a) {
  const int i = blockIdx.x, t = threadIdx.x;
  const bool good = *a.status == 0;
  if (i < a.requests) {
    const int p = good ? a.parents[i] : -1, n = p >= 0 ? a.lengths[p] : 0, place = good ? a.place[i] : -1;
    const int full = div(n, a.d_page), cols = full + (full * a.P != n);
    const int fresh = place >= 0 ? a.free_pages[(a.head ? a.head[0] : 0) + place] : -1;
    for (long c = t; c < a.ldt; c += 256) {
      int page = -1;
      if (c < cols) page = c == full && place >= 0 ? fresh : a.table[(long)p * a.ldt + c];
      a.table_after[(long)i * a.ldt + c] = page;
    }
    if (t == 0) {
      a.lengths_after[i] = n;
      a.copies[3 * i] = place >= 0 ? a.table[(long)p * a.ldt + full] : -1;
      a.copies[3 * i + 1] = place >= 0 ? fresh : -1;
      a.copies[3 * i + 2] = place >= 0 ? n - full * a.P : 0;
    }
  }
  if (good && i < a.before) {
    const int n = a.lengths[i], full = div(n, a.d_page), c = a.children[i];
    if (c != 1)
      for (int col = t; col < full; col += 256) {
        const int p = a.table[(long)i * a.ldt + col];
        if (p >= 0 && p < a.pages) atomicAdd(&a.shared_after[p], c - 1);
      }
    bool alone;
    const int p = t == 0 ? open_page(a, i, n, alone) : -1;
    if (p >= 0 && (c == 0 || !alone)) atomicAdd(&a.shared_after[p], -1);
  }
}

// Pages without a holder (below 0) go back to the list, before its position, in
// descending order.
__global__ __launch_bounds__(NT) void k_fork_count(const int32_t* shared, long pages, long chunk, int32_t* counts) {
  __shared__ int ws[NT / 64];
  const long c0 = blockIdx.x * chunk;
  int n = 0, before, v[PER];
  for (long i0 = c0 + PER * threadIdx.x; i0 < min(c0 + chunk, pages); i0 += ROUND) {
    entries(shared, i0, pages, 0, v);
    n += __popc(flags_of(v, [](int h, int) { return h < 0; }));
  }
  n = block_scan<NT>(n, ws, before);
  if (threadIdx.x == 0) counts[blockIdx.x] = n;
}
template <int NT_, int PER_>
__global__ __launch_bounds__(NT_) void k_fork_free(ForkArgs a) {
  __shared__ int ws[NT_ / 64];
  if (*a.status) return;  // void: the summary is the plan's
  const int head = (a.head ? a.head[0] : 0) + a.summary[0];
  const long c0 = blockIdx.x * a.chunk;
  int all = sum_counts<NT_>(a.counts, blockIdx.x, ws);
  for (long r0 = c0; r0 < min(c0 + a.chunk, (long)a.pages); r0 += NT_ * PER_) {
    const long i0 = r0 + PER_ * threadIdx.x;
    int before, v[PER_];
    entries(a.shared_after, i0, a.pages, 0, v);
    const uint32_t back = flags_of(v, [](int h, int) { return h < 0; });
    const int some = block_scan<NT_>(__popc(back), ws, before);
    int at = head - 1 - all - before;
#pragma unroll
    for (int k = 0; k < PER_; k++)
      if ((back >> k) & 1) {
        if (at >= 0) {
          a.free_after[at] = (int32_t)(i0 + k);
          a.shared_after[i0 + k] = 0;
        }
        at--;
      }
    all += some;
  }
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) {
    const int given = min(all, head);
    a.summary[1] = head - given;
    a.summary[2] = given < all ? SJ_FORK_LIST_FULL : 0;
    a.summary[3] = given;
  }
}

// ---------------------------------------------------------------- compact
//
// The pages of number `after` and more that are not on the free list move, in
// ascending order, into the free pages below, in the list's order.  Which pages
// are free is only on the list.  Where one workgroup can hold all of it (ALONE)
// it does; else each launch waits for the one before: marks on all high pages;
// the list takes its own off, and counts its low pages; they are put in a row,
// the moving pages counted; moves.  The tables are a launch of their own.
//
// 2048 pages to half take 9.8 us (7.3 + 2.5; the five launches took 23.4), 400001
// pages to three quarters 20.8 us (2.9 + 3.5 + 3.3 + 6.6 + 4.6; 78 us with 16
// entries a thread): again launches, and the moves' scattered writes.

struct CompactArgs {
  const int32_t *table, *lengths, *shared, *free_pages, *head;
  int32_t *table_after, *shared_after, *free_after, *copies, *summary;
  int32_t *to;       // workspace [pages - after]: 1 moves, 0 does not; then where to, or -1
  int32_t *targets;  // [free_count] the free pages below
  int32_t *below, *moves;  // the workgroups' counts of both
  long ldt, nfree, pages, after, capacity;
  Chunks list, high;
  int requests, P;
  Div d_page;
};
__device__ __forceinline__ long head_of(const CompactArgs& a) { return a.head ? a.head[0] : 0; }
__device__ __forceinline__ int compact_status(const CompactArgs& a, long head, int below, int moves) {
  int status = 0;
  if (head < 0 || head > a.nfree || moves > below) status |= SJ_PLAN_NO_PAGES;
  if (moves > a.capacity) status |= SJ_PLAN_ROWS;
  return status;
}
__device__ __forceinline__ void compact_summary(const CompactArgs& a, long head, int below, int moves, int status) {
  a.summary[0] = status ? 0 : moves;
  a.summary[1] = status ? (int)head : (int)a.nfree - below + moves;
  a.summary[2] = status;
  a.summary[3] = status ? 0 : below - moves;
}
// entry i of the list after the moves: what is left of the low pages, at its end
template <typename I>
__device__ __forceinline__ int list_after(const CompactArgs& a, long i, const I* targets, int below, int moves) {
  const long j = i - (a.nfree - below);
  return j >= moves ? (int)targets[j] : -1;
}
// the copies behind the last move, by thread `at` of `step`
__device__ __forceinline__ void no_copies(const CompactArgs& a, int moves, long at, long step) {
  for (long i = 3L * moves + at; i < 3 * a.capacity; i += step) a.copies[i] = i % 3 == 2 ? 0 : -1;
}
// a thread's high pages i0 .. i0 + N - 1; flags: those that move, the first to target `at`
template <int N, typename I>
__device__ __forceinline__ void move_pages(const CompactArgs& a, long i0, uint32_t moving, const I* targets, int at,
                                           int status) {
  if (a.after + i0 >= a.pages) return;
  int32_t v[N];
  entries(a.shared + a.after, i0, a.pages - a.after, 0, v);
#pragma unroll
  for (int k = 0; k < N; k++) {
    const long i = i0 + k, p = a.after + i;
    if (p >= a.pages) continue;
    int to = -1;
    if (!status && (moving >> k) & 1) {
      to = (int)targets[at];
      a.shared_after[to] = v[k];
      a.copies[3L * at] = (int32_t)p;
      a.copies[3L * at + 1] = to;
      a.copies[3L * at + 2] = a.P;
      at++;
    }
    a.shared_after[p] = status ? v[k] : 0;
    a.to[i] = to;
  }
}

__global__ __launch_bounds__(NT) void k_compact_marks(CompactArgs a) {
  const long at = (long)blockIdx.x * NT + threadIdx.x, step = (long)gridDim.x * NT;
  copy_ints(a.shared_after, a.shared, a.after, at, step);
  for (long i = at; i < a.pages - a.after; i += step) a.to[i] = 1;
}
__global__ __launch_bounds__(NT) void k_compact_list(CompactArgs a) {
  __shared__ int ws[NT / 64];
  const long head = head_of(a), c0 = blockIdx.x * a.list.chunk;
  int n = 0, before, v[PER];
  for (long i0 = c0 + PER * threadIdx.x; i0 < min(c0 + a.list.chunk, a.nfree); i0 += ROUND) {
    entries(a.free_pages, i0, a.nfree, -1, v);
#pragma unroll
    for (int k = 0; k < PER; k++) {
      if (i0 + k < head) continue;
      n += v[k] >= 0 && v[k] < a.after;
      if (v[k] >= a.after && v[k] < a.pages) a.to[v[k] - a.after] = 0;
    }
  }
  n = block_scan<NT>(n, ws, before);
  if (threadIdx.x == 0) a.below[blockIdx.x] = n;
}
__global__ __launch_bounds__(NT) void k_compact_rank(CompactArgs a) {
  __shared__ int ws[NT / 64];
  const long head = head_of(a), block = blockIdx.x;
  int before, v[PER];
  if (block < a.list.count) {
    const long c0 = block * a.list.chunk;
    int base = sum_counts<NT>(a.below, block, ws);
    for (long r0 = c0; r0 < min(c0 + a.list.chunk, a.nfree); r0 += ROUND) {
      const long i0 = r0 + PER * threadIdx.x;
      entries(a.free_pages, i0, a.nfree, -1, v);
      const uint32_t low = flags_of(v, [&](int p, int k) { return i0 + k >= head && p >= 0 && p < a.after; });
      const int some = block_scan<NT>(__popc(low), ws, before);
      int at = base + before;
#pragma unroll
      for (int k = 0; k < PER; k++)
        if ((low >> k) & 1) a.targets[at++] = v[k];
      base += some;
    }
  } else {
    const long chunk = block - a.list.count, c0 = chunk * a.high.chunk, high = a.pages - a.after;
    int n = 0;
    for (long i0 = c0 + PER * threadIdx.x; i0 < min(c0 + a.high.chunk, high); i0 += ROUND) {
      entries(a.to, i0, high, 0, v);
      n += __popc(flags_of(v, [](int mark, int) { return mark == 1; }));
    }
    n = block_scan<NT>(n, ws, before);
    if (threadIdx.x == 0) a.moves[chunk] = n;
  }
}
__global__ __launch_bounds__(NT) void k_compact_moves(CompactArgs a) {
  __shared__ int ws[NT / 64];
  const long head = head_of(a), block = blockIdx.x;
  const int below = sum_counts<NT>(a.below, a.list.count, ws), moves = sum_counts<NT>(a.moves, a.high.count, ws);
  const int status = compact_status(a, head, below, moves);
  if (block == 0 && threadIdx.x == 0) compact_summary(a, head, below, moves, status);
  no_copies(a, status ? 0 : moves, block * NT + threadIdx.x, (long)gridDim.x * NT);
  if (block < a.list.count) {
    const long c0 = block * a.list.chunk;
    for (long i = c0 + threadIdx.x; i < min(c0 + a.list.chunk, a.nfree); i += NT)
      a.free_after[i] = status ? a.free_pages[i] : list_after(a, i, a.targets, below, moves);
    return;
  }
  const long chunk = block - a.list.count, c0 = chunk * a.high.chunk, high = a.pages - a.after;
  int base = chunk < a.high.count ? sum_counts<NT>(a.moves, chunk, ws) : 0;
  for (long r0 = c0; r0 < min(c0 + a.high.chunk, high); r0 += ROUND) {
    const long i0 = r0 + PER * threadIdx.x;
    int before, v[PER];
    entries(a.to, i0, high, 0, v);
    const uint32_t moving = flags_of(v, [](int mark, int) { return mark == 1; });
    const int some = block_scan<NT>(__popc(moving), ws, before);
    move_pages<PER>(a, i0, moving, a.targets, base + before, status);
    base += some;
  }
}
// pages and list of ALONE entries at most
__global__ __launch_bounds__(1024) void k_compact_alone(CompactArgs a) {
  constexpr int N = ALONE / 1024;
  __shared__ uint32_t listed[ALONE / 32];  // bit i: high page i is on the list
  __shared__ uint16_t targets[ALONE];
  __shared__ int ws[16];
  const int t = threadIdx.x, i0 = N * t;
  const long head = head_of(a), high = a.pages - a.after;
  int32_t v[N];
  entries(a.free_pages, i0, a.nfree, -1, v);
  copy_ints(a.shared_after, a.shared, a.after, t, 1024);
  if (t < ALONE / 32) listed[t] = 0;
  __syncthreads();
  uint32_t low = 0;
#pragma unroll
  for (int k = 0; k < N; k++) {
    const int p = v[k];
    if (i0 + k < head || p < 0 || p >= a.pages) continue;
    if (p < a.after)
      low |= 1u << k;
    else
      atomicOr(&listed[(p - a.after) >> 5], 1u << ((p - a.after) & 31));
  }
  int before;
  const int below = block_scan<1024>(__popc(low), ws, before);
#pragma unroll
  for (int k = 0; k < N; k++)
    if ((low >> k) & 1) targets[before++] = (uint16_t)v[k];
  // the scan's barriers are behind all marks, and before all targets are read
  uint32_t moving = ~(listed[t >> 1] >> (16 * (t & 1))) & 0xffffu;
  const long mine = high - i0;
  moving = mine <= 0 ? 0 : mine < N ? moving & ((1u << mine) - 1) : moving;
  const int moves = block_scan<1024>(__popc(moving), ws, before);
  const int status = compact_status(a, head, below, moves);
  if (t == 0) compact_summary(a, head, below, moves, status);
  no_copies(a, status ? 0 : moves, t, 1024);
  for (long i = t; i < a.nfree; i += 1024)
    a.free_after[i] = status ? a.free_pages[i] : list_after(a, i, targets, below, moves);
  move_pages<N>(a, i0, moving, targets, before, status);
}
__global__ __launch_bounds__(256) void k_compact_tables(CompactArgs a) {
  const bool good = a.summary[2] == 0;
  const long r = blockIdx.x;
  const int n = max(a.lengths[r], 0), full = div(n, a.d_page), cols = full + (full * a.P != n);
  for (long c = threadIdx.x; c < a.ldt; c += 256) {
    int p = a.table[r * a.ldt + c];
    if (good) {
      p = c < cols && p >= 0 && p < a.pages ? p : -1;
      if (p >= a.after) p = a.to[p - a.after];
    }
    a.table_after[r * a.ldt + c] = p;
  }
}

// ------------------------------------------------------------------- copy
//
// One workgroup per copy, layer and cache: reads and writes of 16 bytes, four
// in flight a thread.  600 pages of 16 rows of 512 bf16 in 8 layers take 65.6 us,
// 4.8 TB/s read and written, the rate of a large copy; the filled parts of 64
// pages 3.7 us, a launch and one round trip.

struct CopyArgs {
  uint8_t *k, *v;
  const int32_t* copies;
  long row, layer;  // bytes between rows and layers
  int layers, pages, P, units, tail;  // 16-byte units of a row, its elements behind them
  Div d_units, d_layers;
};
struct __attribute__((packed, aligned(2))) Raw16 {
  u32x4 v;
};

template <typename T>
__global__ __launch_bounds__(256) void k_paged_copy(CopyArgs a) {
  const int t = threadIdx.x, item = blockIdx.x >> 1, i = div(item, a.d_layers), layer = item - i * a.layers;
  const int from = a.copies[3 * (long)i], to = a.copies[3 * (long)i + 1], n = min(a.copies[3 * (long)i + 2], a.P);
  if (from < 0 || from >= a.pages || to < 0 || to >= a.pages || from == to || n <= 0) return;
  uint8_t* base = (blockIdx.x & 1 ? a.v : a.k) + layer * a.layer;
  const uint8_t* x = base + (long)from * a.P * a.row;
  uint8_t* y = base + (long)to * a.P * a.row;
  const long all = (long)n * a.units;
  for (long u0 = t; u0 < all; u0 += 1024) {
    u32x4 v[4];
    long at[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const long u = min(u0 + 256 * j, all - 1);
      const long r = a.units * (long)a.P <= 0x7fffffff ? div((uint32_t)u, a.d_units) : u / a.units;
      at[j] = r * a.row + 16 * (u - r * a.units);
      v[j] = ((const Raw16*)(x + at[j]))->v;
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (u0 + 256 * j < all) ((Raw16*)(y + at[j]))->v = v[j];
  }
  for (long e = t; e < (long)n * a.tail; e += 256) {
    const long r = e / a.tail, at = r * a.row + 16 * a.units + (e - r * a.tail) * (long)sizeof(T);
    *(T*)(y + at) = *(const T*)(x + at);
  }
}

}  // namespace

extern "C" size_t sj_paged_fork_workspace_bytes(long requests, long requests_before, long pages) {
  if (requests < 0 || requests_before < 0 || pages < 0) return 0;
  return 4 * (size_t)(requests + requests_before + chunks_of(pages).count + 4);
}

extern "C" int sj_paged_fork(void* stream, const int32_t* parents, long requests, const int32_t* table, long ldt,
                             const int32_t* lengths, long requests_before, long page_size, long pages,
                             const int32_t* shared, const int32_t* free_pages, long free_count, const int32_t* free_head,
                             int32_t* table_after, int32_t* lengths_after, int32_t* shared_after, int32_t* free_after,
                             int32_t* copies, int32_t* summary, void* workspace, size_t workspace_bytes) {
  SJ_REQUIRE(requests >= 0 && requests <= FORK_ROWS && requests_before >= 0 && requests_before <= FORK_ROWS &&
                 free_count >= 0 && free_count <= 0x7fffffffL,
             "paged fork: %ld requests of %ld, %ld free pages", requests, requests_before, free_count);
  SJ_REQUIRE(page_size > 0 && page_size <= 0x7fffffffL && pages > 0 && pages <= 0x7fffffffL / page_size && ldt > 0 &&
                 ldt <= 0x7fffffffL / page_size,
             "paged fork: %ld pages of %ld, tables of %ld", pages, page_size, ldt);
  SJ_REQUIRE(shared && shared_after && summary && (requests == 0 || (parents && table_after && lengths_after && copies)) &&
                 (requests_before == 0 || (table && lengths)) && (free_count == 0 || (free_pages && free_after)),
             "paged fork: null");
  SJ_REQUIRE(shared != shared_after && (free_count == 0 || free_pages != free_after) &&
                 (requests == 0 || ((const int32_t*)table_after != table && (const int32_t*)lengths_after != lengths)) &&
                 free_head != summary + 1,
             "paged fork: the state after the step needs arrays of its own");
  const size_t need = sj_paged_fork_workspace_bytes(requests, requests_before, pages);
  SJ_REQUIRE(((uintptr_t)workspace & 15) == 0, "paged fork: the workspace is not 16-byte aligned");
  if (need > workspace_bytes || !workspace)
    return sjh::fail(SJ_ERR_CAPACITY, "paged fork workspace: required %zu bytes, available %zu bytes", need,
                     workspace ? workspace_bytes : 0);
  static sj::OncePerDevice once;
  if (int st = sjh::once_per_device(once, [] {
        SJ_HIP(hipFuncSetAttribute((const void*)k_fork_plan, hipFuncAttributeMaxDynamicSharedMemorySize, 8 * FORK_ROWS));
        return SJ_OK;
      }))
    return st;
  ForkArgs a = {};
  a.parents = parents; a.table = table; a.lengths = lengths; a.shared = shared; a.free_pages = free_pages; a.head = free_head;
  a.table_after = table_after; a.lengths_after = lengths_after; a.shared_after = shared_after; a.free_after = free_after;
  a.copies = copies; a.summary = summary;
  a.status = (int32_t*)workspace;
  a.children = a.status + 4;
  a.place = a.children + requests_before;
  a.counts = a.place + requests;
  a.ldt = ldt; a.nfree = free_count;
  a.requests = (int)requests; a.before = (int)requests_before; a.P = (int)page_size; a.pages = (int)pages;
  a.d_page = make_div((uint32_t)page_size);
  hipStream_t s = (hipStream_t)stream;
  const long most = pages > free_count ? pages : free_count, copying = (most + 4095) / 4096;
  k_fork_plan<<<(unsigned)(1 + (copying < 512 ? copying : 512)), 1024, 8 * a.before, s>>>(a);
  if (requests || requests_before)
    k_fork_rows<<<(unsigned)(requests > requests_before ? requests : requests_before), 256, 0, s>>>(a);
  if (pages <= ALONE) {
    a.chunk = ALONE;
    k_fork_free<1024, ALONE / 1024><<<1, 1024, 0, s>>>(a);
  } else {
    const Chunks c = chunks_of(pages);
    a.chunk = c.chunk;
    k_fork_count<<<(unsigned)c.count, NT, 0, s>>>(shared_after, pages, c.chunk, a.counts);
    k_fork_free<NT, PER><<<(unsigned)c.count, NT, 0, s>>>(a);
  }
  SJ_LAUNCH_CHECK("paged fork");
  return SJ_OK;
}

extern "C" size_t sj_paged_compact_workspace_bytes(long pages, long free_count) {
  if (pages < 0 || free_count < 0) return 0;
  return 4 * (size_t)(pages + free_count + chunks_of(pages).count + chunks_of(free_count).count);
}

extern "C" int sj_paged_compact(void* stream, const int32_t* table, long ldt, const int32_t* lengths, long requests,
                                long page_size, long pages, long pages_after, const int32_t* shared,
                                const int32_t* free_pages, long free_count, const int32_t* free_head, int32_t* table_after,
                                int32_t* shared_after, int32_t* free_after, int32_t* copies, long capacity,
                                int32_t* summary, void* workspace, size_t workspace_bytes) {
  SJ_REQUIRE(requests >= 0 && requests <= 1L << 24 && free_count >= 0 && free_count <= 0x7fffffffL && capacity >= 0 &&
                 capacity <= 0x7fffffffL,
             "paged compact: %ld requests, %ld free pages, %ld copies", requests, free_count, capacity);
  SJ_REQUIRE(page_size > 0 && page_size <= 0x7fffffffL && pages > 0 && pages <= 0x7fffffffL / page_size && ldt > 0 &&
                 ldt <= 0x7fffffffL / page_size && pages_after >= 0 && pages_after <= pages,
             "paged compact: %ld pages of %ld to %ld, tables of %ld", pages, page_size, pages_after, ldt);
  SJ_REQUIRE(shared && shared_after && summary && (requests == 0 || (table && lengths && table_after)) &&
                 (free_count == 0 || (free_pages && free_after)) && (capacity == 0 || copies),
             "paged compact: null");
  SJ_REQUIRE(shared != shared_after && (free_count == 0 || free_pages != free_after) &&
                 (requests == 0 || (const int32_t*)table_after != table) && free_head != summary + 1,
             "paged compact: the state after the step needs arrays of its own");
  const size_t need = sj_paged_compact_workspace_bytes(pages, free_count);
  SJ_REQUIRE(((uintptr_t)workspace & 15) == 0, "paged compact: the workspace is not 16-byte aligned");
  if (need > workspace_bytes || !workspace)
    return sjh::fail(SJ_ERR_CAPACITY, "paged compact workspace: required %zu bytes, available %zu bytes", need,
                     workspace ? workspace_bytes : 0);
  CompactArgs a = {};
  a.table = table; a.lengths = lengths; a.shared = shared; a.free_pages = free_pages; a.head = free_head;
  a.table_after = table_after; a.shared_after = shared_after; a.free_after = free_after; a.copies = copies;
  a.summary = summary;
  a.to = (int32_t*)workspace;
  a.targets = a.to + pages;
  a.below = a.targets + free_count;
  a.moves = a.below + chunks_of(free_count).count;
  a.ldt = ldt; a.nfree = free_count; a.pages = pages; a.after = pages_after; a.capacity = capacity;
  a.list = chunks_of(free_count); a.high = chunks_of(pages - pages_after);
  a.requests = (int)requests; a.P = (int)page_size;
  a.d_page = make_div((uint32_t)page_size);
  hipStream_t s = (hipStream_t)stream;
  if (pages <= ALONE && free_count <= ALONE) {
    k_compact_alone<<<1, 1024, 0, s>>>(a);
  } else {
    const long blocks = (pages + 4 * NT - 1) / (4 * NT);
    k_compact_marks<<<(unsigned)(blocks < 1024 ? blocks : 1024), NT, 0, s>>>(a);
    if (a.list.count) k_compact_list<<<(unsigned)a.list.count, NT, 0, s>>>(a);
    const unsigned both = (unsigned)(a.list.count + a.high.count);
    if (both) k_compact_rank<<<both, NT, 0, s>>>(a);
    k_compact_moves<<<both ? both : 1, NT, 0, s>>>(a);
  }
  if (requests) k_compact_tables<<<(unsigned)requests, 256, 0, s>>>(a);
  SJ_LAUNCH_CHECK("paged compact");
  return SJ_OK;
}

extern "C" int sj_paged_copy(void* stream, void* k_cache, void* v_cache, long ldkv, int dtype, long layers,
                             long layer_stride, long pages, long page_size, long width, const int32_t* copies,
                             long count) {
  SJ_REQUIRE(dtype == SJ_F32 || dtype == SJ_BF16, "paged copy dtype %d", dtype);
  SJ_REQUIRE(layers >= 0 && layers <= 65536 && count >= 0 && count <= 1L << 24 && count * layers < 1L << 30 && width > 0 &&
                 width <= ldkv && ldkv <= 0x7fffffffL && layer_stride >= 0,
             "paged copy: %ld copies in %ld layers of %ld (stride %ld)", count, layers, width, ldkv);
  SJ_REQUIRE(page_size > 0 && page_size <= 0x7fffffffL && pages > 0 && pages <= 0x7fffffffL / page_size,
             "paged copy: %ld pages of %ld", pages, page_size);
  if (count == 0 || layers == 0) return SJ_OK;
  SJ_REQUIRE(k_cache && v_cache && copies, "paged copy: null");
  const long size = dtype == SJ_F32 ? 4 : 2;
  CopyArgs a = {};
  a.k = (uint8_t*)k_cache; a.v = (uint8_t*)v_cache; a.copies = copies;
  a.row = ldkv * size; a.layer = layer_stride * size;
  a.layers = (int)layers; a.pages = (int)pages; a.P = (int)page_size;
  a.units = (int)(width * size / 16); a.tail = (int)(width - a.units * 16 / size);
  a.d_units = make_div((uint32_t)(a.units ? a.units : 1));
  a.d_layers = make_div((uint32_t)layers);
  const unsigned blocks = (unsigned)(2 * count * layers);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == SJ_BF16)
    k_paged_copy<bf16_t><<<blocks, 256, 0, s>>>(a);
  else
    k_paged_copy<float><<<blocks, 256, 0, s>>>(a);
  SJ_LAUNCH_CHECK("paged copy");
  return SJ_OK;
}
