// The pages of a paged key-value cache when sequences change: forked, freed,
// copied, and compacted (no counterpart in the reference, whose cache holds one
// sequence: model lib.rs:36-50).
//
// `shared` [pages] counts the holders of a page beyond its first: a page that
// one table row names has 0 and needs no entry when the plan hands it out.  All
// state is written to arrays of its own, so that a void step leaves what was.
#include "chunks.h"
#include "lanes.h"

using namespace sj;

namespace {

constexpr int NT = 256, PER = 4, ROUND = NT * PER;  // a round: four consecutive entries a thread
static_assert(ROUND == CHUNK_ROUND, "a chunk is whole rounds");
constexpr long MOST_BLOCKS = 1L << 23;  // of 256 threads: a launch holds fewer than 2^32
constexpr int ALONE = 16384;  // entries, at most, that one workgroup takes by itself: 16 a thread
constexpr int COMPACT_ALONE = 8192;  // of a compaction (8192 pages 13.8 us, 16.6 in five launches; 16384 18.9 and 16.8)

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
// One workgroup's entries: rounds of four consecutive ones a thread, so that
// neighbouring lanes lie next to each other (16 consecutive ones a thread, each a
// store of its own, took 6 us more for 16384 entries).
template <int N>
__device__ __forceinline__ void entries_alone(const int32_t* x, long n, int fill, int32_t (&v)[N]) {
#pragma unroll
  for (int j = 0; j < N / 4; j++) {
    int32_t u[4];
    entries(x, 4096 * j + 4 * threadIdx.x, n, fill, u);
#pragma unroll
    for (int k = 0; k < 4; k++) v[4 * j + k] = u[k];
  }
}
// of 4 R flags a thread in that order: those before each of its rounds; all
template <int R>
__device__ __forceinline__ int ranks_alone(uint32_t flags, int* ws, int (&before)[R]) {
  int base = 0;
#pragma unroll
  for (int h = 0; h < R / 2; h++) {  // two rounds' counts in one word: neither passes 4096
    const uint32_t f = flags >> (8 * h);
    int at;
    const int all = block_scan<1024>(__popc(f & 15u) | (__popc(f & 240u) << 16), ws, at);
    before[2 * h] = base + (at & 0xffff);
    before[2 * h + 1] = base + (all & 0xffff) + (at >> 16);
    base += (all & 0xffff) + (all >> 16);
  }
  return base;
}
// four entries from i0 on, as far as there are n
__device__ __forceinline__ void put_entries(int32_t* y, long i0, long n, const int32_t (&v)[4]) {
  if (i0 + 4 <= n) {
    ((Int4*)(y + i0))->v = u32x4{(uint32_t)v[0], (uint32_t)v[1], (uint32_t)v[2], (uint32_t)v[3]};
  } else {
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (i0 + k < n) y[i0 + k] = v[k];
  }
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
// back to the list.  Several launches, because the holders of a page are added up
// between them (integers: the order does not matter): children and copies;
// tables and holders; the pages to free counted, then listed by their number (one
// launch where one workgroup holds them, ALONE pages).
//
// Launches and the loads that wait for each other bound it, not bytes: a pool of
// 162233 pages with 2000 requests takes 19.7 us in four launches (5.4 + 8.8 + 2.0 + 3.4; its 6 MB
// are 1.2 us at a copy's rate).  Sixteen entries a thread by loads of 4 bytes, on
// the few workgroups that this leaves, took 9.0 + 12.1 for the last two.

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

// The same in one launch, where one workgroup can hold the holders (ALONE pages
// and list entries) and go over the rows (SMALL_CELLS entries of tables): a
// workgroup for each row after, which finds its place in the list by itself, and
// one for the pool.  16 to 128 requests take 7.9 to 9.0 us, in three launches 11.2
// to 12.2; 256 take 12.7 and 11.9.
constexpr long SMALL_CELLS = 32768;
constexpr int SMALL_REQUESTS = 192;
__global__ __launch_bounds__(1024) void k_fork_small(ForkArgs a) {
  constexpr int N = ALONE / 1024, MANY = 4;
  extern __shared__ __attribute__((aligned(16))) int holders[];  // [ALONE]
  __shared__ int count[1024], first[1024], len[1024], ws[16], wrong, mine[2];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, i = blockIdx.x;
  const bool pool = i == a.requests;
  const int head = a.head ? a.head[0] : 0;
  // this workgroup's row and its pages before, asked for early
  const int r = pool ? -1 : a.parents[i], m = r >= 0 && r < a.before ? a.lengths[r] : 0;
  const int rows_full = bad_length(m, a.ldt, a.P) ? 0 : div(m, a.d_page), cols = rows_full + (rows_full * a.P < m);
  const int32_t* row = a.table + (long)r * a.ldt;
  int32_t v[N];
  if (pool) {
    entries_alone(a.shared, a.pages, 0, v);
    copy_ints(a.free_after, a.free_pages, a.nfree, t, 1024);
  }
  const int p = t < a.requests ? a.parents[t] : -1, n = t < a.before ? a.lengths[t] : 0;
  count[t] = 0;
  first[t] = a.requests;
  len[t] = n;
  if (t == 0) wrong = 0;
  __syncthreads();
  if (p >= 0 && p < a.before) {
    atomicAdd(&count[p], 1);
    atomicMin(&first[p], t);
  }
  if (p >= a.before || bad_length(n, a.ldt, a.P)) wrong = 1;
  const int cell = t < cols ? row[t] : -1;
  __syncthreads();
  const bool bad = wrong;
  bool alone = true, takes = false;
  if (!bad && p >= 0 && open_page(a, p, len[p], alone) >= 0) takes = first[p] != t || !alone;
  int place;
  const int taken = block_scan<1024>(takes, ws, place);
  int status = bad ? SJ_PLAN_LENGTHS : 0;
  if (head < 0 || (long)head + taken > a.nfree) status |= SJ_PLAN_NO_PAGES;
  if (!pool) {
    if (t == i) mine[0] = takes, mine[1] = place;
    __syncthreads();
    const bool good = !status && r >= 0, own = good && mine[0];
    const int fresh = own ? a.free_pages[head + mine[1]] : -1;
    for (long c = t; c < a.ldt; c += 1024) {
      int page = -1;
      if (good && c < cols) page = own && c == rows_full ? fresh : c == t ? cell : row[c];
      a.table_after[i * a.ldt + c] = page;
    }
    if (t == 0) {
      a.lengths_after[i] = good ? m : 0;
      a.copies[3 * i] = own ? row[rows_full] : -1;
      a.copies[3 * i + 1] = fresh;
      a.copies[3 * i + 2] = own ? m - rows_full * a.P : 0;
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < N; k += 4) *(u32x4*)(holders + 1024 * k + 4 * t) = *(const u32x4*)(v + k);
  const int last = !status && t < a.before ? open_page(a, t, n, alone) : -1;
  __syncthreads();
  if (last >= 0 && (count[t] == 0 || !alone)) atomicAdd(&holders[last], -1);
  // a row's full pages by a wave, MANY rows at once
  for (int r0 = w; !status && r0 < a.before; r0 += 16 * MANY) {
    int full[MANY], most = 0;
#pragma unroll
    for (int k = 0; k < MANY; k++) {
      const int q = r0 + 16 * k;
      full[k] = q < a.before && count[q] != 1 ? div(len[q], a.d_page) : 0;
      most = max(most, full[k]);
    }
    for (int c = lane; c < most; c += 64) {
      int page[MANY];
#pragma unroll
      for (int k = 0; k < MANY; k++) page[k] = c < full[k] ? a.table[(r0 + 16 * k) * a.ldt + c] : -1;
#pragma unroll
      for (int k = 0; k < MANY; k++)
        if (page[k] >= 0 && page[k] < a.pages) atomicAdd(&holders[page[k]], count[r0 + 16 * k] - 1);
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; k += 4) *(u32x4*)(v + k) = *(const u32x4*)(holders + 1024 * k + 4 * t);
  const uint32_t back = status ? 0 : flags_of(v, [](int h, int) { return h < 0; });
  int before[4];
  const int all = ranks_alone(back, ws, before), from = status ? 0 : head + taken, given = min(all, from);
#pragma unroll
  for (int j = 0; j < 4; j++) {
    int32_t u[4];
    int at = from - 1 - before[j];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const bool goes = (back >> (4 * j + k)) & 1, room = goes && at >= 0;
      if (room) a.free_after[at] = 4096 * j + 4 * t + k;
      at -= goes;
      u[k] = room ? 0 : v[4 * j + k];
    }
    put_entries(a.shared_after, 4096 * j + 4 * t, a.pages, u);
  }
  if (t == 0) {
    a.summary[0] = status ? 0 : taken;
    a.summary[1] = status ? head : from - given;
    a.summary[2] = status ? status : given < all ? SJ_FORK_LIST_FULL : 0;
    a.summary[3] = given;
  }
}

// ---------------------------------------------------------------- compact
//
// The pages of number `after` and more that are not on the free list move, in
// ascending order, into the free pages below, in the list's order.  Which pages
// are free is only on the list.  Where one workgroup can hold all of it
// (COMPACT_ALONE) it does; else each launch waits for the one before: marks on all high pages;
// the list takes its own off, and counts its low pages; they are put in a row,
// the moving pages counted; moves.  The tables are a launch of their own.
//
// 2048 pages to half take 7.9 us (5.2 + 2.7; five launches 16.6), 400001 pages to
// three quarters 19.7 us (2.9 + 3.4 + 3.5 + 6.8 + 4.7; 78 us with 16 entries a
// thread): again launches, and the moves' scattered writes.

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
// a thread's high pages i0 .. i0 + 3; flags: those that move, the first to target `at`
template <typename I>
__device__ __forceinline__ void move_pages(const CompactArgs& a, long i0, uint32_t moving, const I* targets, int at,
                                           int status) {
  const long high = a.pages - a.after;
  if (i0 >= high) return;
  int32_t v[PER], to[PER];
  entries(a.shared + a.after, i0, high, 0, v);
#pragma unroll
  for (int k = 0; k < PER; k++) {
    to[k] = -1;
    if (!status && (moving >> k) & 1) {
      to[k] = (int)targets[at];
      a.shared_after[to[k]] = v[k];
      a.copies[3L * at] = (int32_t)(a.after + i0 + k);
      a.copies[3L * at + 1] = to[k];
      a.copies[3L * at + 2] = a.P;
      at++;
    }
    if (!status) v[k] = 0;
  }
  put_entries(a.shared_after + a.after, i0, high, v);
  put_entries(a.to, i0, high, to);
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
    move_pages(a, i0, moving, a.targets, base + before, status);
    base += some;
  }
}
// pages and list of COMPACT_ALONE entries at most
__global__ __launch_bounds__(1024) void k_compact_alone(CompactArgs a) {
  constexpr int N = COMPACT_ALONE / 1024;
  __shared__ uint32_t listed[COMPACT_ALONE / 32];  // bit i: high page i is on the list
  __shared__ uint16_t targets[COMPACT_ALONE];
  __shared__ int ws[16];
  const int t = threadIdx.x;
  const long head = head_of(a), high = a.pages - a.after;
  int32_t v[N];
  entries_alone(a.free_pages, a.nfree, -1, v);
  copy_ints(a.shared_after, a.shared, a.after, t, 1024);
  if (t < COMPACT_ALONE / 32) listed[t] = 0;
  __syncthreads();
  const uint32_t low = flags_of(v, [&](int p, int k) {
    if (4096 * (k >> 2) + 4 * t + (k & 3) < head || p < 0 || p >= a.pages) return false;
    if (p >= a.after) atomicOr(&listed[(p - a.after) >> 5], 1u << ((p - a.after) & 31));
    return p < a.after;
  });
  int before[N / 4];
  const int below = ranks_alone(low, ws, before);
#pragma unroll
  for (int k = 0; k < N; k++)
    if ((low >> k) & 1) targets[before[k >> 2]++] = (uint16_t)v[k];
  // the scan's barriers are behind all marks, and before all targets are read
  uint32_t moving = 0;
#pragma unroll
  for (int k = 0; k < N; k++) {
    const int i = 4096 * (k >> 2) + 4 * t + (k & 3);
    moving |= (i < high && !((listed[i >> 5] >> (i & 31)) & 1) ? 1u : 0u) << k;
  }
  const int moves = ranks_alone(moving, ws, before);
  const int status = compact_status(a, head, below, moves);
  if (t == 0) compact_summary(a, head, below, moves, status);
  no_copies(a, status ? 0 : moves, t, 1024);
  for (long i = t; i < a.nfree; i += 1024)
    a.free_after[i] = status ? a.free_pages[i] : list_after(a, i, targets, below, moves);
#pragma unroll
  for (int j = 0; j < N / 4; j++) move_pages(a, 4096 * j + 4 * t, (moving >> (4 * j)) & 15u, targets, before[j], status);
}
__global__ __launch_bounds__(256) void k_compact_tables(CompactArgs a, long first) {
  const bool good = a.summary[2] == 0;
  const long r = first + blockIdx.x;
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
// One workgroup per copy, layer and cache, in launches of MOST_BLOCKS (a loop over
// further ones in the kernel cost small calls a quarter of a microsecond): reads
// and writes of 16 bytes, four in flight a thread.  600 pages of 16 rows of 512
// bf16 in 8 layers take 65.4 us, 4.8 TB/s read and written, the rate of a large
// copy; the filled parts of 64 pages 3.7 us, a launch and one round trip.  A page of
// a layer is one workgroup's whatever its size: 1 to 3 pages of 1 MB (64 rounds) in
// one layer take 35 us, 16 of them in 6 layers 87 (4.6 TB/s).

struct CopyArgs {
  uint8_t *k, *v;
  const int32_t* copies;
  long row, layer;  // bytes between rows and layers
  uint32_t first;  // of the launch, among copies, layers and caches
  int layers, pages, P, units, tail;  // 16-byte units of a row, its elements behind them
  Div d_units, d_layers;
};
struct __attribute__((packed, aligned(2))) Raw16 {
  u32x4 v;
};

template <typename T>
__global__ __launch_bounds__(256) void k_paged_copy(CopyArgs a) {
  const uint32_t part = a.first + blockIdx.x;
  const int t = threadIdx.x, item = (int)(part >> 1), i = div(item, a.d_layers), layer = item - i * a.layers;
  const int from = a.copies[3 * (long)i], to = a.copies[3 * (long)i + 1], n = min(a.copies[3 * (long)i + 2], a.P);
  if (from < 0 || from >= a.pages || to < 0 || to >= a.pages || from == to || n <= 0) return;
  uint8_t* base = (part & 1 ? a.v : a.k) + layer * a.layer;
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
    const long r = e / a.tail, at = r * a.row + 16L * a.units + (e - r * a.tail) * (long)sizeof(T);
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
        SJ_HIP(hipFuncSetAttribute((const void*)k_fork_small, hipFuncAttributeMaxDynamicSharedMemorySize, 4 * ALONE));
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
  if (most <= ALONE && requests <= SMALL_REQUESTS && requests_before <= 1024 && requests_before * ldt <= SMALL_CELLS) {
    k_fork_small<<<(unsigned)requests + 1, 1024, 4 * ALONE, s>>>(a);
    SJ_LAUNCH_CHECK("paged fork");
    return SJ_OK;
  }
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
  return 4 * compact_space(pages, free_count).all;
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
  const CompactSpace at = compact_space(pages, free_count);
  a.targets = a.to + at.targets;
  a.below = a.to + at.below;
  a.moves = a.to + at.moves;
  a.ldt = ldt; a.nfree = free_count; a.pages = pages; a.after = pages_after; a.capacity = capacity;
  a.list = chunks_of(free_count); a.high = chunks_of(pages - pages_after);
  a.requests = (int)requests; a.P = (int)page_size;
  a.d_page = make_div((uint32_t)page_size);
  hipStream_t s = (hipStream_t)stream;
  if (pages <= COMPACT_ALONE && free_count <= COMPACT_ALONE) {
    k_compact_alone<<<1, 1024, 0, s>>>(a);
  } else {
    const long blocks = (pages + 4 * NT - 1) / (4 * NT);
    k_compact_marks<<<(unsigned)(blocks < 1024 ? blocks : 1024), NT, 0, s>>>(a);
    if (a.list.count) k_compact_list<<<(unsigned)a.list.count, NT, 0, s>>>(a);
    const unsigned both = (unsigned)(a.list.count + a.high.count);
    if (both) k_compact_rank<<<both, NT, 0, s>>>(a);
    k_compact_moves<<<both ? both : 1, NT, 0, s>>>(a);
  }
  for (long first = 0; first < requests; first += MOST_BLOCKS)
    k_compact_tables<<<(unsigned)(requests - first < MOST_BLOCKS ? requests - first : MOST_BLOCKS), 256, 0, s>>>(a, first);
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
  const RowUnits row = row_units(width, size);
  a.units = row.units; a.tail = row.tail;
  a.d_units = make_div((uint32_t)(a.units ? a.units : 1));
  a.d_layers = make_div((uint32_t)layers);
  const long parts = 2 * count * layers;
  hipStream_t s = (hipStream_t)stream;
  for (long first = 0; first < parts; first += MOST_BLOCKS) {
    a.first = (uint32_t)first;
    const unsigned blocks = (unsigned)(parts - first < MOST_BLOCKS ? parts - first : MOST_BLOCKS);
    if (dtype == SJ_BF16)
      k_paged_copy<bf16_t><<<blocks, 256, 0, s>>>(a);
    else
      k_paged_copy<float><<<blocks, 256, 0, s>>>(a);
    SJ_LAUNCH_CHECK("paged copy");
  }
  return SJ_OK;
}
