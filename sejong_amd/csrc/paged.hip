// A paged key-value cache for many sequences: the plan of one step (block
// tables, positions and slots from the requests' lengths) and the attention
// of the step's tokens over the pages (no counterpart in the reference, whose
// cache holds one sequence: model lib.rs:36-50, architecture.rs:428-533).
#include <math.h>

#include "common.h"

using namespace sj;

namespace {

// ------------------------------------------------------------------- plan
//
// Token S_r + j of request r (S = exclusive sum of the counts) has position
// len_r + j; the pages that a request grows into are taken from the free list
// in the order of the requests.  Every workgroup sums all the requests itself
// (a few KB that stay in L2, one block scan) and expands 1024 tokens, so the
// plan is one launch and needs no workspace: the bound is that launch, the
// scan's latency and, for prompts, 12 bytes written per token.

constexpr int PT = 1024;  // threads, and tokens, of a workgroup

struct PlanArgs {
  const int32_t *lengths, *counts, *free_pages, *head;
  int32_t *table, *after, *starts, *positions, *slots, *owners, *summary;
  long ldt, nfree, cap;
  int R;
  uint32_t P, pages;
};

__device__ __forceinline__ uint32_t ceil_div(uint32_t n, uint32_t d) { return n / d + (n % d != 0); }

__global__ __launch_bounds__(PT) void k_paged_plan(PlanArgs a) {
  __shared__ long long w_tok[16], w_need[16];
  __shared__ uint32_t w_want[16], w_long[16];
  __shared__ int w_bad[16], w_at[16];
  __shared__ int h_req[PT], h_start[PT], h_first[PT];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int per = (a.R + PT - 1) / PT;
  const int r0 = min(t * per, a.R), r1 = min(r0 + per, a.R);
  long long tok = 0, need = 0;
  uint32_t want = 0, longest = 0;
  int bad = 0;
  for (int r = r0; r < r1; r++) {
    const int n = a.lengths[r], m = a.counts[r];
    if ((n | m) < 0) {
      bad = 1;
    } else {
      const uint32_t w = ceil_div((uint32_t)n + (uint32_t)m, a.P);
      tok += m;
      need += w - ceil_div((uint32_t)n, a.P);
      want = max(want, w);
      longest = max(longest, (uint32_t)n + (uint32_t)m);
    }
  }
  // inclusive sums over the wave, then over the 16 waves
  long long st = tok, sn = need;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const long long u = __shfl_up(st, o, 64), v = __shfl_up(sn, o, 64);
    if (lane >= o) st += u, sn += v;
  }
  want = wave_max(want);
  longest = wave_max(longest);
  bad = __any(bad);
  if (lane == 63) w_tok[wave] = st, w_need[wave] = sn, w_want[wave] = want, w_long[wave] = longest, w_bad[wave] = bad;
  h_req[t] = -1;
  __syncthreads();
  long long all_tok = 0, all_need = 0;
  for (int i = 0; i < 16; i++) {
    if (i < wave) st += w_tok[i], sn += w_need[i];
    all_tok += w_tok[i];
    all_need += w_need[i];
    want = max(want, w_want[i]);
    longest = max(longest, w_long[i]);
    bad |= w_bad[i];
  }
  const long long head = a.head ? a.head[0] : 0;
  int status = 0;
  if (head < 0 || head + all_need > a.nfree) status |= SJ_PLAN_NO_PAGES;
  if (want > (unsigned long long)a.ldt) status |= SJ_PLAN_TABLE_WIDTH;
  if (all_tok > a.cap) status |= SJ_PLAN_ROWS;
  if (bad || longest > 0x7fffffffu) status |= SJ_PLAN_LENGTHS;
  const bool ok = status == 0;

  // the requests again with their places: the first of a request's tokens in
  // this workgroup's range marks where it begins
  const long t0 = (long)blockIdx.x * PT;
  long long s = st - tok, f = sn - need;
  const bool lead = blockIdx.x == 0;
  for (int r = r0; r < r1; r++) {
    const int n = a.lengths[r], m = a.counts[r];
    if (lead) {
      a.starts[r] = ok ? (int)s : 0;
      if (a.after) a.after[r] = ok ? n + m : n;
    }
    if (!ok) continue;
    if (m > 0 && s < t0 + PT && s + m > t0) {
      const int at = s > t0 ? (int)(s - t0) : 0;
      h_req[at] = r;
      h_start[at] = (int)s;
      h_first[at] = (int)f;
    }
    s += m;
    f += ceil_div((uint32_t)n + (uint32_t)m, a.P) - ceil_div((uint32_t)n, a.P);
  }
  if (lead && t == 0) {
    a.starts[a.R] = ok ? (int)all_tok : 0;
    a.summary[0] = ok ? (int)all_tok : 0;
    a.summary[1] = (int)(head + (ok ? all_need : 0));
    a.summary[2] = status;
    a.summary[3] = longest > 0x7fffffffu ? 0x7fffffff : (int)longest;
  }
  __syncthreads();
  // each token's request: the last mark at or before it
  int at = h_req[t] >= 0 ? t : -1;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(at, o, 64);
    if (lane >= o) at = max(at, u);
  }
  if (lane == 63) w_at[wave] = at;
  __syncthreads();
  for (int i = 0; i < wave; i++) at = max(at, w_at[i]);
  const long g = t0 + t;
  if (g >= a.cap) return;
  int pos = -1, slot = -1, owner = -1;
  if (ok && at >= 0 && g < all_tok) {
    owner = h_req[at];
    const int n = a.lengths[owner];
    pos = n + (int)(g - h_start[at]);
    const uint32_t col = (uint32_t)pos / a.P, off = (uint32_t)pos - col * a.P, have = ceil_div((uint32_t)n, a.P);
    int page;
    if (col >= have) {
      page = a.free_pages[head + h_first[at] + (col - have)];
      if (off == 0) a.table[(long)owner * a.ldt + col] = page;  // a page's first position is always a new token here
    } else {
      page = a.table[(long)owner * a.ldt + col];
    }
    if (page >= 0 && (uint32_t)page < a.pages) slot = (int)((uint32_t)page * a.P + off);
  }
  a.positions[g] = pos;
  a.slots[g] = slot;
  a.owners[g] = owner;
}

// -------------------------------------------------------------- attention

struct PagedArgs {
  const void* q;
  long ldq;
  const void *k, *v;
  long ldkv;
  const int32_t* table;
  long ldt;
  const int32_t *owners, *positions;
  void* o;
  long ldo;
  float* lse;
  int requests, rows, HQ, HK, D;
  int pages, P;
  long window;
  float scale;  // log2(e) / sqrt(D): the softmax in powers of two
};

// the keys a row sees, [lo, hi), and its request; false for a padded row
__device__ __forceinline__ bool row_range(const PagedArgs& a, int row, int& owner, int& lo, int& hi) {
  const int pos = a.positions[row];
  owner = a.owners ? a.owners[row] : row;
  if (pos < 0 || owner < 0 || owner >= a.requests) return false;
  const long most = a.ldt * a.P;  // at most 2^31 - 1 (checked on the host)
  hi = (int)(pos + 1L < most ? pos + 1L : most);
  lo = a.window > 0 && pos + 1L > a.window ? (int)(pos + 1L - a.window) : 0;
  if (lo > hi) lo = hi;
  return true;
}

// The first row of scores and sums a wave carries along a walk, merged over
// the four waves of a workgroup (one row and query head).  A lane owns a key
// in the products with q and columns lane + 64 c in the sums over v.
template <typename T>
__global__ __launch_bounds__(256) void k_paged_rows(PagedArgs a) {
  __shared__ float q[256], p[4][64], acc[4][256], wm[4], wl[4];
  __shared__ int slot[4][64];
  const int row = blockIdx.x, h = blockIdx.y, D = a.D;
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  int owner, lo, hi;
  if (!row_range(a, row, owner, lo, hi)) return;
  const int kh = h / (a.HQ / a.HK);
  if (t < D) q[t] = a.scale * load_as_f32(a.q, sizeof(T) == 2 ? SJ_BF16 : SJ_F32, (long)row * a.ldq + (long)h * D + t);
  __syncthreads();
  const T* K = (const T*)a.k + (long)kh * D;
  const T* V = (const T*)a.v + (long)kh * D;
  const int32_t* pages = a.table + (long)owner * a.ldt;
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (long base = lo + 64L * w; base < hi; base += 256) {
    const long j = base + lane;
    int sl = -1;
    if (j < hi) {
      const int col = (int)(j / a.P), pg = pages[col];
      if (pg >= 0 && pg < a.pages) sl = pg * a.P + (int)(j - (long)col * a.P);
    }
    float s = -INFINITY;
    if (sl >= 0) {
      s = 0.f;
      const T* x = K + (long)sl * a.ldkv;
      for (int d = 0; d < D; d++) s = fmaf(q[d], load_as_f32(x, sizeof(T) == 2 ? SJ_BF16 : SJ_F32, d), s);
    }
    // a key without a page or with a score of -inf has no share; a NaN keeps its own
    const bool has = !(s == -INFINITY);
    if (!__any(has)) continue;
    const float mn = fmaxf(m, wave_max(s == s ? s : -INFINITY));
    const float alpha = m == -INFINITY ? 0.f : exp2f(m - mn);
    const float e = has ? exp2f(s - mn) : 0.f;
    l = l * alpha + wave_sum(e);
    m = mn;
    p[w][lane] = e;
    slot[w][lane] = has ? sl : -1;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int c = 0; c < 4; c++) o[c] *= alpha;
    for (int i = 0; i < 64; i++) {
      const int si = slot[w][i];
      if (si < 0) continue;
      const float pi = p[w][i];
#pragma unroll
      for (int c = 0; c < 4; c++)
        if (lane + 64 * c < D)
          o[c] = fmaf(pi, load_as_f32(V, sizeof(T) == 2 ? SJ_BF16 : SJ_F32, (long)si * a.ldkv + lane + 64 * c), o[c]);
    }
    __builtin_amdgcn_wave_barrier();
  }
#pragma unroll
  for (int c = 0; c < 4; c++) acc[w][lane + 64 * c] = o[c];
  if (lane == 0) wm[w] = m, wl[w] = l;
  __syncthreads();
  float M = -INFINITY, L = 0.f, f[4];
  for (int i = 0; i < 4; i++) M = fmaxf(M, wm[i]);
  for (int i = 0; i < 4; i++) {
    f[i] = wl[i] == 0.f ? 0.f : exp2f(wm[i] - M);
    L += wl[i] * f[i];
  }
  if (t < D) {
    float s = 0.f;
    for (int i = 0; i < 4; i++)
      if (wl[i] != 0.f) s += acc[i][t] * f[i];
    store_from_f32(a.o, sizeof(T) == 2 ? SJ_BF16 : SJ_F32, (long)row * a.ldo + (long)h * D + t, L == 0.f ? 0.f : s / L);
  }
  if (a.lse && t == 0) a.lse[(long)row * a.HQ + h] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
}

}  // namespace

extern "C" int sj_paged_plan(void* stream, const int32_t* lengths, const int32_t* counts, long requests,
                             long page_size, long pages, int32_t* table, long ldt, const int32_t* free_pages,
                             long free_count, const int32_t* free_head, int32_t* lengths_after, int32_t* starts,
                             int32_t* positions, int32_t* slots, int32_t* owners, long capacity, int32_t* summary) {
  SJ_REQUIRE(requests >= 0 && requests <= 1L << 24 && capacity >= 0 && capacity <= 0x7fffffffL && free_count >= 0 &&
                 free_count <= 0x7fffffffL,
             "paged plan: %ld requests, %ld rows, %ld free pages", requests, capacity, free_count);
  SJ_REQUIRE(page_size > 0 && page_size <= 0x7fffffffL && pages > 0 && pages <= 0x7fffffffL / page_size && ldt > 0 &&
                 ldt <= 0x7fffffffL / page_size,
             "paged plan: %ld pages of %ld, tables of %ld", pages, page_size, ldt);
  SJ_REQUIRE(starts && summary && (requests == 0 || (lengths && counts && table)) &&
                 (capacity == 0 || (positions && slots && owners)) && (free_count == 0 || free_pages),
             "paged plan: null");
  SJ_REQUIRE(lengths_after == nullptr || (lengths_after != lengths && lengths_after != counts),
             "paged plan: the lengths after the step need an array of their own");
  SJ_REQUIRE(free_head != summary + 1, "paged plan: the free list's position is read while the summary is written");
  PlanArgs a = {};
  a.lengths = lengths; a.counts = counts; a.free_pages = free_pages; a.head = free_head;
  a.table = table; a.after = lengths_after; a.starts = starts; a.positions = positions; a.slots = slots;
  a.owners = owners; a.summary = summary;
  a.ldt = ldt; a.nfree = free_count; a.cap = capacity;
  a.R = (int)requests; a.P = (uint32_t)page_size; a.pages = (uint32_t)pages;
  const long blocks = capacity > PT ? (capacity + PT - 1) / PT : 1;
  k_paged_plan<<<(unsigned)blocks, PT, 0, (hipStream_t)stream>>>(a);
  SJ_LAUNCH_CHECK("paged plan");
  return SJ_OK;
}

extern "C" size_t sj_paged_attention_workspace_bytes(long rows, long hq, long hk, long head_dim) {
  return 0;
}

extern "C" int sj_paged_attention(void* stream, const void* q, long ldq, const void* k_cache, const void* v_cache,
                                  long ldkv, int dtype, long pages, long page_size, const int32_t* table, long ldt,
                                  long requests, const int32_t* owners, const int32_t* positions, long rows, long hq,
                                  long hk, long head_dim, long window, void* o, long ldo, float* lse, void* workspace,
                                  size_t workspace_bytes) {
  SJ_REQUIRE(dtype == SJ_F32 || dtype == SJ_BF16, "paged attention dtype %d", dtype);
  SJ_REQUIRE(rows >= 0 && rows <= 0x7fffffffL && requests >= 0 && requests <= 0x7fffffffL && hq > 0 && hk > 0 &&
                 hq % hk == 0 && hq <= 65535 && head_dim > 0 && head_dim <= 256 && window >= 0 &&
                 ldq >= hq * head_dim && ldo >= hq * head_dim && ldkv >= hk * head_dim,
             "paged attention sequence/head dimensions");
  SJ_REQUIRE(page_size > 0 && page_size <= 0x7fffffffL && pages > 0 && pages <= 0x7fffffffL / page_size && ldt > 0 &&
                 ldt <= 0x7fffffffL / page_size,
             "paged attention: %ld pages of %ld, tables of %ld", pages, page_size, ldt);
  SJ_REQUIRE(owners || rows <= requests, "paged attention: %ld rows of %ld requests without owners", rows, requests);
  if (rows == 0 || requests == 0) return SJ_OK;
  SJ_REQUIRE(q && k_cache && v_cache && table && positions && o, "paged attention: null");
  const size_t need = sj_paged_attention_workspace_bytes(rows, hq, hk, head_dim);
  if (need > workspace_bytes || (need && !workspace))
    return sjh::fail(SJ_ERR_CAPACITY, "paged attention workspace: required %zu bytes, available %zu bytes", need,
                     workspace ? workspace_bytes : 0);
  PagedArgs a = {};
  a.q = q; a.ldq = ldq; a.k = k_cache; a.v = v_cache; a.ldkv = ldkv;
  a.table = table; a.ldt = ldt; a.owners = owners; a.positions = positions;
  a.o = o; a.ldo = ldo; a.lse = lse;
  a.requests = (int)requests; a.rows = (int)rows; a.HQ = (int)hq; a.HK = (int)hk; a.D = (int)head_dim;
  a.pages = (int)pages; a.P = (int)page_size; a.window = window;
  a.scale = (float)(1.4426950408889634 / sqrt((double)head_dim));
  const dim3 grid((unsigned)rows, (unsigned)hq);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == SJ_BF16)
    k_paged_rows<bf16_t><<<grid, 256, 0, s>>>(a);
  else
    k_paged_rows<float><<<grid, 256, 0, s>>>(a);
  SJ_LAUNCH_CHECK("paged attention");
  return SJ_OK;
}
