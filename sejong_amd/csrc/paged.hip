// A paged key-value cache for many sequences: the plan of one step (block
// tables, positions and slots from the requests' lengths) and the attention
// of the step's tokens over the pages (no counterpart in the reference, whose
// cache holds one sequence: model lib.rs:36-50, architecture.rs:428-533).
#include "paged_walk.h"

using namespace sj;

namespace {

// ------------------------------------------------------------------- plan
//
// Token S_r + j of request r (S = exclusive sum of the counts) has position
// len_r + j; the pages that a request grows into are taken from the free list
// in the order of the requests.  Every workgroup sums all the requests itself
// (a few KB that stay in L2, one block scan) and expands 1024 tokens, four to
// a thread, so the plan is one launch and needs no workspace: the bound is
// that launch, the chain of loads lengths -> page ids, and, for prompts, the
// 12 bytes written per token.  64 requests of one token 4.4 us (a launch is
// 3.7), 1500 requests of 395000 tokens 8.1 (with one token a thread and 1024
// threads a workgroup 5.7 and 16.2).

constexpr int PT = 256;    // threads of a workgroup
constexpr int PTOK = 1024; // its tokens

struct PlanArgs {
  const int32_t *lengths, *counts, *free_pages, *head;
  int32_t *table, *after, *starts, *positions, *slots, *owners, *summary;
  long ldt, nfree, cap;
  int R, P;
  Div d_page;
  uint32_t pages;
};

__global__ __launch_bounds__(PT) void k_paged_plan(PlanArgs a) {
  __shared__ uint32_t w_tok[4], w_need[4], w_want[4], w_long[4], w_bad[4];
  __shared__ float w_size[4];
  __shared__ int w_at[4];
  // a request's marks lie where its tokens begin in this workgroup's range
  __shared__ __attribute__((aligned(16))) int h_req[PTOK];
  __shared__ int h_start[PTOK], h_len[PTOK], h_first[PTOK], h_tail[PTOK], h_fresh[PTOK];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int per = (a.R + PT - 1) / PT;
  const int r0 = min(t * per, a.R), r1 = min(r0 + per, a.R);
  const int head = a.head ? a.head[0] : 0;
  // the first of a thread's requests stay in registers (all of 2048)
  constexpr int HELD = 8;
  int hn[HELD], hm[HELD];
#pragma unroll
  for (int i = 0; i < HELD; i++) {
    hn[i] = r0 + i < r1 ? a.lengths[r0 + i] : 0;
    hm[i] = r0 + i < r1 ? a.counts[r0 + i] : 0;
  }
  // 32-bit sums are exact wherever the sum of the counts, watched in fp32, is
  // below 3e9: there are at most as many pages to take as tokens and requests
  uint32_t tok = 0, need = 0, want = 0, longest = 0, bad = 0;
  float size = 0.f;
  auto pages_of = [&](int n) {
    const int q = div(n, a.d_page);
    return (uint32_t)(q + (q * a.P != n));
  };
  auto count = [&](int n, int m) {
    const uint32_t after = (uint32_t)n + (uint32_t)m;
    if ((n | m) < 0 || (int)after < 0) {
      bad = 1;
    } else {
      const uint32_t w = pages_of((int)after);
      tok += m;
      size += (float)m;
      need += w - pages_of(n);
      want = max(want, w);
      longest = max(longest, after);
    }
  };
#pragma unroll
  for (int i = 0; i < HELD; i++)
    if (i < per) count(hn[i], hm[i]);  // past the last request 0 and 0, which count for nothing
#pragma unroll 1
  for (int r = r0 + HELD; r < r1; r++) count(a.lengths[r], a.counts[r]);
  uint32_t st = scan_add(tok), sn = scan_add(need);
  want = wave_max(want);
  longest = wave_max(longest);
  size = wave_sum(size);
  bad = __any(bad);
  if (lane == 63) w_tok[wave] = st, w_need[wave] = sn;
  if (lane == 0) w_want[wave] = want, w_long[wave] = longest, w_bad[wave] = bad, w_size[wave] = size;
  *(int4*)(h_req + 4 * t) = make_int4(-1, -1, -1, -1);
  __syncthreads();
  uint32_t all_tok = 0, all_need = 0;
  size = 0.f;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if (i < wave) st += w_tok[i], sn += w_need[i];
    all_tok += w_tok[i];
    all_need += w_need[i];
    want = max(want, w_want[i]);
    longest = max(longest, w_long[i]);
    bad |= w_bad[i];
    size += w_size[i];
  }
  int status = 0;
  const bool huge = size > 3e9f;
  if (head < 0 || huge || (long)head + all_need > a.nfree) status |= SJ_PLAN_NO_PAGES;
  if (want > (unsigned long)a.ldt) status |= SJ_PLAN_TABLE_WIDTH;
  if (huge || all_tok > a.cap) status |= SJ_PLAN_ROWS;
  if (bad) status |= SJ_PLAN_LENGTHS;
  const bool ok = status == 0;

  // the requests again with their places; a request's page ids are asked for
  // at once: that of the page it is in and the first that it takes
  const long t0 = (long)blockIdx.x * PTOK;
  uint32_t s = st - tok, f = sn - need;
  const bool lead = blockIdx.x == 0;
  auto mark = [&](int r, int n, int m) {
    if (lead) {
      a.starts[r] = ok ? (int)s : 0;
      if (a.after) a.after[r] = ok ? n + m : n;
    }
    if (!ok) return;
    const uint32_t in = div(n, a.d_page), have = pages_of(n), take = pages_of(n + m) - have;
    if (m > 0 && s < t0 + PTOK && (long)s + m > t0) {
      const int at = s > t0 ? (int)(s - t0) : 0;
      const int tail = in < have ? a.table[(long)r * a.ldt + in] : -1;
      const int fresh = take ? a.free_pages[head + f] : -1;
      h_req[at] = r;
      h_start[at] = (int)s;
      h_len[at] = n;
      h_first[at] = (int)f;
      h_tail[at] = tail;
      h_fresh[at] = fresh;
    }
    s += m;
    f += take;
  };
#pragma unroll
  for (int i = 0; i < HELD; i++)
    if (r0 + i < r1) mark(r0 + i, hn[i], hm[i]);
#pragma unroll 1
  for (int r = r0 + HELD; r < r1; r++) mark(r, a.lengths[r], a.counts[r]);
  if (lead && t == 0) {
    a.starts[a.R] = ok ? (int)all_tok : 0;
    a.summary[0] = ok ? (int)all_tok : 0;
    a.summary[1] = head + (ok ? (int)all_need : 0);
    a.summary[2] = status;
    a.summary[3] = (int)longest;
  }
  __syncthreads();
  // each token's request: the last mark at or before it (places from 1, 0: none)
  const int4 marks = *(const int4*)(h_req + 4 * t);
  int at[4];
  at[0] = marks.x >= 0 ? 4 * t + 1 : 0;
  at[1] = marks.y >= 0 ? 4 * t + 2 : at[0];
  at[2] = marks.z >= 0 ? 4 * t + 3 : at[1];
  at[3] = marks.w >= 0 ? 4 * t + 4 : at[2];
  const int upto = scan_max(at[3]);
  if (lane == 63) w_at[wave] = upto;
  int before = __shfl_up(upto, 1, 64);
  if (lane == 0) before = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 3; i++)
    if (i < wave) before = max(before, w_at[i]);
  int pos[4], slot[4], owner[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int h = max(at[i], before) - 1;
    const long g = t0 + 4 * t + i;
    pos[i] = slot[i] = owner[i] = -1;
    if (!ok || h < 0 || g >= (long)all_tok || g >= a.cap) continue;
    owner[i] = h_req[h];
    const int n = h_len[h];
    pos[i] = n + (int)(g - h_start[h]);
    const uint32_t col = div(pos[i], a.d_page), off = (uint32_t)pos[i] - col * a.P, have = pages_of(n);
    int page = h_tail[h];
    if (col >= have) {
      page = col == have ? h_fresh[h] : a.free_pages[(long)head + h_first[h] + (col - have)];
      if (off == 0) a.table[(long)owner[i] * a.ldt + col] = page;  // a fresh page's first position is a new token
    }
    if (page >= 0 && (uint32_t)page < a.pages) slot[i] = (int)((uint32_t)page * a.P + off);
  }
  const long g = t0 + 4 * t;
  if (g + 4 <= a.cap && ((((uintptr_t)a.positions | (uintptr_t)a.slots | (uintptr_t)a.owners) & 15) == 0)) {
    *(int4*)(a.positions + g) = make_int4(pos[0], pos[1], pos[2], pos[3]);
    *(int4*)(a.slots + g) = make_int4(slot[0], slot[1], slot[2], slot[3]);
    *(int4*)(a.owners + g) = make_int4(owner[0], owner[1], owner[2], owner[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (g + i < a.cap) {
        a.positions[g + i] = pos[i];
        a.slots[g + i] = slot[i];
        a.owners[g + i] = owner[i];
      }
  }
}
// -------------------------------------------------------------- attention
//
// The walks are in paged_walk.h.

constexpr int direct_waves(int dc) { return dc == 8 ? 4 : 8; }  // 256 registers a lane at most hold 8

// One workgroup per row, KV head and tile of 16 query heads: its waves take
// the key tiles in turn.  For walks that are short, and rows that are many.
template <typename T, int DC>
__global__ __launch_bounds__(64 * direct_waves(DC)) void k_paged_direct(PagedArgs a) {
  typedef Walk<T, DC> W;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ Shares sh;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6;
  const int nb = a.HK * a.QT, row = div(blockIdx.x, a.d_heads), hb = blockIdx.x - row * nb;
  const int kh = div(hb, a.d_tiles), qt = hb - kh * a.QT;
  int owner, lo, hi;
  if (!row_range(a, row, owner, lo, hi)) return;
  W wk;
  wk.start(a, row, kh, qt, lane);
  const int tiles = tiles_of(hi - lo, W::KT), n = min(16, a.G - qt * 16);
  wk.run(a, a.table + (long)owner * a.ldt, kh, lo, hi, w, tiles, nw, (bf16_t*)(lds + w * W::LDS), lane);
  leave(wk, sh, lds, n, w, lane);
  __syncthreads();
  const int quads = a.D / 4;
  for (int u = threadIdx.x; u < n * quads; u += blockDim.x) {
    const int r = div(u, a.d_quads), d = 4 * (u - r * quads);
    put_result<T>(a, row, kh * a.G + qt * 16 + r, d, joined<T, DC, direct_waves(DC)>(a, sh, lds, nw, r, d));
  }
}

// Walks of any lengths: the tiles of all rows and heads in one line, four by
// four (one per wave), and every workgroup an equal piece of the line.  Each
// workgroup sums the rows' tiles itself (one block scan).  A walk that lies in
// one piece is written as it is; of a walk that is cut, each workgroup leaves
// its totals in the workspace, and the last (meet, lanes.h) joins them in the
// order of the keys.  A workgroup has at most two cut walks, the end of one
// and the beginning of another.  45 requests of 1 to 6000 keys, 4 KV heads of
// 64: 16.8 us, of which the walks are 6 (32 MB), the rows' sums before them 2.5
// and the meeting behind them 5; with the join as a launch of its own 16.7 and
// for one request of 1000 keys 11.6 against 10.4.
constexpr int STREAM_ROWS = 2048;
// Workgroups that 256 CUs hold at once (by registers), and the most there are.
// Three of heads of 33 to 64 a CU, though a lane then spills 2 (bf16) or 4
// (fp32) registers: us with 3 / 2, bf16 | fp32: 45 requests of 1 to 6000 keys
// 16.4 / 19.4 | 22.9 / 25.5, 64 x 4 of 4096 56.3 / 55.5 | 122 / 112, 64 x 8 of
// 8192 245 / 233 | 389 / 380.
constexpr int split_per_cu(int dc) { return dc == 8 ? 1 : dc == 2 || dc == 3 ? 3 : 2; }
constexpr int STREAM_GROUPS = 1024;

template <typename T, int DC>
__global__ __launch_bounds__(256, split_per_cu(DC)) void k_paged_split(PagedArgs a) {
  typedef Walk<T, DC> W;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ Shares sh;
  __shared__ int pre[STREAM_ROWS + 1], ws[4], complete;
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, nb = a.HK * a.QT;
  constexpr int MOST = STREAM_ROWS / 256;
  const int per = (a.rows + 255) / 256;
  int n[MOST], mine = 0;
#pragma unroll
  for (int i = 0; i < MOST; i++) {
    n[i] = 0;
    const int r = t * per + i;
    int owner, lo, hi;
    if (i < per && r < a.rows && row_range(a, r, owner, lo, hi))
      n[i] = max(1, tiles_of(hi - lo, 4 * W::KT));  // a row without keys is written too
    mine += n[i];
  }
  int at = (int)scan_add((uint32_t)mine);
  if (lane == 63) ws[w] = at;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 3; i++)
    if (i < w) at += ws[i];
  at -= mine;
#pragma unroll
  for (int i = 0; i < MOST; i++) {
    const int r = t * per + i;
    if (i < per && r < a.rows) {
      pre[r] = at;
      at += n[i];
    }
  }
  const int all = ws[0] + ws[1] + ws[2] + ws[3];
  const int total = all * nb, piece = (int)(((long)total + gridDim.x - 1) / gridDim.x);
  if (t == 0) pre[a.rows] = all;
  __syncthreads();
  if ((long)blockIdx.x * piece >= total) return;
  int x = blockIdx.x * piece;
  const int e = (int)min((long)total, (long)x + piece);
  W wk;
  while (x < e) {
    // the row that holds place x, the last whose places begin at or before
    // it: counted by 32s, then within
    const int y = div(x, a.d_heads);
    const int r32 = 32 * (__popcll(__ballot(32 * lane < a.rows && pre[min(32 * lane, a.rows)] <= y)) - 1);
    const int row = r32 + __popcll(__ballot(lane < 32 && r32 + lane < a.rows && pre[min(r32 + lane, a.rows)] <= y)) - 1;
    const int first = __builtin_amdgcn_readfirstlane(pre[row]);
    const int places = __builtin_amdgcn_readfirstlane(pre[row + 1]) - first;
    // the walk of the row's: fewer than 2^16, so the fp32 quotient is off by
    // one at most
    const int in = x - first * nb;
    int hb = (int)((float)in * __builtin_amdgcn_rcpf((float)places));
    hb -= in - hb * places < 0;
    hb += in - hb * places >= places;
    const int c0 = in - hb * places, c1 = min(places, c0 + e - x);
    const int kh = div(hb, a.d_tiles), qt = hb - kh * a.QT, nq = min(16, a.G - qt * 16);
    int owner, lo, hi;
    row_range(a, row, owner, lo, hi);
    owner = __builtin_amdgcn_readfirstlane(owner);
    wk.start(a, row, kh, qt, lane);
    wk.run(a, a.table + (long)owner * a.ldt, kh, lo, hi, 4 * c0 + w, min(4 * c1, tiles_of(hi - lo, W::KT)), 4,
           (bf16_t*)(lds + w * W::LDS), lane);
    leave(wk, sh, lds, nq, w, lane);
    __syncthreads();
    const int quads = a.D / 4, items = nq * quads, h0 = kh * a.G + qt * 16;
    if (c0 == 0 && c1 == places) {
      for (int u = t; u < items; u += 256) {
        const int r = div(u, a.d_quads), d = 4 * (u - r * quads);
        put_result<T>(a, row, h0 + r, d, joined<T, DC, 4>(a, sh, lds, 4, r, d));
      }
    } else {
      // part i of the walk is workgroup g0 + i's
      const int x0 = x - c0, g0 = x0 / piece, parts = (x0 + places - 1) / piece - g0 + 1;
      auto slot = [&](int i) { return a.part + (2L * (g0 + i) + (i == 0)) * a.slot; };
      float* s = slot(blockIdx.x - g0);
      for (int u = t; u < items; u += 256) {
        const int r = div(u, a.d_quads), q = u - r * quads;
        const Total v = joined<T, DC, 4>(a, sh, lds, 4, r, 4 * q);
        if (q == 0) part_put(s + 2 * r, v.M, v.L);
        part_put(s + 32 + 2 * u, v.s[0], v.s[1]);
        part_put(s + 32 + 2 * (items + u), v.s[2], v.s[3]);
      }
      auto flag = [&](int i) { return a.flag + 2L * (g0 + i) + (i == 0); };
      if (meet(flag, blockIdx.x - g0, parts, a.number, &complete)) {
        // fewer items than threads: groups of threads share the parts, and
        // join through LDS
        const int span = min(items, 256), groups = 256 / span, gr = t / span;
        f32x4* acc = (f32x4*)lds;             // [256], then their maxima and shares: within the first two waves' parts
        float2* ml = (float2*)(lds + 256 * 16);
        for (int u0 = 0; u0 < items; u0 += span) {
          const int u = u0 + t - gr * span, r = div(u, a.d_quads), q = u - r * quads;
          const bool live = gr < groups && u < items;
          Total v;
          constexpr int MANY = 8;  // parts asked for at once
          for (int i = gr; live && i < parts; i += MANY * groups) {
            float2 m[MANY], p0[MANY], p1[MANY];
#pragma unroll
            for (int k = 0; k < MANY; k++) {
              const float* p = slot(min(i + k * groups, parts - 1));
              m[k] = part_get(p + 2 * r);
              p0[k] = part_get(p + 32 + 2 * u);
              p1[k] = part_get(p + 32 + 2 * (items + u));
            }
#pragma unroll
            for (int k = 0; k < MANY; k++)
              v.add(m[k].x, i + k * groups < parts ? m[k].y : 0.f, f32x4{p0[k].x, p0[k].y, p1[k].x, p1[k].y}, a.scale);
          }
          if (groups > 1) {
            acc[t] = v.s;
            ml[t] = make_float2(v.M, v.L);
            __syncthreads();
            for (int i = 1; gr == 0 && i < groups; i++) v.add(ml[t + i * span].x, ml[t + i * span].y, acc[t + i * span], a.scale);
          }
          if (live && gr == 0) put_result<T>(a, row, h0 + r, 4 * q, v);
        }
      }
    }
    __syncthreads();  // the next walk's waves write where this one was read
    x += c1 - c0;
  }
}

// Heads that are no whole 16-byte chunks: one workgroup per row and query
// head.  A lane owns a key in the products with q and columns lane + 64 c in
// the sums over v.  Bound by that: a group's keys are read once per query head,
// element by element, the values' keys one after another, and a long walk is
// not cut.  64 requests of 2048 keys, 16/4 heads, bf16: heads of 20 210 us (of
// 32, above, 26), of 36 226 (of 64 33); one request of 8192 469 and 818 (12).
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
      const int col = div((int)j, a.d_page), pg = pages[col];
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
  a.R = (int)requests; a.P = (int)page_size; a.pages = (uint32_t)pages;
  a.d_page = make_div((uint32_t)page_size);
  const long blocks = capacity > PTOK ? (capacity + PTOK - 1) / PTOK : 1;
  k_paged_plan<<<(unsigned)blocks, PT, 0, (hipStream_t)stream>>>(a);
  SJ_LAUNCH_CHECK("paged plan");
  return SJ_OK;
}

namespace {

// whether sj_paged_attention may split: by sizes alone, so that the workspace
// query knows it too
bool split_ok(long rows, long head_dim) { return rows <= STREAM_ROWS && head_dim % 4 == 0; }
long slot_floats(long g, long head_dim) { return 32 + (g < 16 ? g : 16) * head_dim; }

// f(Walk<T, DC>) for the head's width
template <typename T, class F>
void by_width(long D, F f) {
  if (D <= 32) f(Walk<T, 1>());
  else if (D <= 64) f(Walk<T, 2>());
  else if (D <= 96 && sizeof(T) == 2) f(Walk<T, sizeof(T) == 2 ? 3 : 4>());
  else if (D <= 128) f(Walk<T, 4>());
  else f(Walk<T, 8>());
}
template <typename T, int DC>
int launch_direct(hipStream_t s, const PagedArgs& a, int waves, Walk<T, DC>) {
  static sj::OncePerDevice once;
  if (int st = sjh::once_per_device(once, [] {
        SJ_HIP(hipFuncSetAttribute((const void*)k_paged_direct<T, DC>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                   direct_waves(DC) * Walk<T, DC>::LDS));
        return SJ_OK;
      }))
    return st;
  waves = waves < direct_waves(DC) ? waves : direct_waves(DC);
  k_paged_direct<T, DC><<<(unsigned)((long)a.rows * a.HK * a.QT), 64 * waves, waves * Walk<T, DC>::LDS, s>>>(a);
  return SJ_OK;
}
template <typename T, int DC>
int launch_split(hipStream_t s, const PagedArgs& a, long most, Walk<T, DC>) {
  static sj::OncePerDevice once;
  if (int st = sjh::once_per_device(once, [] {
        SJ_HIP(hipFuncSetAttribute((const void*)k_paged_split<T, DC>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                   4 * Walk<T, DC>::LDS));
        return SJ_OK;
      }))
    return st;
  // A short line of places (at the most that the tables hold) goes over as many
  // workgroups as the chip holds at once, so that none begins behind another;
  // a long one over more of them, so that they end together
  constexpr int at_once = 256 * split_per_cu(DC);
  const long places = (long)a.rows * a.HK * a.QT * ((most + 4 * Walk<T, DC>::KT - 1) / (4 * Walk<T, DC>::KT));
  k_paged_split<T, DC><<<places < 8 * at_once ? at_once : STREAM_GROUPS, 256, 4 * Walk<T, DC>::LDS, s>>>(a);
  return SJ_OK;
}

template <typename T>
int attend(hipStream_t s, PagedArgs& a, long most, void* workspace) {
  if (a.D % (16 / (int)sizeof(T))) {
    k_paged_rows<T><<<dim3((unsigned)a.rows, (unsigned)a.HQ), 256, 0, s>>>(a);
    return SJ_OK;
  }
  const long units = (long)a.rows * a.HK * a.QT;
  int st = SJ_OK;
  bool direct = !split_ok(a.rows, a.D) || (most / 16 + 1) * units > 0x7fffffffL;
  by_width<T>(a.D, [&](auto w) {
    const long tiles = (most + decltype(w)::KT - 1) / decltype(w)::KT;
    // The direct form, which sums no rows and joins in LDS alone, where a wave
    // has one tile, and where the workgroups are many and the tables not wide.
    // us, direct / split, bf16, requests x KV heads of L keys each | of 1 to L
    // keys, in tables of L:
    //   heads of 64        1 x 2  512    7.7 / 10.2 |
    //                      1 x 2  1024  11.6 / 10.6 |
    //     (16 tiles)      64 x 2  1024  12.6 / 14.0 | 11.2 / 10.6
    //                     64 x 2  2048  21.5 / 20.5 | 18.6 / 10.8
    //                     64 x 4  1024  15.7 / 19.8 | 11.3 / 12.4
    //                     64 x 4  2048  26.6 / 32.8 | 19.1 / 13.3
    //                     64 x 8  2048  50.3 / 59.2 | 28.6 / 19.2
    //     (64 tiles)      64 x 8  4096   119 / 128  | 44.0 / 25.5
    //                     64 x 8  8192   235 / 245  | 74.0 / 33.0
    //                    128 x 8  4096   233 / 236  | 69.5 / 40.8
    //     (16 tiles)     256 x 8  1024   120 / 115  | 29.8 / 37.3
    //                    256 x 8  2048   234 / 215  | 46.1 / 45.8
    //   heads of 128      64 x 8  1024  47.9 / 55.0 | 27.7 / 24.3
    //     (64 tiles)      64 x 8  2048   107 / 111  | 43.6 / 27.8
    //                     64 x 8  4096   205 / 204  | 72.4 / 38.8
    // From 17 to 64 tiles the rule takes up to a sixth off requests of one
    // length and costs very uneven ones up to 1.7 times the split form's time:
    // the lengths, which would tell them apart, are on the device.
    direct = direct || tiles <= 8 || (units >= 128 && tiles <= 16) || (units >= 512 && units < 2048 && tiles <= 64);
    if (direct) st = launch_direct(s, a, tiles <= 4 || units >= 1024 ? 4 : 8, w);
  });
  if (direct) return st;
  a.slot = (int)slot_floats(a.G, a.D);
  a.flag = (unsigned long long*)workspace;
  a.part = (float*)((uint8_t*)workspace + 16 * STREAM_GROUPS);
  a.number = sjh::call_number();
  by_width<T>(a.D, [&](auto w) { st = launch_split(s, a, most, w); });
  return st;
}

}  // namespace

extern "C" size_t sj_paged_attention_workspace_bytes(long rows, long hq, long hk, long head_dim) {
  if (rows <= 0 || hq <= 0 || hk <= 0 || head_dim <= 0 || hq % hk || !split_ok(rows, head_dim)) return 0;
  return 16 * STREAM_GROUPS + 2 * STREAM_GROUPS * (size_t)slot_floats(hq / hk, head_dim) * sizeof(float);
}

int sjh::paged_args(const void* q, long ldq, const void* k_cache, const void* v_cache, long ldkv, int dtype, long pages,
                    long page_size, const int32_t* table, long ldt, long requests, const int32_t* owners,
                    const int32_t* positions, long rows, long hq, long hk, long head_dim, long window, void* o, long ldo,
                    float* lse, PagedArgs& a) {
  SJ_REQUIRE(dtype == SJ_F32 || dtype == SJ_BF16, "paged attention dtype %d", dtype);
  SJ_REQUIRE(rows >= 0 && rows <= 0x7fffffffL && requests >= 0 && requests <= 0x7fffffffL && hq > 0 && hk > 0 &&
                 hq % hk == 0 && hq <= 65535 && head_dim > 0 && head_dim <= 256 && window >= 0 &&
                 ldq >= hq * head_dim && ldo >= hq * head_dim && ldkv >= hk * head_dim,
             "paged attention sequence/head dimensions");
  SJ_REQUIRE(page_size > 0 && page_size <= 0x7fffffffL && pages > 0 && pages <= 0x7fffffffL / page_size && ldt > 0 &&
                 ldt <= 0x7fffffffL / page_size,
             "paged attention: %ld pages of %ld, tables of %ld", pages, page_size, ldt);
  SJ_REQUIRE(owners || rows <= requests, "paged attention: %ld rows of %ld requests without owners", rows, requests);
  a = PagedArgs{};
  if (rows == 0 || requests == 0) return SJ_OK;
  SJ_REQUIRE(q && k_cache && v_cache && table && positions && o, "paged attention: null");
  SJ_REQUIRE(q != o || ldq == ldo || rows == 1, "paged attention: in place with strides %ld and %ld", ldq, ldo);
  a.q = q; a.ldq = ldq; a.k = k_cache; a.v = v_cache; a.ldkv = ldkv;
  a.table = table; a.ldt = ldt; a.owners = owners; a.positions = positions;
  a.o = o; a.ldo = ldo; a.lse = lse;
  a.requests = (int)requests; a.rows = (int)rows; a.HQ = (int)hq; a.HK = (int)hk; a.D = (int)head_dim;
  a.pages = (int)pages; a.P = (int)page_size; a.window = window;
  a.scale = (float)(1.4426950408889634 / sqrt((double)head_dim));
  a.G = (int)(hq / hk);
  a.QT = (a.G + 15) / 16;
  SJ_REQUIRE(rows <= (1L << 23) / (hk * a.QT), "paged attention: %ld rows of %ld heads", rows, hk);
  a.d_page = make_div((uint32_t)page_size);
  a.d_heads = make_div((uint32_t)(hk * a.QT));
  a.d_tiles = make_div((uint32_t)a.QT);
  a.d_quads = make_div((uint32_t)(head_dim / 4 > 0 ? head_dim / 4 : 1));
  return SJ_OK;
}

extern "C" int sj_paged_attention(void* stream, const void* q, long ldq, const void* k_cache, const void* v_cache,
                                  long ldkv, int dtype, long pages, long page_size, const int32_t* table, long ldt,
                                  long requests, const int32_t* owners, const int32_t* positions, long rows, long hq,
                                  long hk, long head_dim, long window, void* o, long ldo, float* lse, void* workspace,
                                  size_t workspace_bytes) {
  PagedArgs a;
  if (int st = sjh::paged_args(q, ldq, k_cache, v_cache, ldkv, dtype, pages, page_size, table, ldt, requests, owners,
                               positions, rows, hq, hk, head_dim, window, o, ldo, lse, a))
    return st;
  if (a.rows == 0) return SJ_OK;
  const size_t need = sj_paged_attention_workspace_bytes(rows, hq, hk, head_dim);
  SJ_REQUIRE(((uintptr_t)workspace & 15) == 0, "paged attention: the workspace is not 16-byte aligned");
  if (need > workspace_bytes || (need && !workspace))
    return sjh::fail(SJ_ERR_CAPACITY, "paged attention workspace: required %zu bytes, available %zu bytes", need,
                     workspace ? workspace_bytes : 0);
  long most = ldt * page_size;
  if (window > 0 && window < most) most = window;
  hipStream_t s = (hipStream_t)stream;
  if (int st = dtype == SJ_BF16 ? attend<bf16_t>(s, a, most, workspace) : attend<float>(s, a, most, workspace)) return st;
  SJ_LAUNCH_CHECK("paged attention");
  return SJ_OK;
}
