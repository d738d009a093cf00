// Attention over the pages of requests that share the beginning of their
// sequences: beams of one prompt, several answers to it, a long document that
// many ask about (no counterpart in the reference, whose cache holds one
// sequence: model lib.rs:36-50).
#include "paged_walk.h"

using namespace sj;

namespace {

//   o = (sum_shared + sum_own) / (l_shared + l_own), both relative to the
//   larger of the two maxima
//
// The keys that the rows of a group share are walked once for all of them: the
// query heads of a KV head of all the group's rows are columns, 32 of them a
// walk (two MFMA tiles on one key's loads).  Every row's own keys are a walk
// of their own, as in paged.hip.  All walks lie in one line of places (four
// key tiles, one per wave), and every workgroup takes an equal piece of it, so
// that few long prefixes and many short tails fill the chip alike.  What a
// workgroup summed of a walk goes to the workspace; a second launch joins the
// parts of each row's two walks.

constexpr int CT = 2, COLS = 16 * CT;
constexpr int MAX_ROWS = 2048, MAX_GROUPS = 1024;
constexpr int GROUPS_OF_WAVES = 1024;  // workgroups, at most

struct SharedArgs {
  PagedArgs p;
  const int32_t *starts, *group_starts, *prefix;
  int groups;
  Div d_group;  // by G
  // left for the join by the first workgroup
  int4* row_info;    // first own key, group (-1: alone), first place in units of the row's walks, places of a walk
  int4* group_info;  // [2 * groups]: first place, places of a walk, blocks of columns, first walk; first row, -, -, -
  int2* line;        // the places of the shared walks, a piece
  float *lead_part, *own_part;
  int lead_slot, own_slot;
};

// index of the last of n ascending values that is at or below y (v[0] is):
// counted by 16s or 32s, then within
template <int STEP>
__device__ __forceinline__ int last_at(const int* v, int n, int y, int lane) {
  const int far = STEP * lane;
  const int c = STEP * (__popcll(__ballot(far < n && v[min(far, n - 1)] <= y)) - 1);
  return c + __popcll(__ballot(lane < STEP && c + lane < n && v[min(c + lane, n - 1)] <= y)) - 1;
}

// workgroups a CU holds (by registers)
template <typename T>
constexpr int per_cu(int dc) { return dc == 8 || (dc == 4 && sizeof(T) == 4) ? 1 : 2; }

template <typename T, int DC>
__global__ __launch_bounds__(256, per_cu<T>(DC)) void k_shared_walks(SharedArgs s) {
  typedef Walk<T, DC, CT> WL;
  typedef Walk<T, DC> W;
  const PagedArgs& a = s.p;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ Shares sh;
  __shared__ int g_request[MAX_GROUPS + 1], g_row[MAX_GROUPS + 1], g_keys[MAX_GROUPS], g_pre[MAX_GROUPS + 1],
      g_walk[MAX_GROUPS + 1];
  __shared__ int pre[MAX_ROWS + 1], from[MAX_ROWS], ws[2][4];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, nb = a.HK * a.QT, ng = s.groups;
  const int most = (int)(a.ldt * a.P);
  constexpr int PLACE = 4 * W::KT, LEAD_PLACE = 4 * WL::KT;  // keys of a place

  // the groups: requests, rows and shared keys
  for (int g = t; g <= ng; g += 256) {
    const int r = min(max(s.group_starts[g], 0), a.requests);
    g_request[g] = r;
    g_row[g] = min(max(s.starts ? s.starts[r] : r, 0), a.rows);
    if (g < ng) g_keys[g] = s.prefix[g];
  }
  __syncthreads();
  bool descends = false;
  for (int g = t; g < ng; g += 256) descends |= g_request[g + 1] < g_request[g] || g_row[g + 1] < g_row[g];
  const bool none = __syncthreads_or(descends);  // no groups then: every row attends alone
  auto blocks_of = [&](int g) {
    const bool has = !none && g_keys[g] > 0 && g_keys[g] <= most;
    return has ? ((g_row[g + 1] - g_row[g]) * a.G + COLS - 1) / COLS : 0;
  };
  {
    constexpr int MOST = MAX_GROUPS / 256;
    const int per = (ng + 255) / 256;
    int places[MOST], walks[MOST], mine = 0, walk = 0;
#pragma unroll
    for (int i = 0; i < MOST; i++) {
      const int g = t * per + i;
      places[i] = walks[i] = 0;
      if (i < per && g < ng) {
        walks[i] = a.HK * blocks_of(g);
        places[i] = walks[i] * tiles_of(max(g_keys[g], 0), LEAD_PLACE);
      }
      mine += places[i];
      walk += walks[i];
    }
    int at = (int)scan_add((uint32_t)mine), at_walk = (int)scan_add((uint32_t)walk);
    if (lane == 63) ws[0][w] = at, ws[1][w] = at_walk;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; i++)
      if (i < w) at += ws[0][i], at_walk += ws[1][i];
    if (t == 255) g_pre[ng] = at, g_walk[ng] = at_walk;
    at -= mine;
    at_walk -= walk;
#pragma unroll
    for (int i = 0; i < MOST; i++) {
      const int g = t * per + i;
      if (i < per && g < ng) {
        g_pre[g] = at;
        g_walk[g] = at_walk;
        at += places[i];
        at_walk += walks[i];
      }
    }
    __syncthreads();
  }
  const int lead = g_pre[ng];

  // the rows: where their own keys begin
  {
    constexpr int MOST = MAX_ROWS / 256;
    const int per = (a.rows + 255) / 256;
    int n[MOST], group[MOST], mine = 0;
#pragma unroll
    for (int i = 0; i < MOST; i++) {
      n[i] = 0;
      group[i] = -1;
      const int r = t * per + i;
      int owner, lo, hi;
      if (i < per && r < a.rows && row_range(a, r, owner, lo, hi)) {
        if (lead > 0 && lo == 0) {
          int g = 0, e = ng;  // the last group that begins at or before the owner
          while (e - g > 1) {
            const int m = (g + e) >> 1;
            if (g_request[m] <= owner) g = m; else e = m;
          }
          // among groups without requests it is the last, the one that has them
          if (owner >= g_request[g] && owner < g_request[g + 1] && r >= g_row[g] && r < g_row[g + 1] && g_keys[g] > 0 &&
              g_keys[g] <= hi)
            group[i] = g, lo = g_keys[g];
        }
        from[r] = lo;
        n[i] = tiles_of(hi - lo, PLACE);
      }
      mine += n[i];
    }
    int at = (int)scan_add((uint32_t)mine);
    if (lane == 63) ws[0][w] = at;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; i++)
      if (i < w) at += ws[0][i];
    if (t == 255) pre[a.rows] = at;
    at -= mine;
#pragma unroll
    for (int i = 0; i < MOST; i++) {
      const int r = t * per + i;
      if (i < per && r < a.rows) {
        pre[r] = at;
        if (blockIdx.x == 0) s.row_info[r] = make_int4(from[r], group[i], at, n[i]);
        at += n[i];
      }
    }
    __syncthreads();
  }
  const int total = lead + pre[a.rows] * nb, piece = max(1, (int)(((long)total + gridDim.x - 1) / gridDim.x));
  if (blockIdx.x == 0) {
    for (int g = t; g < ng; g += 256) {
      s.group_info[2 * g] = make_int4(g_pre[g], tiles_of(max(g_keys[g], 0), LEAD_PLACE), blocks_of(g), g_walk[g]);
      s.group_info[2 * g + 1] = make_int4(g_row[g], 0, 0, 0);
    }
    if (t == 0) *s.line = make_int2(lead, piece);
  }
  // neighbours on the line on one XCD, where there is a piece for everybody:
  // the blocks of columns of one KV head walk the same keys
  const int b = piece > 1 ? (int)((blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3)) : (int)blockIdx.x;
  if ((long)b * piece >= total) return;
  int x = b * piece;
  const int e = (int)min((long)total, (long)x + piece);
  const int quads = a.D / 4;
  while (x < min(e, lead)) {
    const int g = __builtin_amdgcn_readfirstlane(last_at<16>(g_pre, ng, x, lane));
    const int keys = __builtin_amdgcn_readfirstlane(g_keys[g]), places = tiles_of(keys, LEAD_PLACE), in = x - g_pre[g];
    const int walk = __builtin_amdgcn_readfirstlane(in / places), c0 = in - walk * places, c1 = min(places, c0 + e - x);
    const int blocks = blocks_of(g), kh = walk / blocks, cb = walk - kh * blocks;
    const int r0 = g_row[g], cols = min((g_row[g + 1] - r0) * a.G - cb * COLS, COLS), nt = (cols + 15) / 16;
    WL wk;
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
      const int c = 16 * ct + (lane & 15), at = cb * COLS + c, row = div(at, s.d_group), h = at - row * a.G;
      wk.start(a, ct, (const T*)a.q + (long)(r0 + row) * a.ldq + ((long)kh * a.G + h) * a.D, c < cols, lane);
    }
    wk.run(a, a.table + (long)g_request[g] * a.ldt, kh, 0, keys, 4 * c0 + w, min(4 * c1, tiles_of(keys, WL::KT)), 4,
           (bf16_t*)(lds + w * WL::LDS), lane, nt);
    float* part = s.lead_part + (long)(g_walk[g] + walk + b) * s.lead_slot;
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
      if (ct >= nt) break;
      const int n = min(16, cols - 16 * ct);
      leave(wk, sh, lds, n, w, lane, ct);
      __syncthreads();
      for (int u = t; u < n * quads; u += 256) {
        const int r = div(u, a.d_quads), q = u - r * quads;
        const Total v = joined<T, DC, 4, CT>(a, sh, lds, 4, r, 4 * q);
        if (q == 0) *(float2*)(part + 2 * (16 * ct + r)) = make_float2(v.M, v.L);
        *(f32x4*)(part + 2 * COLS + (16 * ct + r) * a.D + 4 * q) = v.s;
      }
      __syncthreads();
    }
    x += c1 - c0;
  }
  while (x < e) {
    const int own = x - lead, y = div(own, a.d_heads);
    const int row = __builtin_amdgcn_readfirstlane(last_at<32>(pre, a.rows, y, lane));
    const int first = __builtin_amdgcn_readfirstlane(pre[row]), places = __builtin_amdgcn_readfirstlane(pre[row + 1]) - first;
    const int in = own - first * nb, hb = __builtin_amdgcn_readfirstlane(in / places);
    const int c0 = in - hb * places, c1 = min(places, c0 + e - x);
    const int kh = div(hb, a.d_tiles), qt = hb - kh * a.QT, n = min(16, a.G - qt * 16);
    int owner, lo, hi;
    row_range(a, row, owner, lo, hi);
    owner = __builtin_amdgcn_readfirstlane(owner);
    lo = __builtin_amdgcn_readfirstlane(from[row]);
    W wk;
    wk.start(a, row, kh, qt, lane);
    wk.run(a, a.table + (long)owner * a.ldt, kh, lo, hi, 4 * c0 + w, min(4 * c1, tiles_of(hi - lo, W::KT)), 4,
           (bf16_t*)(lds + w * W::LDS), lane);
    leave(wk, sh, lds, n, w, lane);
    __syncthreads();
    float* part = s.own_part + (long)(row * nb + hb + b) * s.own_slot;
    for (int u = t; u < n * quads; u += 256) {
      const int r = div(u, a.d_quads), q = u - r * quads;
      const Total v = joined<T, DC, 4>(a, sh, lds, 4, r, 4 * q);
      if (q == 0) *(float2*)(part + 2 * r) = make_float2(v.M, v.L);
      *(f32x4*)(part + 32 + r * a.D + 4 * q) = v.s;
    }
    __syncthreads();
    x += c1 - c0;
  }
}

// One workgroup per row, KV head and tile of 16 query heads: the parts of its
// shared walk and of its own, in the order of the line.  Groups of threads
// share the parts and join through LDS.
template <typename T>
__global__ __launch_bounds__(256) void k_shared_join(SharedArgs s) {
  const PagedArgs& a = s.p;
  __shared__ f32x4 acc[256];
  __shared__ float2 ml[256];
  const int nb = a.HK * a.QT, row = div(blockIdx.x, a.d_heads), hb = blockIdx.x - row * nb;
  const int kh = div(hb, a.d_tiles), qt = hb - kh * a.QT, n = min(16, a.G - qt * 16), quads = a.D / 4;
  int owner, lo, hi;
  if (!row_range(a, row, owner, lo, hi)) return;
  const int4 info = s.row_info[row];
  const int2 line = *s.line;
  const int lead = line.x, piece = line.y, g = info.y;
  int4 group = make_int4(0, 0, 0, 0);
  int r0 = 0;
  if (g >= 0) group = s.group_info[2 * g], r0 = s.group_info[2 * g + 1].x;
  const int items = n * quads, span = min(items, 256), shares = 256 / span, t = threadIdx.x, gr = t / span;
  for (int u0 = 0; u0 < items; u0 += span) {
    const int u = u0 + t - gr * span, r = div(min(u, items - 1), a.d_quads), q = min(u, items - 1) - r * quads;
    const bool live = gr < shares && u < items;
    Total v;
    auto add = [&](const float* base, long slot, int walk, int x0, int places, int c, int ncols) {
      if (places == 0) return;
      const int p0 = x0 / piece, parts = (x0 + places - 1) / piece - p0 + 1;
      for (int i = gr; i < parts; i += shares) {
        const float* p = base + (walk + p0 + i) * slot;
        const float2 m = *(const float2*)(p + 2 * c);
        v.add(m.x, m.y, *(const f32x4*)(p + 2 * ncols + c * a.D + 4 * q), a.scale);
      }
    };
    if (live) {
      if (g >= 0) {
        const int at = (row - r0) * a.G + qt * 16 + r, cb = at / COLS, walk = kh * group.z + cb;
        add(s.lead_part, s.lead_slot, group.w + walk, group.x + walk * group.y, group.y, at - cb * COLS, COLS);
      }
      add(s.own_part, s.own_slot, row * nb + hb, lead + info.z * nb + hb * info.w, info.w, r, 16);
    }
    if (shares > 1) {
      acc[t] = v.s;
      ml[t] = make_float2(v.M, v.L);
      __syncthreads();
      for (int i = 1; gr == 0 && i < shares; i++) v.add(ml[t + i * span].x, ml[t + i * span].y, acc[t + i * span], a.scale);
    }
    if (live && gr == 0) put_result<T>(a, row, kh * a.G + qt * 16 + r, 4 * q, v);
  }
}

struct Layout {
  size_t rows, groups, line, lead, own, bytes;
  long lead_slot, own_slot;
};
// sizes alone: the workspace query knows them too
Layout layout_of(long rows, long hq, long hk, long head_dim, long groups) {
  const long G = hq / hk, QT = (G + 15) / 16;
  Layout l = {};
  l.lead_slot = COLS * (2 + head_dim);
  l.own_slot = 32 + (G < 16 ? G : 16) * head_dim;
  l.groups = 16 * (size_t)rows;
  l.line = l.groups + 32 * (size_t)groups;
  l.lead = l.line + 16;
  // each group's last block of columns may hold fewer than COLS
  const size_t walks = (size_t)hk * (rows * G / COLS + groups);
  l.own = l.lead + 4 * (walks + GROUPS_OF_WAVES) * l.lead_slot;
  l.bytes = l.own + 4 * ((size_t)rows * hk * QT + GROUPS_OF_WAVES) * l.own_slot;
  return l;
}
// whether the prefixes are walked for their groups: by sizes alone, too
bool grouped(long rows, long head_dim, long groups) {
  return groups > 0 && groups <= MAX_GROUPS && rows <= MAX_ROWS && head_dim % 8 == 0;
}

template <typename T, int DC>
int launch_walks(hipStream_t st, const SharedArgs& s, Walk<T, DC>) {
  static sj::OncePerDevice once;
  if (int e = sjh::once_per_device(once, [] {
        SJ_HIP(hipFuncSetAttribute((const void*)k_shared_walks<T, DC>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                   4 * Walk<T, DC>::LDS));
        return SJ_OK;
      }))
    return e;
  k_shared_walks<T, DC><<<256 * per_cu<T>(DC), 256, 4 * Walk<T, DC>::LDS, st>>>(s);
  k_shared_join<T><<<(unsigned)((long)s.p.rows * s.p.HK * s.p.QT), 256, 0, st>>>(s);
  return SJ_OK;
}
template <typename T>
int launch(hipStream_t st, const SharedArgs& s) {
  const int D = s.p.D;
  if (D <= 32) return launch_walks(st, s, Walk<T, 1>());
  if (D <= 64) return launch_walks(st, s, Walk<T, 2>());
  if (D <= 96 && sizeof(T) == 2) return launch_walks(st, s, Walk<T, sizeof(T) == 2 ? 3 : 4>());
  if (D <= 128) return launch_walks(st, s, Walk<T, 4>());
  return launch_walks(st, s, Walk<T, 8>());
}

}  // namespace

extern "C" size_t sj_paged_attention_shared_workspace_bytes(long rows, long hq, long hk, long head_dim, long groups) {
  if (rows <= 0 || hq <= 0 || hk <= 0 || head_dim <= 0 || hq % hk) return 0;
  const size_t alone = sj_paged_attention_workspace_bytes(rows, hq, hk, head_dim);
  if (!grouped(rows, head_dim, groups)) return alone;
  const size_t together = layout_of(rows, hq, hk, head_dim, groups).bytes;
  return together > alone ? together : alone;
}

extern "C" int sj_paged_attention_shared(void* stream, const void* q, long ldq, const void* k_cache, const void* v_cache,
                                         long ldkv, int dtype, long pages, long page_size, const int32_t* table, long ldt,
                                         long requests, const int32_t* owners, const int32_t* positions, long rows,
                                         const int32_t* starts, const int32_t* group_starts, const int32_t* prefix,
                                         long groups, long hq, long hk, long head_dim, long window, void* o, long ldo,
                                         float* lse, void* workspace, size_t workspace_bytes) {
  SJ_REQUIRE(groups >= 0 && groups <= 1L << 24, "paged attention of groups: %ld groups", groups);
  SJ_REQUIRE(groups == 0 || (group_starts && prefix), "paged attention of groups: null");
  SharedArgs s = {};
  if (int st = sjh::paged_args(q, ldq, k_cache, v_cache, ldkv, dtype, pages, page_size, table, ldt, requests, owners,
                               positions, rows, hq, hk, head_dim, window, o, ldo, lse, s.p))
    return st;
  if (s.p.rows == 0) return SJ_OK;
  // all places of the line are counted in 31 bits
  const double places = ((double)rows * hk * (s.p.QT + s.p.G / (double)COLS) + (double)groups * hk) * (ldt * page_size / 64.0 + 1);
  if (!grouped(rows, head_dim, groups) || places >= 2147483647.0)
    return sj_paged_attention(stream, q, ldq, k_cache, v_cache, ldkv, dtype, pages, page_size, table, ldt, requests, owners,
                              positions, rows, hq, hk, head_dim, window, o, ldo, lse, workspace, workspace_bytes);
  const Layout l = layout_of(rows, hq, hk, head_dim, groups);
  const size_t need = sj_paged_attention_shared_workspace_bytes(rows, hq, hk, head_dim, groups);
  SJ_REQUIRE(((uintptr_t)workspace & 15) == 0, "paged attention of groups: the workspace is not 16-byte aligned");
  if (need > workspace_bytes || !workspace)
    return sjh::fail(SJ_ERR_CAPACITY, "paged attention of groups workspace: required %zu bytes, available %zu bytes", need,
                     workspace ? workspace_bytes : 0);
  s.starts = starts; s.group_starts = group_starts; s.prefix = prefix;
  s.groups = (int)groups;
  s.d_group = make_div((uint32_t)s.p.G);
  uint8_t* at = (uint8_t*)workspace;
  s.row_info = (int4*)at;
  s.group_info = (int4*)(at + l.groups);
  s.line = (int2*)(at + l.line);
  s.lead_part = (float*)(at + l.lead);
  s.own_part = (float*)(at + l.own);
  s.lead_slot = (int)l.lead_slot;
  s.own_slot = (int)l.own_slot;
  hipStream_t st = (hipStream_t)stream;
  if (int e = dtype == SJ_BF16 ? launch<bf16_t>(st, s) : launch<float>(st, s)) return e;
  SJ_LAUNCH_CHECK("paged attention of groups");
  return SJ_OK;
}
