// Log probabilities of given tokens with the row's entropy and its most
// likely alternatives, and their gradient (no counterpart in the reference,
// whose cross_entropy, kernels.py:176-191, gives the loss alone).
//
//   m = max x,  rest = sum e^(x - m) without one of the terms that are 1
//   ln p_v = x_v - m - log1p(rest)
//   H = log1p(rest) - sum p_v (x_v - m)
//   dx_v = dlp (1[v = t] - p_v) - dH p_v (ln p_v + H)
//
// The sum leaves one largest term out, so that a peaked row keeps what it
// holds beside its peak (in fp32 1 + 1e-8 is 1, and the log 0).
#include "order.h"

using namespace sj;

namespace {

// One read of the row.  A group of threads (a wave, or a workgroup) holds a
// slice of it in registers: the maximum, then the sums relative to it.  Where
// the sum of all terms is 2 or more, taking the 1 off loses nothing; where it
// is less, the thread that holds the maximum sums again without it.
// The alternatives come from a threshold: the k-th largest of 64 or 256 column
// maxima (disjoint sets of entries) has at least k entries at or above it and
// rarely many more; those are collected in LDS and each finds its place by
// counting the larger ones.  Rows longer than a slice are joined from the
// slices' sums and lists: by the last of their workgroups up to 1024 slices, by
// a second launch where they are more.  us, meeting / second launch: 32 rows of
// 50001 fp32 7.2 / 8.0, with 20 alternatives of 131072 14.0 / 14.1; 1024 slices
// (512 rows of 16384) 11.8 / 12.2; 1792 (256 of 50008) 17.2 / 15.3.
// The bound is the read, and where an entry has 2 bytes the vector units: 7
// operations per entry, one of them an exponential, and per slice, whatever it
// holds, 245 a wave, with 240 more for 8 alternatives (threshold, and the two
// walks that count and place), 530 for 32 and 1225 for 64.  2048 rows of 50001
// bf16, 8 alternatives, four slices of 49 entries a thread (810 operations a
// wave), by the kernel trace: forward 70 us (2.9 TB/s) and join 8, gradient 79
// (5.2 TB/s, a copy's rate); a pass of the three 148.  1024 rows of 131072 fp32
// 97 us (5.5 TB/s).  2048 rows with 8 / 32 / 64 alternatives, us: bf16 of 32000
// 42 / 49 / 70, of 131072 125 / 152 / 216 (at a copy's rate 26 and 105); fp32 of
// 131072 191 / 224 / 325 (211).

constexpr int CAP_SLICE = 1024;  // entries at or above the threshold that LDS holds of a slice
constexpr int SLICE = 8192;      // entries of a slice; twice as many where slices of bf16 are many

struct ScoreArgs {
  const void* x;
  long ldx;
  long rows;
  int V, top, slices, width;  // width: entries of a slice, a multiple of 8
  const int32_t* tokens;
  float *logprob, *entropy, *stats;
  int32_t* ids;
  float* alt;
  u64* flag;      // [rows][slices], of the meetings
  u64 number;
  float* sums;    // [rows][slices] of (m, rest, xs, -)
  u64* keys;      // [rows][slices][top]
};
__device__ __forceinline__ float* part_sums(const ScoreArgs& a, long row) {
  return a.sums + row * a.slices * 4;
}
__device__ __forceinline__ u64* part_keys(const ScoreArgs& a, long row) {
  return a.keys + row * a.slices * a.top;
}

// what every thread of a row's group knows of its token, asked for early
struct Token {
  bool scored;
  float y;
};
template <typename T>
__device__ __forceinline__ Token token_of(const ScoreArgs& a, long row) {
  const int tk = a.tokens ? a.tokens[row] : -1;
  const bool scored = tk >= 0 && tk < a.V;
  return Token{scored, scored ? at_f32((const T*)a.x + row * a.ldx, tk) : 0.f};
}
// a row's numbers from its maximum, rest and xs = sum e^(x - m) (x - m)
__device__ __forceinline__ float write_row(const ScoreArgs& a, long row, float m, float rest, float xs, const Token& tk,
                                           float& ref, bool lead) {
  const bool none = m == -INFINITY && !(rest != rest);
  ref = m == -INFINITY ? 0.f : m;
  const float ll = none ? 0.f : log1pf(rest);
  if (lead) {
    if (a.logprob) a.logprob[row] = tk.scored ? tk.y - ref - ll : 0.f;
    if (a.entropy) a.entropy[row] = none ? 0.f : ll - xs / (1.f + rest);
    if (a.stats) a.stats[2 * row] = ref, a.stats[2 * row + 1] = ll;
  }
  return ll;
}
__device__ __forceinline__ void write_alternative(const ScoreArgs& a, long row, int place, u64 k, float ref, float ll) {
  a.ids[row * a.top + place] = key_index(k);
  a.alt[row * a.top + place] = key_value(k) - ref - ll;
}

// The slices of a row, by one workgroup: the sums relative to the row's
// maximum (slice s holds e^(m_s - m) (1 + rest_s) of them), and the largest of
// the slices' lists.  MEET: the slices were written by workgroups of this
// launch.
struct JoinShared {
  u64 cand[CAP_SLICE], key[64], last[4];
  float max[4], sum[2][4];
  int n, first;
};
template <bool MEET>
__device__ __forceinline__ void join_row(const ScoreArgs& a, int row, const Token& tk, JoinShared& sh) {
  constexpr int CAP = CAP_SLICE;
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  const int S = a.slices, top = a.top, all = S * top;
  const float* sums = part_sums(a, row);
  const u64* keys = part_keys(a, row);
  auto key = [&](int i) { return MEET ? part_get(keys + i) : keys[i]; };
  auto sum_of = [&](int s) {
    if (!MEET) return *(const f32x4*)(sums + 4 * s);
    const float2 p = part_get(sums + 4 * s), q = part_get(sums + 4 * s + 2);
    return f32x4{p.x, p.y, q.x, q.y};
  };
  constexpr int HELD = 4;  // keys a thread keeps from the first look at them
  u64 k[HELD];
#pragma unroll
  for (int i = 0; i < HELD; i++) k[i] = t + 256 * i < all ? key(t + 256 * i) : 0;
  const f32x4 mine = t < S ? sum_of(t) : f32x4{-INFINITY, 0.f, 0.f, 0.f};
  // The threshold: of the slices' j-th keys the i-th largest, i j >= top, has
  // i slices with j keys each at or above it (64 lanes take the slices in
  // turn and keep their largest)
  const int lanes = min(S, 64), j = min(top, 2 * ((top + lanes - 1) / lanes)), i = top ? (top + j - 1) / j : 0;
  u64 col = 0;
  if (w == 0 && top)
    for (int s = lane; s < S; s += 64) col = larger_of(col, key(s * top + j - 1));
  float m = mine[0];
  for (int s = t + 256; s < S; s += 256) m = fmaxf(m, sum_of(s)[0]);
  if (t == 0) sh.n = 0, sh.first = 0x7fffffff;
  m = all_max(m);
  if (lane == 0) sh.max[w] = m;
  if (w == 0) sh.key[lane] = col;
  __syncthreads();
  m = fmaxf(fmaxf(sh.max[0], sh.max[1]), fmaxf(sh.max[2], sh.max[3]));
  u64 T0 = 1;  // fewer than i slices with j keys: every key counts
  if (top) {
    const u64 mine = sh.key[lane];
    int larger = 0;
    for (int c = 0; c < lanes; c++) larger += sh.key[c] > mine;
    const u64 at = __ballot(mine && larger == i - 1);
    if (at) T0 = sh.key[__ffsll(at) - 1];
  }
  if (t < S && mine[0] == m) atomicMin(&sh.first, t);  // the slice that leaves its maximum out
  for (int s = t + 256; s < S; s += 256)
    if (sum_of(s)[0] == m) atomicMin(&sh.first, s);
  auto collect = [&](u64 key) {
    if (key >= T0) {
      const int n = atomicAdd(&sh.n, 1);
      if (n < CAP) sh.cand[n] = key;
    }
  };
#pragma unroll
  for (int i = 0; i < HELD; i++) collect(k[i]);
  for (int i = t + 256 * HELD; i < all; i += 256) collect(key(i));
  __syncthreads();
  const float ref0 = m == -INFINITY ? 0.f : m;
  float rest = 0.f, xs = 0.f;
  auto add = [&](int s, const f32x4& q) {
    if (s == sh.first || q[0] == -INFINITY) {  // without an entry of its own there is nothing to leave out
      rest += q[1];
      xs += q[2];
    } else {
      const float d = q[0] - ref0, f = __builtin_amdgcn_exp2f(d * LOG2E);
      rest += f * (1.f + q[1]);
      xs += f > 0.f ? f * fmaf(d, 1.f + q[1], q[2]) : f;
    }
  };
  if (t < S) add(t, mine);
  for (int s = t + 256; s < S; s += 256) add(s, sum_of(s));
  rest = all_sum(rest);
  xs = all_sum(xs);
  if (lane == 0) sh.sum[0][w] = rest, sh.sum[1][w] = xs;
  __syncthreads();
  rest = (sh.sum[0][0] + sh.sum[0][1]) + (sh.sum[0][2] + sh.sum[0][3]);
  xs = (sh.sum[1][0] + sh.sum[1][1]) + (sh.sum[1][2] + sh.sum[1][3]);
  float ref;
  const float ll = write_row(a, row, m, rest, xs, tk, ref, t == 0);
  if (!top) return;
  const int n = sh.n;
  if (n <= CAP) {
    rank<256>(sh.cand, n, top, t, [&](int place, u64 k) { write_alternative(a, row, place, k, ref, ll); });
    return;
  }
  u64 last = ~0ull;
  for (int j = 0; j < top; j++) {
    u64 k0 = 0;
    for (int i = t; i < all; i += 256) {
      const u64 k = key(i);
      if (k < last && k > k0) k0 = k;
    }
    k0 = all_max(k0);
    __syncthreads();
    if (lane == 0) sh.last[w] = k0;
    __syncthreads();
    last = k0 = larger_of(larger_of(sh.last[0], sh.last[1]), larger_of(sh.last[2], sh.last[3]));
    if (t == 0) write_alternative(a, row, j, k0, ref, ll);
  }
}
template <typename T>
__global__ __launch_bounds__(256) void k_score_join(ScoreArgs a) {
  __shared__ JoinShared sh;
  join_row<false>(a, blockIdx.x, token_of<T>(a, blockIdx.x), sh);
}

// One wave per row (NT = 64) or one workgroup per slice (NT = 256); a thread
// holds EV entries, in units of E that interleave over the threads.  MEET: the
// last of a row's workgroups joins its slices.
template <typename T, int NT, int EV, int E = WIDE<T>, bool MEET = false>
__global__ __launch_bounds__(256) void k_score(ScoreArgs a) {
  typedef Unit<T, E> U;
  constexpr int NU = EV / E, NW = NT / 64, GROUPS = 256 / NT, CAP = NT == 64 ? 64 * EV : CAP_SLICE;
  __shared__ __attribute__((aligned(16))) float s_best[256];
  __shared__ u64 s_cand[GROUPS][CAP], s_last[4];
  __shared__ float s_max[4], s_sum[2][2][4], s_T[4];
  __shared__ int s_n[GROUPS];
  const int gt = threadIdx.x / NT, t = threadIdx.x % NT, lane = threadIdx.x & 63, w = t >> 6;
  auto sync = [] {
    if constexpr (NT == 64)
      sync_wave();
    else
      __syncthreads();
  };
  const int g = blockIdx.x * GROUPS + gt;
  const int row = NT == 64 ? g : g / a.slices;
  if (row >= a.rows) return;  // a whole wave, or nobody
  const int slice = NT == 64 ? 0 : g - row * a.slices;
  const int base = slice * a.width, end = min(a.V, base + a.width), top = a.top;
  const T* x = (const T*)a.x + (long)row * a.ldx;
  auto index = [&](int i) { return base + E * (t + NT * (i / E)) + i % E; };
  U u[NU];
#pragma unroll
  for (int i = 0; i < NU; i++) {
    const int v = base + E * (t + NT * i);
    if (v + E <= end) u[i].r = *(const typename U::Raw*)(x + v);
  }
  const Token tk = token_of<T>(a, row);
  // units past the end are left out everywhere; one that crosses it is filled
  // with -inf
  constexpr int PART = 4, PARTS = EV / PART;  // maxima of parts: the search below passes those without
  float pm[PARTS], best = -INFINITY;
  auto f = [&](int i) { return u[i / E].get(i % E); };  // as stored: bf16 entries are widened at each use
#pragma unroll
  for (int i = 0; i < NU; i++) {
    const int v = base + E * (t + NT * i);
    if (v < end) {
      if (v + E > end) {
#pragma unroll
        for (int e = 0; e < E; e++) u[i].set(e, v + e < end ? at_f32(x, v + e) : -INFINITY);
      }
#pragma unroll
      for (int j = i * E / PART; j < (i + 1) * E / PART; j++) {
        pm[j] = fmaxf(fmaxf(f(PART * j), f(PART * j + 1)), fmaxf(f(PART * j + 2), f(PART * j + 3)));
        best = fmaxf(best, pm[j]);
      }
    }
  }
  float m = all_max(best);
  if (t == 0) s_n[gt] = 0;
  if (NT > 64) {
    s_best[threadIdx.x] = best;
    if (lane == 0) s_max[w] = m;
    sync();
    m = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
  }
  // The threshold.  Up to 32 alternatives by the first wave of the group from
  // 64 columns, for more of them by every wave from the threads' 256: the 64th
  // largest of 64 would be the least, with some 300 entries above it and at
  // times 1000 (2048 rows of 32000 bf16, 64 alternatives: 133 -> 74 us).
  if (top && (w == 0 || top > 32)) {
    const bool all = NT > 64 && top > 32;
    float col = best;
    if (NT > 64 && !all) col = fmaxf(fmaxf(best, s_best[lane + 64]), fmaxf(s_best[lane + 128], s_best[lane + 192]));
    float* cols = s_best + (NT > 64 ? 0 : gt * 64);
    if (!all) cols[lane] = col;
    sync_wave();
    int larger = 0;
    for (int j = 0; j < (all ? 256 : 64); j += 64)
#pragma unroll
      for (int i = 0; i < 64; i += 4) {
        const f32x4 c = *(const f32x4*)(cols + j + i);
        larger += (c[0] > col) + (c[1] > col) + (c[2] > col) + (c[3] > col);
      }
    const float least = all_min(larger < top ? col : INFINITY);
    if (NT == 64 ? lane == 0 : all ? lane == 0 : lane < 4) s_T[NT == 64 ? gt : all ? w : lane] = least;
  }
  const float ref = m == -INFINITY ? 0.f : m;
  float rest = 0.f, xs = 0.f;
  // Terms 2^(x log2e - c) with c = ref log2e rounded: one fused step and the
  // exponential.  c stands for a reference that is off by delta / log2e, known
  // exactly, so the sums come back to ref by one factor.
  const float c = ref * LOG2E, delta = fmaf(ref, LOG2E, -c);
#pragma unroll
  for (int i = 0; i < NU; i++) {
    const int v = base + E * (t + NT * i);
    if (v < end) {
      if (v + E > end && ref > -1e20f) {  // the filling: a share of 0 and no NaN
#pragma unroll
        for (int e = 0; e < E; e++)
          if (v + e >= end) u[i].set(e, -1e30f);
      }
#pragma unroll
      for (int e = 0; e < E; e++) {
        const float d = fmaf(f(i * E + e), LOG2E, -c), y = __builtin_amdgcn_exp2f(d);
        rest += y;
        xs = fmaf(y, d, xs);
      }
    }
  }
  const float back = __builtin_amdgcn_exp2f(-delta);
  rest *= back;
  xs = fmaf(xs * back, 0.6931471805599453f, -rest * (delta * 0.6931471805599453f));
  // The sums with the difference first, and without one entry that equals
  // `skip`: entries of -inf have a share of 0 and no entropy, a NaN stays
  auto slowly = [&](float skip) {
    rest = xs = 0.f;
    bool left = skip != skip;
#pragma unroll
    for (int i = 0; i < NU; i++)
      if (base + E * (t + NT * i) < end)
#pragma unroll
        for (int e = 0; e < E; e++) {
          const float y = f(i * E + e);
          const bool out = !left && y == skip;
          left |= out;
          const float d = y - ref, p = out ? 0.f : __builtin_amdgcn_exp2f(d * LOG2E);
          rest += p;
          xs = fmaf(p, fmaxf(d, -1e4f), xs);  // below -104 a share is 0
        }
  };
  // -inf or NaN among the entries, or a reference whose rounding leaves the
  // powers' range
  if (__any(!(fabsf(xs) < INFINITY)) || fabsf(ref) > 1e6f) slowly(NAN);
  auto total = [&](float& r, float& y, int k) {
    r = all_sum(r);
    y = all_sum(y);
    if (NT > 64) {
      if (lane == 0) s_sum[k][0][w] = r, s_sum[k][1][w] = y;
      sync();
      r = (s_sum[k][0][0] + s_sum[k][0][1]) + (s_sum[k][0][2] + s_sum[k][0][3]);
      y = (s_sum[k][1][0] + s_sum[k][1][1]) + (s_sum[k][1][2] + s_sum[k][1][3]);
    }
  };
  float l = rest, lx = xs;
  total(l, lx, 0);
  if (l < 2.f) {
    int first = 0;
    if (NT > 64) while (first < NW - 1 && s_max[first] != m) first++;
    const u64 mask = __ballot(best == m);
    if (w == first && mask && lane == __ffsll(mask) - 1) slowly(m);
    total(rest, xs, 1);
  } else {
    rest = l - 1.f;
    xs = lx;
  }
  const bool whole = NT == 64 || a.slices == 1;
  float ll = 0.f, rref = 0.f;
  if (whole) {
    ll = write_row(a, row, m, rest, xs, tk, rref, t == 0);
  } else if (t == 0) {
    float* p = part_sums(a, row) + 4 * slice;
    if constexpr (MEET)
      part_put(p, m, rest), part_put(p + 2, xs, 0.f);
    else
      *(f32x4*)p = f32x4{m, rest, xs, 0.f};
  }
  u64* list = whole ? nullptr : part_keys(a, row) + (long)slice * top;
  auto put = [&](int place, u64 k) {
    if (whole)
      write_alternative(a, row, place, k, rref, ll);
    else if constexpr (MEET)
      part_put(list + place, k);
    else
      list[place] = k;
  };
  auto done = [&] {
    if constexpr (MEET) {
      __shared__ JoinShared sh;
      __shared__ int complete;
      if (meet([&](int i) { return a.flag + (long)row * a.slices + i; }, slice, a.slices, a.number, &complete))
        join_row<true>(a, row, tk, sh);
    }
  };
  if (!top) return done();
  sync();
  const float T0 = NT == 64 ? s_T[gt] : fminf(fminf(s_T[0], s_T[1]), fminf(s_T[2], s_T[3]));
  // counted first, so that a wave takes its places in the list at once
  uint32_t mine = 0;
#pragma unroll
  for (int j = 0; j < PARTS; j++)
    if (index(PART * j) < end && pm[j] >= T0)
#pragma unroll
      for (int i = PART * j; i < PART * (j + 1); i++) mine += f(i) >= T0 && index(i) < end;
  const uint32_t upto = scan_add(mine);
  int from = 0;
  if (lane == 63 && upto) from = atomicAdd(&s_n[gt], (int)upto);
  from = __builtin_amdgcn_readlane(from, 63) + (int)(upto - mine);
#pragma unroll
  for (int j = 0; j < PARTS; j++)
    if (index(PART * j) < end && pm[j] >= T0) {
#pragma unroll
      for (int i = PART * j; i < PART * (j + 1); i++)
        if (f(i) >= T0 && index(i) < end) {
          if (from < CAP) s_cand[gt][from] = order_key(f(i), index(i));
          from++;
        }
    }
  sync();
  int n = s_n[gt];
  const int held = min(top, end - base);  // a row's last slice may have fewer entries
  if (n > CAP || n < held) {
    // many entries equal to the threshold (a masked row's -inf): those above
    // it, then the equal ones by windows of the index until there are enough
    sync();
    if (t == 0) s_n[gt] = 0;
    sync();
    auto collect = [&](int lo, int hi, bool equal) {
      for (int v = lo + t; v < hi; v += NT) {
        const float y = at_f32(x, v);
        if (equal ? y == T0 : y > T0) {
          const int k = atomicAdd(&s_n[gt], 1);
          if (k < CAP) s_cand[gt][k] = order_key(y, v);
        }
      }
      sync();
      n = s_n[gt];
      sync();
    };
    collect(base, end, false);
    for (int lo = base; n < held && lo < end; lo += CAP / 4) collect(lo, min(lo + CAP / 4, end), true);
  }
  if (n <= CAP && n >= held) {
    rank<NT>(s_cand[gt], n, top, t, put);
    for (int i = held + t; i < top; i += NT) put(i, 0);
    return done();
  }
  // more than LDS holds above the threshold, or fewer entries than asked for
  // beside NaN: the largest below the last, `top` times (then none, key 0)
  u64 last = ~0ull;
  for (int j = 0; j < top; j++) {
    u64 k0 = 0;
    for (int v = base + t; v < end; v += NT) {
      const u64 k = order_key(at_f32(x, v), v);
      if (k < last && k > k0) k0 = k;
    }
    k0 = all_max(k0);
    if (NT > 64) {
      sync();
      if (lane == 0) s_last[w] = k0;
      sync();
#pragma unroll
      for (int i = 0; i < NW; i++) k0 = s_last[i] > k0 ? s_last[i] : k0;
    }
    last = k0;
    if (t == 0) put(j, k0);
  }
  done();
}

struct ScoreBwdArgs {
  const void* x;
  long ldx, rows;
  int V, chunks;
  const int32_t* tokens;
  const float *stats, *entropy, *dlp, *dent;
  void* dx;
  long lddx;
};

// A wave takes 4 units of 16 bytes per lane of a row: read, and written once
template <typename T, typename O>
__global__ __launch_bounds__(256) void k_score_bwd(ScoreBwdArgs a) {
  typedef Unit<T, WIDE<T>> U;
  constexpr int E = U::E, NU = 4;
  const long wave = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const long row = wave / a.chunks;
  if (row >= a.rows) return;
  const int base = (int)(wave - row * a.chunks) * (64 * E * NU);
  const T* x = (const T*)a.x + row * a.ldx;
  O* dx = (O*)a.dx + row * a.lddx;
  U u[NU];
#pragma unroll
  for (int i = 0; i < NU; i++) {
    const int v = base + E * (lane + 64 * i);
    if (v + E <= a.V) u[i].r = *(const typename U::Raw*)(x + v);
  }
  const int tk = a.tokens ? a.tokens[row] : -1;
  const bool scored = tk >= 0 && tk < a.V;
  const float m = a.stats[2 * row], ll = a.stats[2 * row + 1], yt = scored ? at_f32(x, tk) : 0.f;
  const float dlp = a.dlp && scored ? a.dlp[row] : 0.f, dh = a.dent ? a.dent[row] : 0.f, H = a.dent ? a.entropy[row] : 0.f;
  auto grad = [&](float y) {
    const float lp = y - m - ll, p = __builtin_amdgcn_exp2f(lp * LOG2E);
    // a share of 0 (lp = -inf) has none of the entropy's part; a NaN is in p
    return -p * (dlp + dh * (fmaxf(lp, -1e4f) + H));
  };
#pragma unroll
  for (int i = 0; i < NU; i++) {
    const int v = base + E * (lane + 64 * i);
    if (v + E <= a.V) {
      float d[E];
#pragma unroll
      for (int e = 0; e < E; e++) d[e] = grad(u[i].get(e));
      if constexpr (sizeof(O) == 2) {
        struct __attribute__((packed, aligned(2))) P { uint32_t w[E / 2]; } o;
#pragma unroll
        for (int e = 0; e < E; e += 2) o.w[e / 2] = pack2(f2bf(d[e]), f2bf(d[e + 1]));
        *(P*)(dx + v) = o;
      } else {
        struct __attribute__((packed, aligned(4))) P { float w[E]; } o;
#pragma unroll
        for (int e = 0; e < E; e++) o.w[e] = d[e];
        *(P*)(dx + v) = o;
      }
    } else {
      for (int e = 0; e < E && v + e < a.V; e++) {
        const float d = grad(at_f32(x, v + e));
        if constexpr (sizeof(O) == 2) dx[v + e] = f2bf(d); else dx[v + e] = d;
      }
    }
  }
  // the token's own entry, 1 - p formed without losing a small remainder, by
  // the lane that wrote it
  const int mine = tk - base;
  if (scored && mine >= 0 && mine < 64 * E * NU && (mine / E) % 64 == lane) {
    const float lp = yt - m - ll, p = __builtin_amdgcn_exp2f(lp * LOG2E);
    const float d = fmaf(dlp, -expm1f(lp), -p * (dh * (fmaxf(lp, -1e4f) + H)));
    if constexpr (sizeof(O) == 2) dx[tk] = f2bf(d); else dx[tk] = d;
  }
}

// the slices of a row, at most: what the workspace holds
long slices_of(long vocab) { return (vocab + SLICE - 1) / SLICE; }

template <typename T>
void launch_score(hipStream_t s, ScoreArgs& a) {
  const unsigned waves = (unsigned)((a.rows + 3) / 4), rows = (unsigned)a.rows;
  a.slices = 1;
  a.width = (a.V + 7) / 8 * 8;
  if (a.V <= 512) {
    k_score<T, 64, 8, 4><<<waves, 256, 0, s>>>(a);  // units of 4: the columns of the threshold are alike
  } else if (a.V <= 1024) {
    k_score<T, 64, 16><<<waves, 256, 0, s>>>(a);
  } else if (a.V <= 4096) {
    k_score<T, 256, 16><<<rows, 256, 0, s>>>(a);
  } else {
    const bool few = a.V <= SLICE || a.rows * slices_of(a.V) <= 1024;
    // entries a thread holds of a long slice: 64 of fp32 leave 3 waves a SIMD
    // (2048 rows of 50008, 8 alternatives: 97 us, with 32 84); of bf16 1024
    // rows of 131072 take 65 us, with 32 72
    constexpr int LONG = sizeof(T) == 2 ? 64 : 32;
    const int most = few ? SLICE : 256 * LONG;
    a.slices = (a.V + most - 1) / most;
    a.width = ((a.V + a.slices - 1) / a.slices + 7) / 8 * 8;  // alike, so that they end together
    if (few && a.slices > 1) {
      a.number = sjh::call_number();
      k_score<T, 256, 32, WIDE<T>, true><<<rows * a.slices, 256, 0, s>>>(a);
    } else {
      if (few)
        k_score<T, 256, 32><<<rows, 256, 0, s>>>(a);
      else
        k_score<T, 256, LONG><<<rows * a.slices, 256, 0, s>>>(a);
      if (a.slices > 1) k_score_join<T><<<rows, 256, 0, s>>>(a);
    }
  }
}
template <typename T>
void launch_bwd(hipStream_t s, ScoreBwdArgs& a, int dx_dtype) {
  const int chunk = 64 * WIDE<T> * 4;
  a.chunks = (a.V + chunk - 1) / chunk;
  const unsigned blocks = (unsigned)((a.rows * a.chunks + 3) / 4);
  if (dx_dtype == SJ_BF16)
    k_score_bwd<T, bf16_t><<<blocks, 256, 0, s>>>(a);
  else
    k_score_bwd<T, float><<<blocks, 256, 0, s>>>(a);
}

}  // namespace

extern "C" size_t sj_token_logprobs_workspace_bytes(long rows, long vocab, long top) {
  if (rows <= 0 || vocab <= SLICE || top < 0) return 0;
  return (size_t)rows * slices_of(vocab) * (24 + 8 * (size_t)top);
}

extern "C" int sj_token_logprobs(void* stream, const void* x, int dtype, long ldx, long rows, long vocab,
                                 const int32_t* tokens, long top, float* logprob, float* entropy, float* stats,
                                 int32_t* top_ids, float* top_logprob, void* workspace, size_t workspace_bytes) {
  SJ_REQUIRE(dtype == SJ_F32 || dtype == SJ_BF16, "token log probabilities dtype %d", dtype);
  SJ_REQUIRE(rows >= 0 && rows <= 0x7fffffffL && vocab > 0 && vocab <= 1L << 24 && ldx >= vocab,
             "token log probabilities: %ld rows of %ld (stride %ld)", rows, vocab, ldx);
  SJ_REQUIRE(top >= 0 && top <= SJ_LOGPROBS_MAX_TOP && top <= vocab, "token log probabilities: %ld alternatives of %ld",
             top, vocab);
  SJ_REQUIRE(rows * slices_of(vocab) < 1L << 23, "token log probabilities: %ld rows of %ld", rows, vocab);
  if (rows == 0) return SJ_OK;
  SJ_REQUIRE(x && (logprob == nullptr || tokens) && (top == 0 || (top_ids && top_logprob)),
             "token log probabilities: null");
  const size_t need = sj_token_logprobs_workspace_bytes(rows, vocab, top);
  SJ_REQUIRE(((uintptr_t)workspace & 15) == 0, "token log probabilities: the workspace is not 16-byte aligned");
  if (need > workspace_bytes || (need && !workspace))
    return sjh::fail(SJ_ERR_CAPACITY, "token log probabilities workspace: required %zu bytes, available %zu bytes", need,
                     workspace ? workspace_bytes : 0);
  ScoreArgs a = {};
  a.x = x; a.ldx = ldx; a.rows = rows; a.V = (int)vocab; a.top = (int)top;
  a.tokens = tokens; a.logprob = logprob; a.entropy = entropy; a.stats = stats; a.ids = top_ids; a.alt = top_logprob;
  const size_t all = (size_t)rows * slices_of(vocab);
  a.sums = (float*)workspace;
  a.flag = (u64*)workspace + 2 * all;
  a.keys = a.flag + all;
  if (dtype == SJ_BF16)
    launch_score<bf16_t>((hipStream_t)stream, a);
  else
    launch_score<float>((hipStream_t)stream, a);
  SJ_LAUNCH_CHECK("token log probabilities");
  return SJ_OK;
}

extern "C" int sj_token_logprobs_bwd(void* stream, const void* x, int dtype, long ldx, long rows, long vocab,
                                     const int32_t* tokens, const float* stats, const float* entropy,
                                     const float* dlogprob, const float* dentropy, void* dx, int dx_dtype, long lddx) {
  SJ_REQUIRE((dtype == SJ_F32 || dtype == SJ_BF16) && (dx_dtype == SJ_F32 || dx_dtype == SJ_BF16),
             "token log probabilities backward dtypes %d, %d", dtype, dx_dtype);
  SJ_REQUIRE(rows >= 0 && rows <= 0x7fffffffL && vocab > 0 && vocab <= 1L << 24 && ldx >= vocab && lddx >= vocab,
             "token log probabilities backward: %ld rows of %ld (strides %ld, %ld)", rows, vocab, ldx, lddx);
  SJ_REQUIRE(rows * slices_of(vocab) < 1L << 23, "token log probabilities backward: %ld rows of %ld", rows, vocab);
  if (rows == 0) return SJ_OK;
  SJ_REQUIRE(x && stats && dx && (dlogprob == nullptr || tokens) && (dentropy == nullptr || entropy),
             "token log probabilities backward: null");
  SJ_REQUIRE(x != dx || (dtype == dx_dtype && (ldx == lddx || rows == 1)),
             "token log probabilities backward: in place with dtypes %d and %d, strides %ld and %ld", dtype, dx_dtype, ldx,
             lddx);
  ScoreBwdArgs a = {};
  a.x = x; a.ldx = ldx; a.rows = rows; a.V = (int)vocab; a.tokens = tokens; a.stats = stats; a.entropy = entropy;
  a.dlp = dlogprob; a.dent = dentropy; a.dx = dx; a.lddx = lddx;
  if (dtype == SJ_BF16)
    launch_bwd<bf16_t>((hipStream_t)stream, a, dx_dtype);
  else
    launch_bwd<float>((hipStream_t)stream, a, dx_dtype);
  SJ_LAUNCH_CHECK("token log probabilities backward");
  return SJ_OK;
}
