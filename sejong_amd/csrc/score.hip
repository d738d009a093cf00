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
#include <math.h>

#include "common.h"

using namespace sj;

namespace {

// One read of the row.  A group of threads (a wave, or a workgroup) holds a
// slice of it in registers.  Each thread keeps its largest entry apart while
// it looks at its entries, so that the sums run over the others and the one
// term to leave out is known; then the sums relative to the group's maximum.
// The alternatives come from a threshold: the k-th largest of 64 column maxima
// (64 disjoint sets of entries) has at least k entries at or above it and
// rarely many more; those are collected in LDS and each finds its place by
// counting the larger ones.  Rows longer than a slice are joined from the
// slices' sums and lists by a second launch.
// The bound is the read: per entry there are about 14 operations, one of them
// an exponential.

constexpr float LOG2E = 1.4426950408889634f;
constexpr int CAP = 1024;   // entries at or above the threshold that LDS holds
constexpr int SLICE = 8192; // entries of a workgroup's slice

typedef unsigned long long u64;

// a wave's own exchange through LDS: its accesses are in order, the compiler
// must keep them so
__device__ __forceinline__ void sync_wave() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// the order of the alternatives: larger values first, NaN behind everything,
// the lowest index first among equals; a larger key comes first, and no two
// entries of a row have the same
__device__ __forceinline__ u64 order_key(float x, int v) {
  uint32_t b = __float_as_uint(x + 0.f);  // -0 is 0
  b = x != x ? 0u : (b >> 31) ? ~b : (b | 0x80000000u);
  return ((u64)b << 32) | (uint32_t)(0x7fffffff - v);
}
__device__ __forceinline__ int key_index(u64 k) { return 0x7fffffff - (int)(uint32_t)k; }
// the value again; a NaN's place and no entry at all give -inf
__device__ __forceinline__ float key_value(u64 k) {
  const uint32_t b = (uint32_t)(k >> 32);
  return b == 0u ? -INFINITY : __uint_as_float((b >> 31) ? b ^ 0x80000000u : ~b);
}

// E entries at any element alignment, as fp32
template <typename T>
struct Unit;
template <>
struct Unit<float> {
  static constexpr int E = 4;
  struct __attribute__((packed, aligned(4))) Raw { float v[4]; } r;
  __device__ __forceinline__ float get(int i) const { return r.v[i]; }
};
template <>
struct Unit<bf16_t> {
  static constexpr int E = 8;
  struct __attribute__((packed, aligned(2))) Raw { u32x4 v; } r;
  __device__ __forceinline__ float get(int i) const {
    const uint32_t w = r.v[i >> 1];
    return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
  }
};
__device__ __forceinline__ float at_f32(const float* x, long i) { return x[i]; }
__device__ __forceinline__ float at_f32(const bf16_t* x, long i) { return bf2f(x[i]); }

struct ScoreArgs {
  const void* x;
  long ldx;
  long rows;
  int V, top, slices;
  const int32_t* tokens;
  float *logprob, *entropy, *stats;
  int32_t* ids;
  float* alt;
  uint8_t* part;  // per row and slice: rest, xs, the largest key, then `top` keys
};
__device__ __forceinline__ float* part_at(const ScoreArgs& a, long row, int slice) {
  return (float*)(a.part + (row * a.slices + slice) * (16 + 8L * a.top));
}

// a row's numbers from its maximum, rest and xs = sum e^(x - m) (x - m)
template <typename T>
__device__ __forceinline__ float write_row(const ScoreArgs& a, long row, float m, float rest, float xs, float& ref,
                                           bool lead) {
  const bool none = m == -INFINITY && !(rest != rest);
  ref = m == -INFINITY ? 0.f : m;
  const float ll = none ? 0.f : log1pf(rest);
  if (lead) {
    const int tk = a.tokens ? a.tokens[row] : -1;
    if (a.logprob) a.logprob[row] = tk >= 0 && tk < a.V ? at_f32((const T*)a.x + row * a.ldx, tk) - ref - ll : 0.f;
    if (a.entropy) a.entropy[row] = none ? 0.f : ll - xs / (1.f + rest);
    if (a.stats) a.stats[2 * row] = ref, a.stats[2 * row + 1] = ll;
  }
  return ll;
}

// One wave per row (NT = 64) or one workgroup per slice (NT = 256); a thread
// holds EV entries, in units of 16 bytes that interleave over the threads.
template <typename T, int NT, int EV>
__global__ __launch_bounds__(256) void k_score(ScoreArgs a) {
  typedef Unit<T> U;
  constexpr int E = U::E, NU = EV / E, NW = NT / 64, GROUPS = 256 / NT;
  __shared__ u64 s_key[256], s_cand[GROUPS][CAP], s_red[4], s_T[GROUPS];
  __shared__ float s_sum[2][4];
  __shared__ int s_n[GROUPS];
  const int gt = threadIdx.x / NT, t = threadIdx.x % NT, lane = threadIdx.x & 63, w = t >> 6;
  auto sync = [] {
    if constexpr (NT == 64)
      sync_wave();
    else
      __syncthreads();
  };
  const long g = (long)blockIdx.x * GROUPS + gt;
  const long row = NT == 64 ? g : g / a.slices;
  if (row >= a.rows) return;  // a whole wave, or nobody
  const int slice = NT == 64 ? 0 : (int)(g - row * a.slices);
  const int base = slice * (NT * EV), end = min(a.V, base + NT * EV);
  const T* x = (const T*)a.x + row * a.ldx;
  U u[NU];
  float f[EV];
#pragma unroll
  for (int i = 0; i < NU; i++) {
    const int v = base + E * (t + NT * i);
    if (v + E <= end) u[i].r = *(const typename U::Raw*)(x + v);
  }
  // the largest entry apart (the lowest index of it), the others in f
  float best = -INFINITY;
  int at = -1;
#pragma unroll
  for (int i = 0; i < NU; i++) {
    const int v = base + E * (t + NT * i);
    if (v + E <= end) {
#pragma unroll
      for (int e = 0; e < E; e++) {
        const float y = u[i].get(e);
        const bool up = y > best;
        f[i * E + e] = up ? best : y;
        at = up ? v + e : at;
        best = up ? y : best;
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; e++) {
        const float y = v + e < end ? at_f32(x, v + e) : -INFINITY;
        const bool up = y > best;
        f[i * E + e] = up ? best : y;
        at = up ? v + e : at;
        best = up ? y : best;
      }
    }
  }
  u64 key = 0;
  if (at >= 0) {
    key = order_key(best, at);
  } else if (a.top) {  // nothing but -inf and NaN: the first of them in order
#pragma unroll 1
    for (int i = 0; i < EV; i++) {
      const int v = base + E * (t + NT * (i / E)) + i % E;
      if (v < end) {
        const u64 k = order_key(at_f32(x, v), v);
        key = k > key ? k : key;
      }
    }
  }
  u64 first = wave_max(key);
  if (NT > 64) {
    s_key[threadIdx.x] = key;
    if (lane == 0) s_red[w] = first;
    if (t == 0) s_n[0] = 0;
    sync();
#pragma unroll
    for (int i = 0; i < NW; i++) first = s_red[i] > first ? s_red[i] : first;
  } else if (t == 0) {
    s_n[gt] = 0;
  }
  const float m = key_value(first), ref = m == -INFINITY ? 0.f : m;
  // Two partial sums: the smallest entries of a thread's row of terms are the
  // first (f holds what each new maximum displaced)
  float rest = 0.f, xs = 0.f;
#pragma unroll
  for (int i = 0; i < EV; i++) {
    const float d = f[i] - ref, e = __builtin_amdgcn_exp2f(d * LOG2E);
    rest += e;
    xs = fmaf(e, fmaxf(d, -1e30f), xs);  // a share of 0 has no entropy; a NaN is in e
  }
  if (!(key == first && at >= 0)) {
    const float d = best - ref, e = __builtin_amdgcn_exp2f(d * LOG2E);
    rest += e;
    xs = fmaf(e, fmaxf(d, -1e30f), xs);
  }
  rest = wave_sum(rest);
  xs = wave_sum(xs);
  const int top = a.top;
  if (NT > 64) {
    if (lane == 0) s_sum[0][w] = rest, s_sum[1][w] = xs;
  }
  // the threshold, by the first wave of the group
  if (w == 0 && top) {
    u64 col = key;
    if (NT > 64) {
#pragma unroll
      for (int i = 1; i < NW; i++) col = s_key[lane + 64 * i] > col ? s_key[lane + 64 * i] : col;
    }
    s_key[NT > 64 ? lane : threadIdx.x] = col;
    sync_wave();
    int larger = 0;
    const u64* keys = s_key + (NT > 64 ? 0 : gt * 64);
#pragma unroll 8
    for (int i = 0; i < 64; i++) larger += keys[i] > col;
    // fewer than `top` columns with an entry: everything counts
    const u64 mask = __ballot(larger == top - 1 && col);
    if (mask ? lane == __ffsll(mask) - 1 : lane == 0) s_T[gt] = mask ? col : 1;
  }
  sync();
  if (NT > 64) {
    rest = s_sum[0][0];
    xs = s_sum[1][0];
#pragma unroll
    for (int i = 1; i < NW; i++) rest += s_sum[0][i], xs += s_sum[1][i];
  }
  float ll = 0.f, rref;
  const bool whole = NT == 64 || a.slices == 1;
  float* part = nullptr;
  if (whole) {
    ll = write_row<T>(a, row, m, rest, xs, rref, t == 0);
  } else {
    part = part_at(a, row, slice);
    if (t == 0) part[0] = rest, part[1] = xs, *(u64*)(part + 2) = first;
  }
  if (!top) return;
  auto put = [&](int place, u64 k) {
    if (whole) {
      a.ids[row * top + place] = key_index(k);
      a.alt[row * top + place] = at_f32(x, key_index(k)) - rref - ll;
    } else {
      ((u64*)(part + 4))[place] = k;
    }
  };
  const u64 T0 = s_T[gt];
  if (key >= T0) {
#pragma unroll 1
    for (int i = 0; i < NU; i++) {
      const int v = base + E * (t + NT * i);
#pragma unroll
      for (int e = 0; e < E; e++) {
        if (v + e >= end) break;
        const u64 k = order_key(at_f32(x, v + e), v + e);
        if (k >= T0) {
          const int n = atomicAdd(&s_n[gt], 1);
          if (n < CAP) s_cand[gt][n] = k;
        }
      }
    }
  }
  sync();
  const int n = s_n[gt];
  if (n <= CAP) {
    for (int i = t; i < n; i += NT) {
      const u64 k = s_cand[gt][i];
      int place = 0;
      for (int c = 0; c < n; c++) place += s_cand[gt][c] > k;
      if (place < top) put(place, k);
    }
    for (int i = n + t; i < top; i += NT) put(i, 0);  // a slice of fewer entries
    return;
  }
  // more than LDS holds (no natural row): the largest below the last, `top` times
  u64 last = ~0ull;
  for (int j = 0; j < top; j++) {
    u64 k0 = 0;
    for (int v = base + t; v < end; v += NT) {
      const u64 k = order_key(at_f32(x, v), v);
      if (k < last && k > k0) k0 = k;
    }
    k0 = wave_max(k0);
    if (NT > 64) {
      sync();
      if (lane == 0) s_red[w] = k0;
      sync();
#pragma unroll
      for (int i = 0; i < NW; i++) k0 = s_red[i] > k0 ? s_red[i] : k0;
    }
    last = k0;
    if (t == 0) put(j, k0);
  }
}

// The slices of a row, one wave per row: the sums relative to the row's
// maximum (slice s holds e^(m_s - m) (1 + rest_s) of them), and the largest of
// the slices' lists.
template <typename T>
__global__ __launch_bounds__(64) void k_score_join(ScoreArgs a) {
  __shared__ u64 cand[CAP];
  const int lane = threadIdx.x;
  const long row = blockIdx.x;
  const int S = a.slices, top = a.top;
  u64 first = 0, T0 = 1;
  for (int s = lane; s < S; s += 64) {
    const u64* p = (const u64*)part_at(a, row, s);
    first = p[1] > first ? p[1] : first;
    if (top && p[1 + top] > T0) T0 = p[1 + top];  // a slice's last: `top` entries are as large
  }
  first = wave_max(first);
  T0 = wave_max(T0);
  const float m = key_value(first), ref0 = m == -INFINITY ? 0.f : m;
  float rest = 0.f, xs = 0.f;
  for (int s = lane; s < S; s += 64) {
    const float* p = part_at(a, row, s);
    const u64 k = *(const u64*)(p + 2);
    const float ms = key_value(k), r = p[0], y = p[1];
    if (k == first || ms == -INFINITY) {  // without an entry of its own there is nothing to leave out
      rest += r;
      xs += y;
    } else {
      const float d = ms - ref0, f = __builtin_amdgcn_exp2f(d * LOG2E);
      rest += f * (1.f + r);
      xs += f > 0.f ? f * fmaf(d, 1.f + r, y) : f;
    }
  }
  rest = wave_sum(rest);
  xs = wave_sum(xs);
  float ref;
  const float ll = write_row<T>(a, row, m, rest, xs, ref, lane == 0);
  if (!top) return;
  const T* x = (const T*)a.x + row * a.ldx;
  auto put = [&](int place, u64 k) {
    a.ids[row * top + place] = key_index(k);
    a.alt[row * top + place] = at_f32(x, key_index(k)) - ref - ll;
  };
  int n = 0;
  const int all = S * top;
  for (int b = 0; b < all; b += 64) {
    const int i = b + lane, s = i / top;
    const u64 k = i < all ? ((const u64*)part_at(a, row, s))[2 + i - s * top] : 0;
    const bool in = k >= T0;
    const u64 mask = __ballot(in);
    const int to = n + __popcll(mask & ((1ull << lane) - 1));
    if (in && to < CAP) cand[to] = k;
    n += __popcll(mask);
  }
  sync_wave();
  if (n <= CAP) {
    for (int i = lane; i < n; i += 64) {
      const u64 k = cand[i];
      int place = 0;
      for (int c = 0; c < n; c++) place += cand[c] > k;
      if (place < top) put(place, k);
    }
    return;
  }
  u64 last = ~0ull;
  for (int j = 0; j < top; j++) {
    u64 k0 = 0;
    for (int i = lane; i < all; i += 64) {
      const u64 k = ((const u64*)part_at(a, row, i / top))[2 + i % top];
      if (k < last && k > k0) k0 = k;
    }
    last = k0 = wave_max(k0);
    if (lane == 0) put(j, k0);
  }
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
  typedef Unit<T> U;
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
    return -p * (dlp + dh * (fmaxf(lp, -1e30f) + H));
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
    const float d = fmaf(dlp, -expm1f(lp), -p * (dh * (fmaxf(lp, -1e30f) + H)));
    if constexpr (sizeof(O) == 2) dx[tk] = f2bf(d); else dx[tk] = d;
  }
}

long slices_of(long vocab) { return (vocab + SLICE - 1) / SLICE; }

template <typename T>
void launch_score(hipStream_t s, const ScoreArgs& a) {
  const unsigned waves = (unsigned)((a.rows + 3) / 4);
  if (a.V <= 512) {
    k_score<T, 64, 8><<<waves, 256, 0, s>>>(a);
  } else if (a.V <= 1024) {
    k_score<T, 64, 16><<<waves, 256, 0, s>>>(a);
  } else if (a.V <= 4096) {
    k_score<T, 256, 16><<<(unsigned)a.rows, 256, 0, s>>>(a);
  } else {
    k_score<T, 256, 32><<<(unsigned)(a.rows * a.slices), 256, 0, s>>>(a);
    if (a.slices > 1) k_score_join<T><<<(unsigned)a.rows, 64, 0, s>>>(a);
  }
}
template <typename T>
void launch_bwd(hipStream_t s, ScoreBwdArgs& a, int dx_dtype) {
  const int chunk = 64 * Unit<T>::E * 4;
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
  return (size_t)rows * slices_of(vocab) * (16 + 8 * (size_t)top);
}

extern "C" int sj_token_logprobs(void* stream, const void* x, int dtype, long ldx, long rows, long vocab,
                                 const int32_t* tokens, long top, float* logprob, float* entropy, float* stats,
                                 int32_t* top_ids, float* top_logprob, void* workspace, size_t workspace_bytes) {
  SJ_REQUIRE(dtype == SJ_F32 || dtype == SJ_BF16, "token log probabilities dtype %d", dtype);
  SJ_REQUIRE(rows >= 0 && rows <= 0x7fffffffL && vocab > 0 && vocab <= 1L << 24 && ldx >= vocab,
             "token log probabilities: %ld rows of %ld (stride %ld)", rows, vocab, ldx);
  SJ_REQUIRE(top >= 0 && top <= SJ_LOGPROBS_MAX_TOP && top <= vocab, "token log probabilities: %ld alternatives of %ld",
             top, vocab);
  SJ_REQUIRE(rows <= (1L << 24) / slices_of(vocab), "token log probabilities: %ld rows of %ld", rows, vocab);
  if (rows == 0) return SJ_OK;
  SJ_REQUIRE(x && (logprob == nullptr || tokens) && (top == 0 || (top_ids && top_logprob)),
             "token log probabilities: null");
  const size_t need = sj_token_logprobs_workspace_bytes(rows, vocab, top);
  if (need > workspace_bytes || (need && !workspace))
    return sjh::fail(SJ_ERR_CAPACITY, "token log probabilities workspace: required %zu bytes, available %zu bytes", need,
                     workspace ? workspace_bytes : 0);
  ScoreArgs a = {};
  a.x = x; a.ldx = ldx; a.rows = rows; a.V = (int)vocab; a.top = (int)top; a.slices = (int)slices_of(vocab);
  a.tokens = tokens; a.logprob = logprob; a.entropy = entropy; a.stats = stats; a.ids = top_ids; a.alt = top_logprob;
  a.part = (uint8_t*)workspace;
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
  SJ_REQUIRE(rows <= (1L << 24) / slices_of(vocab), "token log probabilities backward: %ld rows of %ld", rows, vocab);
  if (rows == 0) return SJ_OK;
  SJ_REQUIRE(x && stats && dx && (dlogprob == nullptr || tokens) && (dentropy == nullptr || entropy),
             "token log probabilities backward: null");
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
