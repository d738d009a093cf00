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

constexpr int ST = 256;

// the order of the alternatives: larger values first, NaN behind everything,
// the lowest index first among equals; a larger key comes first, and no two
// entries of a row have the same
__device__ __forceinline__ uint64_t order_key(float x, int v) {
  uint32_t b = __float_as_uint(x + 0.f);  // -0 is 0
  b = x != x ? 0u : (b >> 31) ? ~b : (b | 0x80000000u);
  return ((uint64_t)b << 32) | (uint32_t)(0x7fffffff - v);
}

struct ScoreArgs {
  const void* x;
  int dt;
  long ldx;
  long rows;
  int V, top;
  const int32_t* tokens;
  float *logprob, *entropy, *stats;
  int32_t* ids;
  float* alt;
};

__global__ __launch_bounds__(ST) void k_score_rows(ScoreArgs a) {
  __shared__ float rf[ST / 64];
  __shared__ uint64_t rk[ST / 64];
  const int t = threadIdx.x;
  const long r = blockIdx.x, base = r * a.ldx;
  float m = -INFINITY;
  for (int v = t; v < a.V; v += ST) {
    const float x = load_as_f32(a.x, a.dt, base + v);
    m = x > m ? x : m;
  }
  m = wave_max(m);
  if ((t & 63) == 0) rf[t >> 6] = m;
  __syncthreads();
  for (int i = 0; i < ST / 64; i++) m = fmaxf(m, rf[i]);
  __syncthreads();
  const float ref = m == -INFINITY ? 0.f : m;
  float rest = 0.f, ones = 0.f, xs = 0.f;
  for (int v = t; v < a.V; v += ST) {
    const float x = load_as_f32(a.x, a.dt, base + v), d = x - ref;
    if (x == m) {
      ones += 1.f;
    } else {
      const float e = expf(d);
      rest += e;
      xs += e > 0.f ? e * d : e;  // a share of 0 has no entropy; NaN stays
    }
  }
  rest = block_sum<float, ST>(rest, rf);
  ones = block_sum<float, ST>(ones, rf);
  xs = block_sum<float, ST>(xs, rf);
  const bool none = m == -INFINITY && rest == 0.f;  // every entry -inf
  rest += ones - 1.f;
  const float ll = none ? 0.f : log1pf(rest);
  if (t == 0) {
    const int tk = a.tokens ? a.tokens[r] : -1;
    if (a.logprob) a.logprob[r] = tk >= 0 && tk < a.V ? load_as_f32(a.x, a.dt, base + tk) - ref - ll : 0.f;
    if (a.entropy) a.entropy[r] = none ? 0.f : ll - xs / (1.f + rest);
    if (a.stats) a.stats[2 * r] = ref, a.stats[2 * r + 1] = ll;
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < a.top; k++) {
    uint64_t best = 0;
    for (int v = t; v < a.V; v += ST) {
      const uint64_t key = order_key(load_as_f32(a.x, a.dt, base + v), v);
      if (key < last && key > best) best = key;
    }
    best = wave_max(best);
    if ((t & 63) == 0) rk[t >> 6] = best;
    __syncthreads();
    for (int i = 0; i < ST / 64; i++) best = best > rk[i] ? best : rk[i];
    __syncthreads();
    last = best;
    if (t == 0) {
      const int v = 0x7fffffff - (int)(uint32_t)best;
      a.ids[r * a.top + k] = v;
      a.alt[r * a.top + k] = load_as_f32(a.x, a.dt, base + v) - ref - ll;
    }
  }
}

struct ScoreBwdArgs {
  const void* x;
  int dt;
  long ldx;
  int V;
  const int32_t* tokens;
  const float *stats, *entropy, *dlp, *dent;
  void* dx;
  int ddt;
  long lddx;
};

__global__ __launch_bounds__(ST) void k_score_bwd(ScoreBwdArgs a) {
  const long r = blockIdx.x;
  const int tk = a.tokens ? a.tokens[r] : -1;
  const bool scored = tk >= 0 && tk < a.V;
  const float m = a.stats[2 * r], ll = a.stats[2 * r + 1];
  const float dlp = a.dlp && scored ? a.dlp[r] : 0.f, dh = a.dent ? a.dent[r] : 0.f, H = a.dent ? a.entropy[r] : 0.f;
  for (int v = threadIdx.x; v < a.V; v += ST) {
    const float lp = load_as_f32(a.x, a.dt, r * a.ldx + v) - m - ll, p = expf(lp);
    const float own = scored && v == tk ? -expm1f(lp) : -p;
    const float ent = p > 0.f ? p * (lp + H) : p;
    store_from_f32(a.dx, a.ddt, r * a.lddx + v, dlp * own - dh * ent);
  }
}

}  // namespace

extern "C" size_t sj_token_logprobs_workspace_bytes(long rows, long vocab, long top) { return 0; }

extern "C" int sj_token_logprobs(void* stream, const void* x, int dtype, long ldx, long rows, long vocab,
                                 const int32_t* tokens, long top, float* logprob, float* entropy, float* stats,
                                 int32_t* top_ids, float* top_logprob, void* workspace, size_t workspace_bytes) {
  SJ_REQUIRE(dtype == SJ_F32 || dtype == SJ_BF16, "token log probabilities dtype %d", dtype);
  SJ_REQUIRE(rows >= 0 && rows <= 0x7fffffffL && vocab > 0 && vocab <= 1L << 30 && ldx >= vocab,
             "token log probabilities: %ld rows of %ld (stride %ld)", rows, vocab, ldx);
  SJ_REQUIRE(top >= 0 && top <= SJ_LOGPROBS_MAX_TOP && top <= vocab, "token log probabilities: %ld alternatives of %ld",
             top, vocab);
  if (rows == 0) return SJ_OK;
  SJ_REQUIRE(x && (logprob == nullptr || tokens) && (top == 0 || (top_ids && top_logprob)),
             "token log probabilities: null");
  const size_t need = sj_token_logprobs_workspace_bytes(rows, vocab, top);
  if (need > workspace_bytes || (need && !workspace))
    return sjh::fail(SJ_ERR_CAPACITY, "token log probabilities workspace: required %zu bytes, available %zu bytes", need,
                     workspace ? workspace_bytes : 0);
  ScoreArgs a = {};
  a.x = x; a.dt = dtype; a.ldx = ldx; a.rows = rows; a.V = (int)vocab; a.top = (int)top;
  a.tokens = tokens; a.logprob = logprob; a.entropy = entropy; a.stats = stats; a.ids = top_ids; a.alt = top_logprob;
  k_score_rows<<<(unsigned)rows, ST, 0, (hipStream_t)stream>>>(a);
  SJ_LAUNCH_CHECK("token log probabilities");
  return SJ_OK;
}

extern "C" int sj_token_logprobs_bwd(void* stream, const void* x, int dtype, long ldx, long rows, long vocab,
                                     const int32_t* tokens, const float* stats, const float* entropy,
                                     const float* dlogprob, const float* dentropy, void* dx, int dx_dtype, long lddx) {
  SJ_REQUIRE((dtype == SJ_F32 || dtype == SJ_BF16) && (dx_dtype == SJ_F32 || dx_dtype == SJ_BF16),
             "token log probabilities backward dtypes %d, %d", dtype, dx_dtype);
  SJ_REQUIRE(rows >= 0 && rows <= 0x7fffffffL && vocab > 0 && vocab <= 1L << 30 && ldx >= vocab && lddx >= vocab,
             "token log probabilities backward: %ld rows of %ld (strides %ld, %ld)", rows, vocab, ldx, lddx);
  if (rows == 0) return SJ_OK;
  SJ_REQUIRE(x && stats && dx && (dlogprob == nullptr || tokens) && (dentropy == nullptr || entropy),
             "token log probabilities backward: null");
  ScoreBwdArgs a = {};
  a.x = x; a.dt = dtype; a.ldx = ldx; a.V = (int)vocab; a.tokens = tokens; a.stats = stats; a.entropy = entropy;
  a.dlp = dlogprob; a.dent = dentropy; a.dx = dx; a.ddt = dx_dtype; a.lddx = lddx;
  k_score_bwd<<<(unsigned)rows, ST, 0, (hipStream_t)stream>>>(a);
  SJ_LAUNCH_CHECK("token log probabilities backward");
  return SJ_OK;
}
