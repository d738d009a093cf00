// One step of beam search: of all beams of a prompt and all tokens, those whose
// sequences are the most likely (no counterpart in the reference, which samples
// one sequence).
//
//   L_b = ln sum_v e^(x_bv),  total_bv = s_b + (x_bv - L_b)
//   rank_bv = total_bv / length_b^power
//
// Totals of different beams may lie next to each other, and which is the larger
// decides what the search goes on with: sums, totals and ranks are 64 bits.
// Within a beam the order is that of its logits, which are exact: where 64 bits
// leave the same total of them (a score of -1e30 all of it), they decide.
//
// What bounds it.  A prompt's step is two dependent halves, its rows and then
// all of its beams, and each ends with reductions of one workgroup: 64 prompts of
// 4 beams over 257 f32 take 7.8 us, 2 of them the launch's.  Over 8 rows of
// 131072 f32 (4 MB, 1 us at a copy's rate) 256 workgroups take 15.4 us with the
// meeting of their parts (64 kept: 26); a launch of its own for the second half
// had 8.5 + 15.2.  Over 384 rows of 50001 bf16 (38 MB, 7.5 us) the first half takes
// 25.6 us, of which the vector units work 12.5: 18 of their 25 operations an entry
// are the powers of e in 64 bits.  A workgroup loads its slice, then computes, and
// all begin together; what else the time is has not been shown.  The second half
// takes 7.2.
#include <type_traits>

#include "order.h"

using namespace sj;

namespace {

constexpr int SLICE = 4096;   // entries of a slice where slices are few
constexpr int NEAR = 256;     // lists whose sums and first entries LDS holds
constexpr int CAP = 1024;     // entries at or above a threshold that LDS holds
constexpr int MEETING = 1024; // slices of a call whose workgroups meet within the launch, at most

struct BeamArgs {
  const void* x;
  long ldx;
  int groups, B, V, keep, k;  // k: entries of a slice's list, min(keep, V)
  int slices, width;          // of a row; width: entries of a slice, a multiple of 8
  const float* scores;
  const int32_t *lengths, *ended;
  int end_token;
  double power;
  int32_t *parents, *tokens;
  float* scores_after;
  int32_t *lengths_after, *ended_after;
  u64* flag;  // [rows][slices], of the meetings
  u64 number;
  u64* sums;  // [rows][slices] of (maximum, sum)
  u64* keys;  // [groups][k][beams][slices]
};

// 2^t for -1000 <= t <= 1/2, to 2^-40: 2^n times a polynomial of degree 8 (least
// largest relative error over half a step to each side, 7.8e-13).  NaN is NaN:
// the last 12 bits of one that was 32 bits or comes of infinities are 0.
__device__ __forceinline__ double power2(double t) {
  const double magic = 6755399441055744.0;  // 1.5 2^52: the nearest whole number lies in the low bits
  const double tm = t + magic, f = t - (tm - magic);
  double p = 1.3175896059925506e-06;
  p = fma(p, f, 1.530973869952211e-05);
  p = fma(p, f, 0.00015403851471546215);
  p = fma(p, f, 0.0013333452055198773);
  p = fma(p, f, 0.009618128543494182);
  p = fma(p, f, 0.05550410939355053);
  p = fma(p, f, 0.2402265069887592);
  p = fma(p, f, 0.6931471805465064);
  p = fma(p, f, 0.9999999999997622);
  const long long b = __double_as_longlong(p);
  return __hiloint2double((int)(b >> 32) + (__double2loint(tm) << 20), (int)b);
}
constexpr double LOG2E_64 = 1.4426950408889634;
constexpr double FAR = 690.0;  // a power of e that no sum of 1 or more sees, and that 64 bits hold
// e^(x - ref), x - ref <= 0; below -FAR it is that of -FAR, 1e-300
__device__ __forceinline__ double power_of(float x, float ref) {
  const double d = (double)x - (double)ref;
  return power2((d < -FAR ? -FAR : d) * LOG2E_64);
}

// the order of finite ranks as whole numbers above 0
__device__ __forceinline__ u64 rank_key(double r) {
  const u64 b = (u64)__double_as_longlong(r + 0.0);
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}

// ---------------------------------------------------------------- one row
//
// NT threads (a wave or a workgroup) hold entries [base, end) of a row, EV a
// thread: the maximum, the sum of powers relative to it, and the k largest
// entries in their order (put(place, key), key 0 where there are fewer).  As in
// the token scores the largest come from a threshold, the k-th largest of 64 or
// 256 column maxima.  -inf is in no list; in a row with NaN they hold anything,
// since its sum leaves it without candidates.
template <int NT, int EV>
struct RowShared {
  static constexpr int CAPR = NT == 64 ? 512 : CAP;
  u64 cand[CAPR], last[4];
  double sum[4];
  __attribute__((aligned(16))) float best[NT];
  float max[4], T[4];
  int n;
};

template <typename T, int NT, int EV, int E, class P>
__device__ __forceinline__ void row_best(const T* x, int base, int end, int k, RowShared<NT, EV>& sh, float& m_out,
                                         double& sum_out, P put) {
  typedef Unit<T, E> U;
  constexpr int NU = EV / E, NW = NT / 64, CAPR = RowShared<NT, EV>::CAPR;
  const int t = threadIdx.x % NT, lane = threadIdx.x & 63, w = t >> 6;
  auto sync = [] {
    if constexpr (NT == 64)
      sync_wave();
    else
      __syncthreads();
  };
  auto index = [&](int i) { return base + E * (t + NT * (i / E)) + i % E; };
  U u[NU];
#pragma unroll
  for (int i = 0; i < NU; i++) {
    const int v = base + E * (t + NT * i);
    if (v + E <= end) u[i].r = *(const typename U::Raw*)(x + v);
  }
  constexpr int PART = 4, PARTS = EV / PART;
  float pm[PARTS], best = -INFINITY, least_of = INFINITY;
  auto f = [&](int i) { return u[i / E].get(i % E); };
#pragma unroll
  for (int i = 0; i < NU; i++) {
    const int v = base + E * (t + NT * i);
    if (v < end) {
      if (v + E > end) {  // a unit that crosses the end is filled with -inf
#pragma unroll
        for (int e = 0; e < E; e++) u[i].set(e, v + e < end ? at_f32(x, v + e) : -INFINITY);
      }
#pragma unroll
      for (int j = i * E / PART; j < (i + 1) * E / PART; j++) {
        pm[j] = fmaxf(fmaxf(f(PART * j), f(PART * j + 1)), fmaxf(f(PART * j + 2), f(PART * j + 3)));
        best = fmaxf(best, pm[j]);
        least_of = fminf(least_of, fminf(fminf(f(PART * j), f(PART * j + 1)), fminf(f(PART * j + 2), f(PART * j + 3))));
      }
    }
  }
  float m = all_max(best);
  if (t == 0) sh.n = 0;
  if (NT > 64) {
    sh.best[t] = best;
    if (lane == 0) sh.max[w] = m;
    sync();
    m = fmaxf(fmaxf(sh.max[0], sh.max[1]), fmaxf(sh.max[2], sh.max[3]));
  }
  if (w == 0 || k > 32) {
    const bool all = NT > 64 && k > 32;
    float col = best;
    if (NT > 64 && !all) col = fmaxf(fmaxf(best, sh.best[lane + 64]), fmaxf(sh.best[lane + 128], sh.best[lane + 192]));
    if (!all) sh.best[lane] = col;
    sync_wave();
    int larger = 0;
    for (int j = 0; j < (all ? 256 : 64); j += 64)
#pragma unroll
      for (int i = 0; i < 64; i += 4) {
        const f32x4 c = *(const f32x4*)(sh.best + j + i);
        larger += (c[0] > col) + (c[1] > col) + (c[2] > col) + (c[3] > col);
      }
    const float least = all_min(larger < k ? col : INFINITY);
    if (NT == 64 ? lane == 0 : all ? lane == 0 : lane < 4) sh.T[NT == 64 ? 0 : all ? w : lane] = least;
  }
  // Entries too far below the maximum for power2 (a mask's) are moved up to
  // where they still count for nothing; where there is nothing but -inf, the
  // sum is only asked for NaN
  const float ref = m == -INFINITY ? 0.f : m;
  const double scaled = -(double)ref * LOG2E_64;
  // past 1024 the rounding of the scaled maximum is no longer less than the
  // polynomial's error: there, too, the difference comes first, which is exact
  const bool far = (double)least_of - (double)ref < -FAR || !(fabsf(ref) <= 1024.f);
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < NU; i++)
    if (base + E * (t + NT * i) < end) {
      if (__any(far)) {
#pragma unroll
        for (int e = 0; e < E; e++) sum += power_of(f(i * E + e), ref);
      } else {
#pragma unroll
        for (int e = 0; e < E; e++) sum += power2(fma((double)f(i * E + e), LOG2E_64, scaled));
      }
    }
  sum = wave_sum(sum);
  if (NT > 64) {
    if (lane == 0) sh.sum[w] = sum;
    sync();
    sum = (sh.sum[0] + sh.sum[1]) + (sh.sum[2] + sh.sum[3]);
  } else {
    sync();
  }
  m_out = m;
  sum_out = m == -INFINITY && sum == sum ? 0.0 : sum;
  const float T0 = NT == 64 ? sh.T[0] : fminf(fminf(sh.T[0], sh.T[1]), fminf(sh.T[2], sh.T[3]));
  uint32_t mine = 0;
#pragma unroll
  for (int j = 0; j < PARTS; j++)
    if (index(PART * j) < end && pm[j] >= T0)
#pragma unroll
      for (int i = PART * j; i < PART * (j + 1); i++) mine += f(i) >= T0 && f(i) > -INFINITY && index(i) < end;
  const uint32_t upto = scan_add(mine);
  int from = 0;
  if (lane == 63 && upto) from = atomicAdd(&sh.n, (int)upto);
  from = __builtin_amdgcn_readlane(from, 63) + (int)(upto - mine);
#pragma unroll
  for (int j = 0; j < PARTS; j++)
    if (index(PART * j) < end && pm[j] >= T0) {
#pragma unroll
      for (int i = PART * j; i < PART * (j + 1); i++)
        if (f(i) >= T0 && f(i) > -INFINITY && index(i) < end) {
          if (from < CAPR) sh.cand[from] = order_key(f(i), index(i));
          from++;
        }
    }
  sync();
  const int n = sh.n;
  if (n <= CAPR) {
    rank<NT>(sh.cand, n, k, t, put);
    for (int i = n + t; i < k; i += NT) put(i, 0ull);
    return;
  }
  // more than LDS holds at the threshold (a mask's lowest value in all but fewer
  // than k entries): the largest below the last, k times.  8 rows of 131072 with
  // five entries left: 16 kept 220 us, 64 kept 2.5 ms; with -inf 17 and 22.
  u64 last = ~0ull;
  for (int j = 0; j < k; j++) {
    u64 k0 = 0;
    for (int v = base + t; v < end; v += NT) {
      const u64 key = order_key(at_f32(x, v), v);
      if (key < last && key > k0) k0 = key;
    }
    k0 = all_max(k0);
    if (NT > 64) {
      sync();
      if (lane == 0) sh.last[w] = k0;
      sync();
#pragma unroll
      for (int i = 0; i < NW; i++) k0 = larger_of(k0, sh.last[i]);
    }
    last = k0;
    if (t == 0) put(j, k0);
  }
}

// ------------------------------------------------------------- the prompt
//
// One workgroup takes the lists of a prompt's beams together: their sums, the
// ranks of all entries, and the `keep` first of them, again through a threshold.
struct GroupShared {
  double base[64], factor[64], score[64];  // the beam's L, length^power
  int live[64];                            // 0: no candidate, 1: its tokens, 2: ended
  int order[64];                           // the beams of the second, then of the third
  u64 cand[CAP], tie[CAP];                 // ranks' keys, and the order among equals
  __attribute__((aligned(16))) u64 best[256];
  u64 last[4];
  uint16_t pick[CAP];
  int cols[4], n, picked;
};
// sums and entries of the lists, as many as LDS holds
struct Near {
  u64 sums[2 * NEAR], keys[4 * NEAR];
};
// tie: its place among those of the same rank, the largest first: the lowest beam
// (6 bits from 56), the largest logit (32 from 24), the lowest token (24)
struct Candidate {
  u64 key;  // 0: none
  u64 tie;
};
__device__ __forceinline__ u64 tie_of(int beam, u64 key) {  // key: the list's
  return (u64)(63 - beam) << 56 | (key >> 32) << 24 | (key & 0xffffffu);
}
__device__ __forceinline__ int tie_beam(u64 tie) { return 63 - (int)(tie >> 56); }
__device__ __forceinline__ float tie_value(u64 tie) { return key_value(tie << 8); }
__device__ __forceinline__ int tie_token(u64 tie) { return 0xffffff - (int)(tie & 0xffffffu); }

// of a wave's columns, among the n in LDS, the least of those with fewer than keep
// larger ones (equal columns have one place)
__device__ __forceinline__ u64 least_of_first(const u64* best, int n, u64 col, int keep) {
  int larger = 0;
#pragma unroll 4
  for (int i = 0; i < n; i += 2) {
    const ulonglong2 q = *(const ulonglong2*)(best + i);
    larger += (q.x > col) + (q.y > col);
  }
  // that is a column with the most larger ones, below keep <= 64: found bit by bit
  uint64_t lanes = __ballot(col != 0 && larger < keep);
  if (lanes == 0) return ~0ull;
#pragma unroll
  for (int bit = 5; bit >= 0; bit--) {
    const uint64_t set = lanes & __ballot((larger >> bit) & 1);
    if (set) lanes = set;
  }
  const int lane = __builtin_ctzll(lanes);
  return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(col >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)col, lane);
}

template <bool MEET>
__device__ __forceinline__ void group_best(const BeamArgs& a, int g, GroupShared& sh, Near& near, bool there) {
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, B = a.B, S = a.slices, k = a.k, keep = a.keep;
  const long row0 = (long)g * B;
  const u64* keys = a.keys + row0 * S * k;
  const int lists = B * S, all = lists * k;  // all lists' first entries, then their second ones
  const u64* sums = a.sums + 2 * row0 * S;
  auto get = [&](const u64* p) { return MEET ? part_get(p) : *p; };
  // the first two entries of every list; few of the others are looked at
  const int near_sums = min(2 * lists, 2 * NEAR), near_keys = min(all, min(4 * NEAR, max(512, 2 * lists)));
  if (!there) {
    // two of each a thread, all on their way at once; near_sums is at most 512
    u64 s0 = 0, s1 = 0, k0 = 0, k1 = 0;
    if (t < near_sums) s0 = get(sums + t);
    if (t < near_keys) k0 = get(keys + t);
    if (t + 256 < near_sums) s1 = get(sums + t + 256);
    if (t + 256 < near_keys) k1 = get(keys + t + 256);
    if (t < near_sums) near.sums[t] = s0;
    if (t < near_keys) near.keys[t] = k0;
    if (t + 256 < near_sums) near.sums[t + 256] = s1;
    if (t + 256 < near_keys) near.keys[t + 256] = k1;
#pragma unroll 4
    for (int i = t + 512; i < near_keys; i += 256) near.keys[i] = get(keys + i);
  }
  auto sum_at = [&](int i) { return i < near_sums ? near.sums[i] : get(sums + i); };
  auto key_at = [&](int i) { return i < near_keys ? near.keys[i] : get(keys + i); };
  if (t == 0) sh.n = 0;
  __syncthreads();
  // 16 lanes a beam
  for (int b = t >> 4; b < B; b += 16) {
    const int l = t & 15;
    const long row = row0 + b;
    const float score = a.scores[row];
    const bool ended = a.ended && a.ended[row];
    const int len = a.lengths ? a.lengths[row] : 0;
    float M = -INFINITY;
    double sum = 0.0;
    if (!ended) {
      for (int s = l; s < S; s += 16) M = fmaxf(M, __uint_as_float((uint32_t)sum_at(2 * (b * S + s))));
#pragma unroll
      for (int d = 8; S > 1 && d; d >>= 1) M = fmaxf(M, __shfl_xor(M, d, 64));
#pragma unroll 1
      for (int s = l; s < S; s += 16) {
        const float m = __uint_as_float((uint32_t)sum_at(2 * (b * S + s)));
        const double v = __longlong_as_double((long long)sum_at(2 * (b * S + s) + 1));
        sum += v * power_of(m, M == -INFINITY ? 0.f : M);
      }
#pragma unroll
      for (int d = 8; S > 1 && d; d >>= 1) sum += __shfl_xor(sum, d, 64);
    }
    // one logarithm for both
    const double after = (double)max(ended ? (long)len : len + 1L, 1L), ln = log(l == 0 ? sum : after);
    if (l == 0) {
      int live = score == score && fabsf(score) < INFINITY ? 2 : 0;
      const double base = (double)M + ln;
      if (live && !ended) live = base == base && fabs(base) < INFINITY ? 1 : 0;
      sh.base[b] = base;
      sh.score[b] = score;
      sh.live[b] = live;
    } else if (l == 1) {
      sh.factor[b] = power2(a.power * ln * LOG2E_64);  // up to 2^496
    }
  }
  __syncthreads();
  // the beams with candidates: those whose tokens are, then the ended ones
  const int state = lane < B ? sh.live[lane] : 0;
  const uint64_t with = __ballot(state == 1), done = __ballot(state == 2), below = (1ull << lane) - 1;
  const int beams_open = __popcll(with);
  const bool in_order = beams_open == B;
  if (!in_order) {
    if (w == 0 && state == 1) sh.order[__popcll(with & below)] = lane;
    if (w == 0 && state == 2) sh.order[beams_open + __popcll(done & below)] = lane;
    __syncthreads();
  }
  // their lists: one for each slice of an open beam, one of one entry of an ended one
  const int open = beams_open * S, closed = __popcll(done), some_lists = open + closed;
  auto candidate = [&](int list, int place) {
    Candidate c = {0, 0};
    const bool ended = list >= open;
    const int nth = ended ? list - open + beams_open : list / S, b = in_order ? nth : sh.order[nth];
    double total = sh.score[b];
    if (ended) {
      if (place) return c;
      c.tie = tie_of(b, order_key(0.f, max(a.end_token, 0)));
    } else {
      const u64 key = key_at(place * lists + b * S + list - nth * S);
      const float x = key_value(key);
      if (key == 0 || x == -INFINITY) return c;
      total += (double)x - sh.base[b];
      c.tie = tie_of(b, key);
    }
    c.key = rank_key(a.power == 0.0 ? total : total / sh.factor[b]);
    return c;
  };
  // Each list is in order: `each` threads go down every each-th entry of it, and
  // stop at the first below the threshold.  (Over the lists of all beams, a
  // search's first step, which has one open beam, left most threads without any:
  // 3 prompts of 16 beams over 89268, 32 kept, 41 us.)
  const int per = max(some_lists, 1), each = max(256 / per, 1), from = t / per;
  const int list0 = t < each * per ? t - from * per : some_lists;
  // (up to 64 entries are simply all ranked: 9.4 us with a threshold for 64 prompts
  // of 4 beams over 257, 7.8 without)
  u64 T0 = 1;
  if (open * k + closed > 64) {
    u64 best = 0;
#pragma unroll 1
    for (int list = list0; list < some_lists; list += 256)
      if (from < k) best = larger_of(best, candidate(list, from).key);
    // the threshold: the keep-th largest of 64 columns' largest (of 256 above 32,
    // where the 64th of 64 would let thousands pass), 1 where fewer columns have any.
    // Few entries lie above it, as the lists' first ones are spread over the columns.
    sh.best[t] = best;
    __syncthreads();
    const bool many = keep > 32;
    if (w == 0 || many) {
      u64 col = best;
      if (!many) {
        col = larger_of(larger_of(best, sh.best[lane + 64]), larger_of(sh.best[lane + 128], sh.best[lane + 192]));
        sync_wave();
        sh.best[lane] = col;
        sync_wave();
      }
      const u64 least = least_of_first(sh.best, many ? 256 : 64, col, keep);
      const int some = __popcll(__ballot(col != 0));
      if (lane == 0) {
        sh.last[w] = least;
        sh.cols[w] = some;
      }
    }
    __syncthreads();
    int some = sh.cols[0];
    T0 = sh.last[0];
    for (int i = 1; many && i < 4; i++) {
      T0 = min(T0, sh.last[i]);
      some += sh.cols[i];
    }
    if (some < keep) T0 = 1;
  }
#pragma unroll 1
  for (int list = list0; list < some_lists; list += 256)
#pragma unroll 1
    for (int place = from; place < k; place += each) {
      const Candidate q = candidate(list, place);
      if (q.key < T0) break;
      const int n = atomicAdd(&sh.n, 1);
      if (n < CAP) sh.cand[n] = q.key, sh.tie[n] = q.tie;
    }
  __syncthreads();
  auto write = [&](int place, bool some, u64 tie) {
    const long at = (long)g * keep + place;
    const int b = some ? tie_beam(tie) : 0, token = tie_token(tie);
    const long row = row0 + b;
    const bool was = some && sh.live[b] == 2;
    const double total = sh.score[b] + (was ? 0.0 : (double)tie_value(tie) - sh.base[b]);
    a.parents[at] = some ? (int)row : -1;
    a.tokens[at] = !some ? -1 : was ? a.end_token : token;
    a.scores_after[at] = some ? (float)total : -INFINITY;
    if (a.lengths_after) a.lengths_after[at] = some ? (a.lengths ? a.lengths[row] : 0) + (was ? 0 : 1) : 0;
    if (a.ended_after) a.ended_after[at] = !some || was || token == a.end_token;
  };
  const int n = sh.n;
  if (n <= CAP) {
    // Every entry's place is the number of larger ones.  Among many only the keep
    // largest of 256 columns, and what lies with them, can have one below keep (384
    // rows, 32 kept: up to 700 entries, 41 us for all against all, 22 this way).
    int m = n;
    if (n > 192) {
      u64 col = 0;
      for (int i = t; i < n; i += 256) col = larger_of(col, sh.cand[i]);
      sh.best[t] = col;
      if (t == 0) sh.picked = 0;
      __syncthreads();
      const u64 least = least_of_first(sh.best, 256, col, keep);
      if (lane == 0) sh.last[w] = least;
      __syncthreads();
      const u64 T1 = min(min(sh.last[0], sh.last[1]), min(sh.last[2], sh.last[3]));
      for (int i = t; i < n; i += 256)
        if (sh.cand[i] >= T1) sh.pick[atomicAdd(&sh.picked, 1)] = (uint16_t)i;
      __syncthreads();
      m = sh.picked;
    }
    for (int q = t >> 2; q < m; q += 64) {
      const int i = n > 192 ? sh.pick[q] : q;
      const u64 key = sh.cand[i], tie = sh.tie[i];
      uint32_t place = 0, same = 0;
#pragma unroll 4
      for (int j = t & 3; j < n; j += 4) {
        const u64 other = sh.cand[j];
        place += other > key;
        same += other == key;
      }
      if (same > (uint32_t)((i & 3) == (t & 3)))  // another of the same rank
        for (int j = t & 3; j < n; j += 4) place += sh.cand[j] == key && sh.tie[j] > tie;
      place += dpp<0xB1>(place);
      place += dpp<0x4E>(place);
      if ((t & 3) == 0 && (int)place < keep) write((int)place, true, tie);
    }
    for (int i = n + t; i < keep; i += 256) write(i, false, 0);
    return;
  }
  // more of the same rank than LDS holds: the first behind the last, keep times
  u64 last = ~0ull, last_tie = 0;
  for (int j = 0; j < keep; j++) {
    Candidate top = {0, 0};
    for (int i = t; i < some_lists * k; i += 256) {
      const Candidate q = candidate(i % per, i / per);
      const bool behind = q.key && (q.key < last || (q.key == last && q.tie < last_tie));
      if (behind && (q.key > top.key || (q.key == top.key && q.tie > top.tie))) top = q;
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) {
      const u64 key = __shfl_xor(top.key, d, 64), tie = __shfl_xor(top.tie, d, 64);
      if (key > top.key || (key == top.key && tie > top.tie)) top = Candidate{key, tie};
    }
    __syncthreads();
    if (lane == 0) sh.cand[w] = top.key, sh.tie[w] = top.tie;
    __syncthreads();
    for (int i = 0; i < 4; i++)
      if (sh.cand[i] > top.key || (sh.cand[i] == top.key && sh.tie[i] > top.tie)) top = Candidate{sh.cand[i], sh.tie[i]};
    if (t == 0) write(j, top.key != 0, top.tie);
    last = top.key;
    last_tie = top.tie;
  }
}

// One wave per row (NT = 64: a workgroup has four rows of a prompt) or one
// workgroup per slice.  MEET: the last of a prompt's workgroups takes its beams
// together.
template <typename T, int NT, int EV, int E = WIDE<T>, bool MEET = false>
__global__ __launch_bounds__(256) void k_beam_rows(BeamArgs a) {
  __shared__ union {
    RowShared<NT, EV> row[256 / NT];
    std::conditional_t<MEET, GroupShared, int> group;
  } sh;
  __shared__ std::conditional_t<MEET, Near, int> near;
  const int gt = threadIdx.x / NT;
  // the prompt's parts, and the row and slice of this one
  const int parts = NT == 64 ? (a.B + 3) / 4 : a.B * a.slices, g = blockIdx.x / parts, part = blockIdx.x - g * parts;
  const int beam = NT == 64 ? 4 * part + gt : part / a.slices, slice = NT == 64 ? 0 : part - beam * a.slices;
  const long row = (long)g * a.B + beam;
  const bool there = MEET && NT == 64 && parts == 1;  // the lists go from LDS to LDS
  if (beam < a.B && !(a.ended && a.ended[row])) {
    const int base = slice * a.width, end = min(a.V, base + a.width);
    float m;
    double sum;
    const int lists = a.B * a.slices;
    u64* list = a.keys + (long)g * lists * a.k + beam * a.slices + slice;
    row_best<T, NT, EV, E>((const T*)a.x + row * a.ldx, base, end, a.k, sh.row[gt], m, sum, [&](int place, u64 key) {
      if constexpr (MEET) {
        if (there)  // slice 0 is all
          near.keys[place * lists + beam] = key;
        else
          part_put(list + (long)place * lists, key);
      } else {
        list[(long)place * lists] = key;
      }
    });
    if (threadIdx.x % NT == 0) {
      u64* p = a.sums + 2 * (row * a.slices + slice);
      if constexpr (MEET) {
        const u64 own[2] = {(u64)__float_as_uint(m), (u64)__double_as_longlong(sum)};
        for (int i = 0; i < 2; i++)
          if (there)
            near.sums[2 * beam + i] = own[i];
          else
            part_put(p + i, own[i]);
      } else {
        p[0] = __float_as_uint(m);
        p[1] = (u64)__double_as_longlong(sum);
      }
    }
  }
  if constexpr (MEET) {
    __shared__ int complete;
    u64* flags = a.flag + (long)g * a.B * a.slices;
    if (there)
      __syncthreads();
    else if (!meet([&](int i) { return flags + i; }, part, parts, a.number, &complete))
      return;
    group_best<true>(a, g, sh.group, near, there);
  }
}
__global__ __launch_bounds__(256) void k_beam_join(BeamArgs a) {
  __shared__ GroupShared sh;
  __shared__ Near near;
  group_best<false>(a, blockIdx.x, sh, near, false);
}

long slices_of(long vocab) { return (vocab + SLICE - 1) / SLICE; }

template <typename T>
void launch_select(hipStream_t s, BeamArgs& a) {
  const long rows = (long)a.groups * a.B;
  a.slices = 1;
  a.width = (a.V + 7) / 8 * 8;
  a.number = sjh::call_number();
  if (a.V <= 1024) {
    const unsigned blocks = (unsigned)(a.groups * ((a.B + 3) / 4));
    if (a.V <= 512)
      k_beam_rows<T, 64, 8, 4, true><<<blocks, 256, 0, s>>>(a);
    else
      k_beam_rows<T, 64, 16, WIDE<T>, true><<<blocks, 256, 0, s>>>(a);
  } else {
    const bool meets = a.V <= SLICE || rows * slices_of(a.V) <= MEETING;
    constexpr int LONG = sizeof(T) == 2 ? 64 : 32;  // entries a thread holds where slices are many
    const int most = meets ? SLICE : 256 * LONG;
    a.slices = (a.V + most - 1) / most;
    a.width = ((a.V + a.slices - 1) / a.slices + 7) / 8 * 8;
    const unsigned blocks = (unsigned)(rows * a.slices);
    if (meets) {
      k_beam_rows<T, 256, 16, WIDE<T>, true><<<blocks, 256, 0, s>>>(a);
    } else {
      k_beam_rows<T, 256, LONG><<<blocks, 256, 0, s>>>(a);
      k_beam_join<<<(unsigned)a.groups, 256, 0, s>>>(a);
    }
  }
}

}  // namespace

extern "C" size_t sj_beam_select_workspace_bytes(long groups, long beams, long vocab, long keep) {
  if (groups <= 0 || beams <= 0 || vocab <= 0 || keep <= 0) return 0;
  return (size_t)groups * beams * slices_of(vocab) * (24 + 8 * (size_t)(keep < vocab ? keep : vocab));
}

extern "C" int sj_beam_select(void* stream, const void* x, int dtype, long ldx, long groups, long beams, long vocab,
                              const float* scores, const int32_t* lengths, const int32_t* ended, int32_t end_token,
                              double length_power, long keep, int32_t* parents, int32_t* tokens, float* scores_after,
                              int32_t* lengths_after, int32_t* ended_after, void* workspace, size_t workspace_bytes) {
  SJ_REQUIRE(dtype == SJ_F32 || dtype == SJ_BF16, "beam selection dtype %d", dtype);
  SJ_REQUIRE(groups >= 0 && groups <= 1L << 24 && beams > 0 && beams <= SJ_BEAM_MAX && keep > 0 && keep <= SJ_BEAM_MAX &&
                 vocab > 0 && vocab <= 1L << 24 && ldx >= vocab,
             "beam selection: %ld prompts of %ld beams, %ld of %ld (stride %ld)", groups, beams, keep, vocab, ldx);
  // the most workgroups of a launch: more than MEETING slices are of 8192 entries or more
  SJ_REQUIRE(groups * beams * ((vocab + 2 * SLICE - 1) / (2 * SLICE)) < 1L << 23, "beam selection: %ld rows of %ld", groups * beams, vocab);
  SJ_REQUIRE(end_token >= -1 && end_token < vocab, "beam selection: end token %d of %ld", end_token, vocab);
  SJ_REQUIRE(length_power >= 0.0 && length_power <= 16.0, "beam selection: length power %g", length_power);
  if (groups == 0) return SJ_OK;
  SJ_REQUIRE(x && scores && parents && tokens && scores_after && (length_power == 0.0 || lengths) &&
                 (lengths_after == nullptr || lengths),
             "beam selection: null");
  SJ_REQUIRE((const float*)scores_after != scores && (!lengths_after || (const int32_t*)lengths_after != lengths) &&
                 (!ended_after || (const int32_t*)ended_after != ended),
             "beam selection: the beams after the step need arrays of their own");
  const size_t need = sj_beam_select_workspace_bytes(groups, beams, vocab, keep);
  SJ_REQUIRE(((uintptr_t)workspace & 15) == 0, "beam selection: the workspace is not 16-byte aligned");
  if (need > workspace_bytes || !workspace)
    return sjh::fail(SJ_ERR_CAPACITY, "beam selection workspace: required %zu bytes, available %zu bytes", need,
                     workspace ? workspace_bytes : 0);
  BeamArgs a = {};
  a.x = x; a.ldx = ldx; a.groups = (int)groups; a.B = (int)beams; a.V = (int)vocab; a.keep = (int)keep;
  a.k = (int)(keep < vocab ? keep : vocab);
  a.scores = scores; a.lengths = lengths; a.ended = ended; a.end_token = end_token; a.power = length_power;
  a.parents = parents; a.tokens = tokens; a.scores_after = scores_after;
  a.lengths_after = lengths_after; a.ended_after = ended_after;
  const size_t all = (size_t)groups * beams * slices_of(vocab);
  a.sums = (u64*)workspace;
  a.flag = a.sums + 2 * all;
  a.keys = a.flag + all;
  if (dtype == SJ_BF16)
    launch_select<bf16_t>((hipStream_t)stream, a);
  else
    launch_select<float>((hipStream_t)stream, a);
  SJ_LAUNCH_CHECK("beam selection");
  return SJ_OK;
}
