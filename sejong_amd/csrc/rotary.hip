// Rotary positions at given positions (no counterpart in the reference, whose
// rope, kernels.py:103-113, counts rows and rotates whole heads): interleaved
// or half layout, the first rotary_dim columns of each head, frequencies
// scaled for long contexts; and the same fused with the write of a step's keys
// and values into the slots of a paged cache.
//
//   (a, b) -> A (a cos t - b sin t, a sin t + b cos t),  t = position * f_i
//
// A frequency is held as the fraction of a turn it makes per position, in
// 64-bit fixed point: position * turns modulo 2^64 is the angle's fraction of
// a turn with no further rounding (in fp32 the angle of position 2^20 is
// already 0.06 off), for one integer multiply instead of a double multiply and
// its range reduction.  A workgroup asks for all its elements first (up to four
// units a thread), forms the cosines and sines of its rows once in LDS while
// they come, and all the heads of those rows read them: the bound is the read
// and the write of the rows.  16384 rows of 20 heads of 64, bf16: 16.5 us (5.1
// TB/s, a copy's rate; one unit at a time behind the angles 28); 4099 rows of 6
// heads of 96, fp32: 5.1; 104 rows with the append: 4.0, a launch.
#include <math.h>

#include "lanes.h"

using namespace sj;

namespace {

constexpr int RT = 256;
constexpr int RPAIRS = 1024;  // at most this many (row, pair) angles of a workgroup in LDS
constexpr int RU = 4;         // units of a thread

// one frequency per thread, in double
__global__ void k_rope_frequencies(uint64_t* turns, int half, sj_rope_scaling s) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= half) return;
  const double d = 2.0 * half;
  double lt = log((double)s.theta);
  if (s.kind == SJ_ROPE_SCALE_BASE && half > 1) lt += log((double)s.factor) * d / (d - 2.0);
  double f = exp(-2.0 * i / d * lt);
  const double tau = 6.283185307179586476925286766559;
  if (s.kind == SJ_ROPE_SCALE_LINEAR) f /= (double)s.factor;
  if (s.kind == SJ_ROPE_SCALE_PARTS) {
    const double n = (double)s.context * f / tau;
    double g = (n - (double)s.slow_turns) / ((double)s.fast_turns - (double)s.slow_turns);
    g = g < 0.0 ? 0.0 : g > 1.0 ? 1.0 : g;
    f = f * (g + (1.0 - g) / (double)s.factor);
  }
  double t = f / tau;
  t -= floor(t);
  turns[i] = (uint64_t)(t * 18446744073709551616.0);
}

// where a group of heads of a row comes from and goes to
struct RopeSeg {
  const void* x;
  long ldx;
  void* y;
  long ldy;
  int heads;   // heads of this segment
  int rotate;  // 0: copied
};

struct RopeArgs {
  RopeSeg seg[3];
  int nseg;
  long rows;
  int heads;  // of all segments
  int D, half, layout;
  const int32_t* positions;
  const int32_t* slots;  // null: every row counts
  long nslots;
  const uint64_t* turns;
  float amplitude, sign;
  int rb;  // rows of a workgroup
  int rot_units, units, per_row;  // units of a head's rotated part, of a head, of a row
  Div d_half, d_units, d_row;
};

// EL elements of T as they lie (element-aligned: the hardware takes
// global vectors at any element alignment)
template <typename T, int EL>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
  T v[EL];
};
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16_t v) { return bf2f(v); }
__device__ __forceinline__ void from_f(float v, float& o) { o = v; }
__device__ __forceinline__ void from_f(float v, bf16_t& o) { o = f2bf(v); }

// EL: elements of a unit.  Interleaved: a unit is EL / 2 pairs, or EL copied
// columns.  Half: a unit is EL first and EL second elements of pairs, or EL
// copied columns.  The rounding is sj_rope's: stored values in, fp32 products,
// one rounding to the storage type.
template <typename T, int EL, bool HALF>
__global__ __launch_bounds__(RT) void k_rope_rows(RopeArgs a) {
  typedef Pack<T, EL> P;
  __shared__ float2 cs[RPAIRS];
  const int t = threadIdx.x, half = a.half;
  // blocks of rows; where a row has more units than a workgroup takes, rb is 1
  // and blockIdx.y counts its parts
  const long r0 = (long)blockIdx.x * a.rb;
  const int nr = (int)(a.rows - r0 < a.rb ? a.rows - r0 : a.rb);
  const int total = nr * a.per_row, u0 = blockIdx.y * (RT * RU) + t;
  P lo[RU], hi[RU];
  T* y[RU];      // where the unit goes; null: nowhere
  int pair[RU];  // its angles, -1: copied
#pragma unroll
  for (int j = 0; j < RU; j++) {
    const int i = u0 + RT * j;
    y[j] = nullptr;
    pair[j] = -1;
    if (i >= total) continue;
    const int r = div(i, a.d_row), hu = i - r * a.per_row, head = div(hu, a.d_units), u = hu - head * a.units;
    const long row = r0 + r;
    RopeSeg sg = a.seg[0];
    int h = head;
    long dst = row;
    if (a.nseg > 1) {  // q | k | v
      const int sl = a.slots[row];
      if (sl < 0 || sl >= a.nslots) continue;  // a padded row: nothing of it is written
      if (h >= sg.heads) {
        h -= sg.heads;
        sg = a.seg[1];
        if (h >= sg.heads) h -= sg.heads, sg = a.seg[2];
        dst = sl;
      }
    }
    const T* x = (const T*)sg.x + row * sg.ldx + (long)h * a.D;
    const int o = !HALF || u < a.rot_units ? u * EL : 2 * half + (u - a.rot_units) * EL;
    y[j] = (T*)sg.y + dst * sg.ldy + (long)h * a.D + o;
    lo[j] = *(const P*)(x + o);
    if (HALF && u < a.rot_units) hi[j] = *(const P*)(x + o + half);
    if (u < a.rot_units) pair[j] = sg.rotate ? r * half + (HALF ? u * EL : u * (EL / 2)) : HALF ? -2 : -1;
  }
  for (int i = t; i < nr * half; i += RT) {
    const int r = div(i, a.d_half), p = i - r * half;
    const uint64_t ph = (uint64_t)(int64_t)a.positions[r0 + r] * a.turns[p];
    float s, c;
    sincospif((float)(int32_t)(ph >> 32) * 4.656612873077393e-10f, &s, &c);  // half turns: 2^-31
    cs[i] = make_float2(c * a.amplitude, s * a.amplitude * a.sign);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < RU; j++) {
    if (!y[j]) continue;
    if (pair[j] >= 0) {
      const float2* c = cs + pair[j];
      if constexpr (HALF) {
#pragma unroll
        for (int e = 0; e < EL; e++) {
          const float va = to_f(lo[j].v[e]), vb = to_f(hi[j].v[e]);
          const float2 q = c[e];
          from_f(va * q.x - vb * q.y, lo[j].v[e]);
          from_f(va * q.y + vb * q.x, hi[j].v[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < EL / 2; e++) {
          const float va = to_f(lo[j].v[2 * e]), vb = to_f(lo[j].v[2 * e + 1]);
          const float2 q = c[e];
          from_f(va * q.x - vb * q.y, lo[j].v[2 * e]);
          from_f(va * q.y + vb * q.x, lo[j].v[2 * e + 1]);
        }
      }
    }
    *(P*)y[j] = lo[j];
    if (HALF && pair[j] != -1) *(P*)(y[j] + half) = hi[j];
  }
}

template <typename T, int EL>
void launch_el(hipStream_t s, const RopeArgs& a, dim3 grid) {
  if (a.layout == SJ_ROPE_HALF)
    k_rope_rows<T, EL, true><<<grid, RT, 0, s>>>(a);
  else if constexpr (EL > 1)
    k_rope_rows<T, EL, false><<<grid, RT, 0, s>>>(a);
}

int launch(hipStream_t s, RopeArgs& a, int dtype) {
  const int width = dtype == SJ_BF16 ? 8 : 4;
  int el = width;  // the widest unit that divides the head, its rotated part and (half layout) each half
  const int part = a.layout == SJ_ROPE_HALF ? a.half : 2 * a.half;
  while (el > 1 && (a.D % el || part % el)) el >>= 1;
  const int unit = a.layout == SJ_ROPE_HALF ? 2 * el : el;  // columns of a rotated unit
  a.rot_units = 2 * a.half / unit;
  a.units = a.rot_units + (a.D - 2 * a.half) / el;
  a.per_row = a.heads * a.units;
  // as many rows as a workgroup has units and angles for, but few enough that
  // a short call reaches every CU
  a.rb = RT * RU / a.per_row;
  if (a.half && a.rb > RPAIRS / a.half) a.rb = RPAIRS / a.half;
  while (a.rb > 1 && (a.rows + a.rb - 1) / a.rb < 512) a.rb = (a.rb + 1) / 2;
  if (a.rb < 1) a.rb = 1;
  a.d_half = make_div(a.half ? a.half : 1);
  a.d_units = make_div(a.units);
  a.d_row = make_div(a.per_row);
  const dim3 grid((unsigned)((a.rows + a.rb - 1) / a.rb), (unsigned)(a.rb > 1 ? 1 : (a.per_row + RT * RU - 1) / (RT * RU)));
  if (dtype == SJ_BF16) {
    if (el == 8) launch_el<bf16_t, 8>(s, a, grid);
    else if (el == 4) launch_el<bf16_t, 4>(s, a, grid);
    else if (el == 2) launch_el<bf16_t, 2>(s, a, grid);
    else launch_el<bf16_t, 1>(s, a, grid);
  } else {
    if (el == 4) launch_el<float, 4>(s, a, grid);
    else if (el == 2) launch_el<float, 2>(s, a, grid);
    else launch_el<float, 1>(s, a, grid);
  }
  SJ_LAUNCH_CHECK("rope rows");
  return SJ_OK;
}

bool head_ok(long head_dim, long rotary_dim, int layout) {
  return head_dim > 0 && head_dim % 2 == 0 && head_dim <= 1024 && rotary_dim >= 0 && rotary_dim % 2 == 0 &&
         rotary_dim <= head_dim && (layout == SJ_ROPE_INTERLEAVED || layout == SJ_ROPE_HALF);
}

}  // namespace

extern "C" int sj_rope_frequencies(void* stream, uint64_t* turns, long rotary_dim, const sj_rope_scaling* scaling) {
  SJ_REQUIRE(turns && scaling && rotary_dim > 0 && rotary_dim % 2 == 0 && rotary_dim <= 1024,
             "rope frequencies: rotary width %ld", rotary_dim);
  const sj_rope_scaling s = *scaling;
  SJ_REQUIRE(s.kind >= SJ_ROPE_SCALE_NONE && s.kind <= SJ_ROPE_SCALE_PARTS, "rope frequencies: scaling kind %d", s.kind);
  SJ_REQUIRE(isfinite(s.theta) && s.theta > 0.f && (s.kind == SJ_ROPE_SCALE_NONE || (isfinite(s.factor) && s.factor > 0.f)),
             "rope frequencies: theta %g, factor %g", (double)s.theta, (double)s.factor);
  SJ_REQUIRE(s.kind != SJ_ROPE_SCALE_PARTS || (isfinite(s.context) && s.context > 0.f && isfinite(s.fast_turns) &&
                                               isfinite(s.slow_turns) && s.fast_turns > s.slow_turns),
             "rope frequencies: original context %g, turns %g .. %g", (double)s.context, (double)s.slow_turns,
             (double)s.fast_turns);
  const int half = (int)(rotary_dim / 2);
  k_rope_frequencies<<<(half + 63) / 64, 64, 0, (hipStream_t)stream>>>(turns, half, s);
  SJ_LAUNCH_CHECK("rope frequencies");
  return SJ_OK;
}

extern "C" int sj_rope_rows(void* stream, const void* x, long ldx, void* y, long ldy, int dtype, long rows, long heads,
                            long head_dim, long rotary_dim, int layout, const int32_t* positions,
                            const uint64_t* turns, float amplitude, int inverse) {
  SJ_REQUIRE(dtype == SJ_F32 || dtype == SJ_BF16, "rope rows dtype %d", dtype);
  SJ_REQUIRE(head_ok(head_dim, rotary_dim, layout), "rope rows: head width %ld, rotary width %ld, layout %d", head_dim,
             rotary_dim, layout);
  SJ_REQUIRE(rows >= 0 && heads > 0 && heads <= 16384 && ldx >= heads * head_dim && ldy >= heads * head_dim,
             "rope rows dimensions");
  if (rows == 0) return SJ_OK;
  SJ_REQUIRE(x && y && positions && (turns || rotary_dim == 0), "rope rows: null");
  SJ_REQUIRE(x != y || ldx == ldy || rows == 1, "rope rows: in place with strides %ld and %ld", ldx, ldy);
  SJ_REQUIRE(rows < 1L << 24, "rope rows: %ld rows", rows);
  RopeArgs a = {};
  a.seg[0] = RopeSeg{x, ldx, y, ldy, (int)heads, 1};
  a.nseg = 1;
  a.rows = rows;
  a.heads = (int)heads;
  a.D = (int)head_dim;
  a.half = (int)(rotary_dim / 2);
  a.layout = layout;
  a.positions = positions;
  a.turns = turns;
  a.amplitude = amplitude;
  a.sign = inverse ? -1.f : 1.f;
  return launch((hipStream_t)stream, a, dtype);
}

extern "C" int sj_paged_append(void* stream, const void* q, long ldq, const void* k, long ldk, const void* v, long ldv,
                               int dtype, long rows, long hq, long hk, long head_dim, long rotary_dim, int layout,
                               const int32_t* positions, const int32_t* slots, const uint64_t* turns, float amplitude,
                               void* q_out, long ldqo, void* k_cache, void* v_cache, long ldkv, long cache_slots) {
  SJ_REQUIRE(dtype == SJ_F32 || dtype == SJ_BF16, "paged append dtype %d", dtype);
  SJ_REQUIRE(head_ok(head_dim, rotary_dim, layout), "paged append: head width %ld, rotary width %ld, layout %d",
             head_dim, rotary_dim, layout);
  SJ_REQUIRE(rows >= 0 && hq >= 0 && hk > 0 && hq <= 16384 && hk <= 16384 && ldq >= hq * head_dim &&
                 ldqo >= hq * head_dim && ldk >= hk * head_dim && ldv >= hk * head_dim && ldkv >= hk * head_dim &&
                 cache_slots >= 0,
             "paged append dimensions");
  if (rows == 0) return SJ_OK;
  SJ_REQUIRE(k && v && positions && slots && (turns || rotary_dim == 0) && k_cache && v_cache && (hq == 0 || (q && q_out)),
             "paged append: null");
  SJ_REQUIRE(hq == 0 || q != q_out || ldq == ldqo || rows == 1, "paged append: queries in place with strides %ld and %ld",
             ldq, ldqo);
  SJ_REQUIRE(rows < 1L << 24, "paged append: %ld rows", rows);
  RopeArgs a = {};
  a.seg[0] = RopeSeg{q, ldq, q_out, ldqo, (int)hq, 1};
  a.seg[1] = RopeSeg{k, ldk, k_cache, ldkv, (int)hk, 1};
  a.seg[2] = RopeSeg{v, ldv, v_cache, ldkv, (int)hk, 0};
  a.nseg = 3;
  a.rows = rows;
  a.heads = (int)(hq + 2 * hk);
  a.D = (int)head_dim;
  a.half = (int)(rotary_dim / 2);
  a.layout = layout;
  a.positions = positions;
  a.slots = slots;
  a.nslots = cache_slots;
  a.turns = turns;
  a.amplitude = amplitude;
  a.sign = 1.f;
  return launch((hipStream_t)stream, a, dtype);
}
