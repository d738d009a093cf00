// A wave's walk over the pages of a paged key-value cache, and the joins of
// what several waves, workgroups or launches summed of one query.
#pragma once
#include <math.h>

#include "lanes.h"

namespace sj {

// -------------------------------------------------------------- attention
//
//   o = sum_j e^(s_j - m) v_j / l,  m = max s_j,  l = sum_j e^(s_j - m)
//
// One wave walks tiles of 16 to 128 keys of one KV head for up to 16 of its
// query heads at once, with the running maximum and sum of each query: the
// group's query heads are the columns of one MFMA tile, so a key is read once
// for all of them, and padding the group to 16 columns costs matrix time that
// a memory-bound walk has to spare.
//   S^T [keys][queries] = K q^T: the K rows go from memory straight into the
//     operand (lane = key, 16 bytes of the row).
//   O^T [columns][queries] += V^T P^T: a lane holds P^T for the keys 4g .. 4g
//     + 3 of each 16, exactly as S^T left it, so the product takes its keys in
//     that order and P moves nowhere; a query is one lane column in both, so
//     the rescaling by the running maximum needs no exchange either.
// bf16: V^T is read from a tile that the wave keeps in LDS for itself (no
// barriers), with ds_read_b64_tr_b16.  P feeds the product as two bf16 planes:
// one rounding to 8 bits would cost as much as the output's own, the second
// plane costs matrix time that is free here.  fp32: the fp32 MFMA, whose
// operands are single values, takes V as it lies; nothing is rounded.
// The loads of a tile are in flight while the one before is computed, its page
// ids one tile earlier still.  64 requests of 4000 to 16384 keys, 8 KV heads of
// 128, bf16: 2.3 GB in 424 us (5.4 TB/s, above a copy's 5.1); one wave per row
// and head without the matrix cores took 4748.

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
  Div d_page, d_heads, d_tiles, d_quads;  // by P, by HK QT, by QT, by D / 4
  long window;
  float scale;  // log2(e) / sqrt(D): the softmax in powers of two
  int G, QT;    // query heads of a KV head, and their tiles of 16
  // split walks
  unsigned long long* flag;  // [2 * workgroups], of the meetings
  unsigned long long number;
  float* part;  // [2 * workgroups][slot]
  int slot;     // floats of a walk's totals: 16 maxima and sums of shares, min(G, 16) rows of D
};

// the keys that a row at position pos sees, [lo, hi); false for a padded row
__device__ __forceinline__ bool range_of(const PagedArgs& a, int pos, int owner, int& lo, int& hi) {
  if (pos < 0 || owner < 0 || owner >= a.requests) return false;
  const long most = a.ldt * a.P;  // at most 2^31 - 1 (checked on the host)
  hi = (int)(pos + 1L < most ? pos + 1L : most);
  lo = a.window > 0 && pos + 1L > a.window ? (int)(pos + 1L - a.window) : 0;
  if (lo > hi) lo = hi;
  return true;
}
// those of a row, and its request
__device__ __forceinline__ bool row_range(const PagedArgs& a, int row, int& owner, int& lo, int& hi) {
  const int pos = a.positions[row];
  owner = a.owners ? a.owners[row] : row;
  return range_of(a, pos, owner, lo, hi);
}

// 16 bytes at any alignment
struct __attribute__((packed, aligned(2))) Raw16 {
  u32x4 v;
};
struct __attribute__((packed, aligned(2))) Raw8 {
  u32x2 v;
};
__device__ __forceinline__ u32x4 load16(const void* p) { return ((const Raw16*)p)->v; }

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef float f32x2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t cvt2(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2v){a, b}, bf16x2v));
}

// A wave's walk.  CT: the tiles of 16 queries that it serves at once (one key
// tile's loads feed all of them).  DC: the head in units of 32 columns; heads between the sizes
// are walked as the next one, their missing columns read again and multiplied
// by 0 (64 requests of 2048 keys, 16/4 heads, bf16: heads of 104 57 us, of 128
// 54, of 160 106, of 192 111, of 256 121).  E: elements of 16
// bytes, KT: keys of a tile, NC: 16-byte chunks that a lane holds of a row.
template <typename T, int DC, int CT = 1>
struct Walk {
  static constexpr bool BF = sizeof(T) == 2;
  static constexpr int DP = 32 * DC, E = BF ? 8 : 4;
  // 8 KB of keys a tile, and as much of values; wide heads by what the
  // products take at least (32 keys in bf16, 16 in fp32); two tiles of queries at
  // once leave registers for half of the narrowest's
  static constexpr int KT = BF ? (DC == 1 ? (CT == 1 ? 128 : 64) : DC == 2 ? 64 : 32) : (DC == 1 ? 64 : DC == 2 ? 32 : 16), KS = KT / 16;
  static constexpr int NC = DP / (4 * E);
  // fp32 V: a lane takes VW columns of a key, 16 lanes NV blocks of them
  static constexpr int VW = BF ? 1 : (DC == 1 ? 2 : 4), NV = BF ? 1 : DP / (16 * VW);
  static constexpr int NO = DP / 16;            // output tiles of 16 columns
  static constexpr int STRIDE = DP + 8;         // bf16 V tile in LDS: rows 16 bytes apart in the banks
  static constexpr int LDS = BF ? (KT * STRIDE * 2 > 64 * DP ? KT * STRIDE * 2 : 64 * DP) : 64 * DP;  // >= 16 x DP floats
  // chunks that may lie past the head
  static constexpr int FIRST_TAIL = DC == 1 ? 0 : DC == 8 ? NC / 2 : BF ? DC - 1 : (DC == 4 ? 4 : NC - 2);

  u32x4 q[CT][NC];
  u32x4 k[KS][NC];
  u32x4 v[BF ? KS : 4 * KS][BF ? NC : (NV * VW + 3) / 4];
  f32x4 o[CT][NO];
  float m[CT], l[CT];
  int pid[KS], sl[KS];
  uint32_t absent;  // fp32: of the lane's V keys (4g + i of each 16), those without a slot

  // tile ct's query of this lane (lane & 15), at x; has: there is one
  __device__ __forceinline__ void start(const PagedArgs& a, int ct, const T* x, bool has, int lane) {
    const int g = lane >> 4;
#pragma unroll
    for (int c = 0; c < NC; c++) {
      const int d = (4 * c + g) * E;
      q[ct][c] = has && d < a.D ? load16(x + d) : u32x4{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int i = 0; i < NO; i++) o[ct][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    m[ct] = -INFINITY;
    l[ct] = 0.f;
  }
  // the query heads 16 qt .. of KV head kh, of one row
  __device__ __forceinline__ void start(const PagedArgs& a, int row, int kh, int qt, int lane) {
    const int h = qt * 16 + (lane & 15);
    start(a, 0, (const T*)a.q + (long)row * a.ldq + ((long)kh * a.G + h) * a.D, h < a.G, lane);
  }
  // page ids of the tile's keys (lane & 15 of each 16), -1 past the range
  __device__ __forceinline__ void look(const PagedArgs& a, const int32_t* pages, int base, int hi, int lane) {
#pragma unroll
    for (int s = 0; s < KS; s++) {
      const uint32_t j = key_at(base, 16 * s + (lane & 15));
      pid[s] = is_key(j, hi) ? pages[div(j, a.d_page)] : -1;
    }
  }
  __device__ __forceinline__ void place(const PagedArgs& a, int base, int lane) {
#pragma unroll
    for (int s = 0; s < KS; s++) {
      const bool in = (uint32_t)pid[s] < (uint32_t)a.pages;
      sl[s] = in ? pid[s] * a.P + in_page(key_at(base, 16 * s + (lane & 15)), a.d_page, a.P) : -1;
    }
  }
  // a key without a slot reads slot 0 and is masked in scores() and store_v()
  __device__ __forceinline__ void load_k(const PagedArgs& a, const T* K, int lane) {
    const int g = lane >> 4;
#pragma unroll
    for (int s = 0; s < KS; s++) {
      const T* x = K + (long)max(sl[s], 0) * a.ldkv;
#pragma unroll
      for (int c = 0; c < NC; c++) {
        const int d = (4 * c + g) * E;
        k[s][c] = load16(x + (c < FIRST_TAIL || d < a.D ? d : 0));
      }
    }
  }
  __device__ __forceinline__ void load_v(const PagedArgs& a, const T* V, int lane) {
    const int g = lane >> 4;
#pragma unroll
    for (int s = 0; s < KS; s++) {
      if constexpr (BF) {
        const T* x = V + (long)max(sl[s], 0) * a.ldkv;
#pragma unroll
        for (int c = 0; c < NC; c++) {
          const int d = (4 * c + g) * E;
          v[s][c] = load16(x + (c < FIRST_TAIL || d < a.D ? d : 0));
        }
      } else {
        // lane (column block lane & 15, keys 4g + i): one value of each key
        // and column is one operand
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int slot = __shfl(sl[s], 4 * g + i, 64);
          const float* x = (const float*)V + (long)max(slot, 0) * a.ldkv;
          if constexpr (VW == 4) {
#pragma unroll
            for (int b = 0; b < NV; b++) {
              const int d = 64 * b + 4 * (lane & 15);
              v[4 * s + i][b] = load16(x + (d < a.D ? d : 0));
            }
          } else {
            const int d = 2 * (lane & 15);
            const u32x2 y = ((const Raw8*)(x + (d < a.D ? d : 0)))->v;
            v[4 * s + i][0] = u32x4{y[0], y[1], 0u, 0u};
          }
        }
      }
    }
  }
  // S^T of the tile, the running maximum, and P in place of S; nt: the tiles of
  // queries that hold any
  __device__ __forceinline__ void scores(const PagedArgs& a, f32x4 (&p)[CT][KS], int nt, int lane) {
    const int g = lane >> 4;
    absent = 0;
#pragma unroll
    for (int s = 0; s < KS; s++) {
      f32x4 acc[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ct++) acc[ct] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NC; c++) {
        u32x4 kk = k[s][c];
        if (c >= FIRST_TAIL && (4 * c + g) * E >= a.D) kk = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
          if (ct && ct >= nt) continue;
          if constexpr (BF) {
            acc[ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kk),
                                                              __builtin_bit_cast(bf16x8, q[ct][c]), acc[ct], 0, 0, 0);
          } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
              acc[ct] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kk[e]), __uint_as_float(q[ct][c][e]), acc[ct],
                                                             0, 0, 0);
          }
        }
      }
      const uint64_t good = __ballot(sl[s] >= 0);
      if ((good & 0xffffu) != 0xffffu) {
        absent |= ((uint32_t)(~good >> (4 * g)) & 15u) << (4 * s);
#pragma unroll
        for (int ct = 0; ct < CT; ct++)
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (!((good >> (4 * g + i)) & 1)) acc[ct][i] = -INFINITY;
      }
#pragma unroll
      for (int ct = 0; ct < CT; ct++) p[ct][s] = acc[ct];
    }
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
      if (ct && ct >= nt) continue;
      float t = -INFINITY;
#pragma unroll
      for (int s = 0; s < KS; s++)
#pragma unroll
        for (int i = 0; i < 4; i++) t = fmaxf(t, p[ct][s][i]);
      t = fmaxf(t, __shfl_xor(t, 16, 64));
      t = fmaxf(t, __shfl_xor(t, 32, 64));
      const float mn = fmaxf(m[ct], t);
      // no key with a share so far: the reference is 0, and every power 0.  The
      // difference first, then the scale: s * c - m * c in one fused step would
      // keep the rounding of m * c, at large scores more than the powers' range
      const float c = a.scale, ref = mn == -INFINITY ? 0.f : mn;
      const float alpha = m[ct] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m[ct] - ref) * c);
      m[ct] = mn;
      float sum = 0.f;
#pragma unroll
      for (int s = 0; s < KS; s++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          p[ct][s][i] = __builtin_amdgcn_exp2f((p[ct][s][i] - ref) * c);
          sum += p[ct][s][i];
        }
      l[ct] = l[ct] * alpha + sum;  // this lane's keys alone: joined in run()
#pragma unroll
      for (int i = 0; i < NO; i++) o[ct][i] *= alpha;
    }
  }
  // bf16: the V rows to the wave's LDS tile, keys without a slot as zeros
  __device__ __forceinline__ void store_v(bf16_t* tile, int lane) {
    if constexpr (BF) {
      const int g = lane >> 4;
#pragma unroll
      for (int s = 0; s < KS; s++)
#pragma unroll
        for (int c = 0; c < NC; c++)
          *(u32x4*)(tile + (16 * s + (lane & 15)) * STRIDE + (4 * c + g) * 8) =
              sl[s] >= 0 ? v[s][c] : u32x4{0u, 0u, 0u, 0u};
    }
  }
  __device__ __forceinline__ void sums(const bf16_t* tile, const f32x4 (&p)[CT][KS], int nt, int lane) {
    if constexpr (BF) {
      const int g = lane >> 4, e = (lane >> 2) & 3, c4 = 4 * (lane & 3);
#pragma unroll
      for (int s = 0; s < KS; s += 2) {
        u32x4 ph[CT], pl[CT];
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
          if (ct && ct >= nt) continue;
#pragma unroll
          for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const float x = p[ct][s + h][2 * i], y = p[ct][s + h][2 * i + 1];
              const uint32_t w = cvt2(x, y);
              ph[ct][2 * h + i] = w;
              pl[ct][2 * h + i] = cvt2(x - __uint_as_float(w << 16), y - __uint_as_float(w & 0xffff0000u));
            }
        }
#pragma unroll
        for (int d = 0; d < NO; d++) {
          s16x4 r[2];
#pragma unroll
          for (int h = 0; h < 2; h++)
            r[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_s16x4*)(tile + (16 * (s + h) + 4 * g + e) * STRIDE + 16 * d + c4));
          const bf16x8 vt = __builtin_bit_cast(bf16x8, __builtin_shufflevector(r[0], r[1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
          for (int ct = 0; ct < CT; ct++) {
            if (ct && ct >= nt) continue;
            o[ct][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt, __builtin_bit_cast(bf16x8, ph[ct]), o[ct][d], 0, 0, 0);
            o[ct][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt, __builtin_bit_cast(bf16x8, pl[ct]), o[ct][d], 0, 0, 0);
          }
        }
      }
    } else {
      if (__any(absent)) {  // whatever such a slot holds, it counts 0 times 0
#pragma unroll
        for (int i = 0; i < 4 * KS; i++)
          if ((absent >> i) & 1)
#pragma unroll
            for (int b = 0; b < NV; b++) v[i][b] = u32x4{0u, 0u, 0u, 0u};
      }
#pragma unroll
      for (int ct = 0; ct < CT; ct++) {
        if (ct && ct >= nt) continue;
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
          for (int i = 0; i < 4; i++)
#pragma unroll
            for (int b = 0; b < NV; b++)
#pragma unroll
              for (int t = 0; t < VW; t++)
                o[ct][b * VW + t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[4 * s + i][b][t]), p[ct][s][i],
                                                                        o[ct][b * VW + t], 0, 0, 0);
      }
    }
  }
  // tiles t0, t0 + step, .. below t1 of the keys [lo, hi)
  __device__ __forceinline__ void run(const PagedArgs& a, const int32_t* pages, int kh, int lo, int hi, int t0, int t1,
                                      int step, bf16_t* tile, int lane, int nt = CT) {
    if (t0 >= t1) return;
    const T* K = (const T*)a.k + (long)kh * a.D;
    const T* V = (const T*)a.v + (long)kh * a.D;
    const int inc = step * KT;  // keys past hi are masked, and tiles past t1 not taken
    int base = lo + t0 * KT;
    look(a, pages, base, hi, lane);
    place(a, base, lane);
    load_k(a, K, lane);
    load_v(a, V, lane);
    const bool more = t0 + step < t1;
    if (more) look(a, pages, base + inc, hi, lane);
    for (int t = t0; t < t1; t += step) {
      f32x4 p[CT][KS];
      scores(a, p, nt, lane);
      if constexpr (BF) store_v(tile, lane);
      const bool next = t + step < t1;
      if (next) {
        base += inc;
        place(a, base, lane);
        load_k(a, K, lane);
        if constexpr (BF) load_v(a, V, lane);
        if (t + 2 * step < t1) look(a, pages, base + inc, hi, lane);
      }
      __builtin_amdgcn_wave_barrier();
      sums(tile, p, nt, lane);
      __builtin_amdgcn_wave_barrier();
      if constexpr (!BF) {
        if (next) load_v(a, V, lane);
      }
    }
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
      l[ct] += __shfl_xor(l[ct], 16, 64);
      l[ct] += __shfl_xor(l[ct], 32, 64);
    }
  }
  // four columns of this lane's query of tile ct: i-th quad of the lane, its
  // first column
  static constexpr int QUADS = DP / 16;
  __device__ __forceinline__ int quad(int ct, int i, int lane, f32x4& x) const {
    const int g = lane >> 4;
    if constexpr (BF) {
      x = o[ct][i];
      return 16 * i + 4 * g;
    } else if constexpr (VW == 4) {
      const int b = i >> 2, e = i & 3;
#pragma unroll
      for (int t = 0; t < 4; t++) x[t] = o[ct][4 * b + t][e];
      return 64 * b + 16 * g + 4 * e;
    } else {
#pragma unroll
      for (int t = 0; t < 4; t++) x[t] = o[ct][t & 1][2 * i + (t >> 1)];
      return 8 * g + 4 * i;
    }
  }
};

__device__ __forceinline__ float natural_lse(float m, float l, float c) {
  return l == 0.f ? -INFINITY : (m * c + log2f(l)) * 0.6931471805599453f;
}
template <typename T>
__device__ __forceinline__ void put4(T* y, const f32x4& x, float inv) {
  if constexpr (sizeof(T) == 2) {
    struct __attribute__((packed, aligned(2))) P { uint32_t a, b; };
    *(P*)y = P{cvt2(x[0] * inv, x[1] * inv), cvt2(x[2] * inv, x[3] * inv)};
  } else {
    struct __attribute__((packed, aligned(4))) P { float a, b, c, d; };
    *(P*)y = P{x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv};
  }
}

// The waves of a workgroup join what each summed of one walk: rows of sums in
// each wave's LDS part, maxima and sums of shares beside.  NW: as many waves
// as there can be, nw of them here.
struct Shares {
  float m[8][16], l[8][16];
};
template <typename T, int DC, int CT>
__device__ __forceinline__ void leave(const Walk<T, DC, CT>& wk, Shares& sh, uint8_t* lds, int n, int w, int lane, int ct = 0) {
  typedef Walk<T, DC, CT> W;
  const int q = lane & 15;
  if (lane < 16) sh.m[w][lane] = wk.m[ct], sh.l[w][lane] = wk.l[ct];
  float* mine = (float*)(lds + w * W::LDS);
#pragma unroll
  for (int i = 0; i < W::QUADS; i++) {
    f32x4 x;
    const int d = wk.quad(ct, i, lane, x);
    if (q < n) *(f32x4*)(mine + q * W::DP + d) = x;
  }
}
// running totals of one query: the largest maximum M, the sum of shares L and
// four columns s relative to it
struct Total {
  float M = -INFINITY, L = 0.f;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  __device__ __forceinline__ void add(float m, float l, const f32x4& x, float scale) {
    if (l == 0.f) return;  // no key with a share
    // with NaN scores alone there is no maximum: the NaN is in l and x
    const float mn = fmaxf(M, m), f0 = L == 0.f ? 0.f : mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((M - mn) * scale);
    const float f1 = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - mn) * scale);
    s = s * f0 + x * f1;
    L = L * f0 + l * f1;
    M = mn;
  }
};
template <typename T, int DC, int NW, int CT = 1>
__device__ __forceinline__ Total joined(const PagedArgs& a, const Shares& sh, const uint8_t* lds, int nw, int r, int d) {
  typedef Walk<T, DC, CT> W;
  float m[NW], l[NW];
  f32x4 x[NW];
#pragma unroll
  for (int i = 0; i < NW; i++) {
    const int k = i < nw ? i : 0;
    m[i] = sh.m[k][r];
    l[i] = i < nw ? sh.l[k][r] : 0.f;
    x[i] = *(const f32x4*)((const float*)(lds + k * W::LDS) + r * W::DP + d);
  }
  Total t;
#pragma unroll
  for (int i = 0; i < NW; i++) t.add(m[i], l[i], x[i], a.scale);
  return t;
}
template <typename T>
__device__ __forceinline__ void put_result(const PagedArgs& a, int row, int h, int d, const Total& t) {
  put4((T*)a.o + (long)row * a.ldo + (long)h * a.D + d, t.s, t.L == 0.f ? 0.f : 1.f / t.L);
  if (a.lse && d == 0) a.lse[(long)row * a.HQ + h] = natural_lse(t.M, t.L, a.scale);
}

}  // namespace sj

namespace sjh {
// the checks of an attention call's arguments, and the arguments (no rows:
// nothing to do) without those of a split walk
int paged_args(const void* q, long ldq, const void* k_cache, const void* v_cache, long ldkv, int dtype, long pages,
               long page_size, const int32_t* table, long ldt, long requests, const int32_t* owners,
               const int32_t* positions, long rows, long hq, long hk, long head_dim, long window, void* o, long ldo,
               float* lse, sj::PagedArgs& a);
}  // namespace sjh
