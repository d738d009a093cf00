// A paged key-value cache for many sequences: the plan of one step (block
// tables, positions and slots from the requests' lengths) and the attention
// of the step's tokens over the pages (no counterpart in the reference, whose
// cache holds one sequence: model lib.rs:36-50, architecture.rs:428-533).
#include <math.h>

#include "lanes.h"

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

// A wave's walk.  DC: the head in units of 32 columns; heads between the sizes
// are walked as the next one, their missing columns read again and multiplied
// by 0 (64 requests of 2048 keys, 16/4 heads, bf16: heads of 104 57 us, of 128
// 54, of 160 106, of 192 111, of 256 121).  E: elements of 16
// bytes, KT: keys of a tile, NC: 16-byte chunks that a lane holds of a row.
template <typename T, int DC>
struct Walk {
  static constexpr bool BF = sizeof(T) == 2;
  static constexpr int DP = 32 * DC, E = BF ? 8 : 4;
  // 8 KB of keys a tile, and as much of values; wide heads by what the
  // products take at least (32 keys in bf16, 16 in fp32)
  static constexpr int KT = BF ? (DC == 1 ? 128 : DC == 2 ? 64 : 32) : (DC == 1 ? 64 : DC == 2 ? 32 : 16), KS = KT / 16;
  static constexpr int NC = DP / (4 * E);
  // fp32 V: a lane takes VW columns of a key, 16 lanes NV blocks of them
  static constexpr int VW = BF ? 1 : (DC == 1 ? 2 : 4), NV = BF ? 1 : DP / (16 * VW);
  static constexpr int NO = DP / 16;            // output tiles of 16 columns
  static constexpr int STRIDE = DP + 8;         // bf16 V tile in LDS: rows 16 bytes apart in the banks
  static constexpr int LDS = BF ? (KT * STRIDE * 2 > 64 * DP ? KT * STRIDE * 2 : 64 * DP) : 64 * DP;  // >= 16 x DP floats
  // chunks that may lie past the head
  static constexpr int FIRST_TAIL = DC == 1 ? 0 : DC == 8 ? NC / 2 : BF ? DC - 1 : (DC == 4 ? 4 : NC - 2);

  u32x4 q[NC];
  u32x4 k[KS][NC];
  u32x4 v[BF ? KS : 4 * KS][BF ? NC : (NV * VW + 3) / 4];
  f32x4 o[NO];
  float m, l;
  int pid[KS], sl[KS];
  uint32_t absent;  // fp32: of the lane's V keys (4g + i of each 16), those without a slot

  __device__ __forceinline__ void start(const PagedArgs& a, int row, int kh, int qt, int lane) {
    const int col = lane & 15, g = lane >> 4, h = qt * 16 + col;
    const T* x = (const T*)a.q + (long)row * a.ldq + ((long)kh * a.G + h) * a.D;
#pragma unroll
    for (int c = 0; c < NC; c++) {
      const int d = (4 * c + g) * E;
      q[c] = h < a.G && d < a.D ? load16(x + d) : u32x4{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int i = 0; i < NO; i++) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.f;
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
  // S^T of the tile, the running maximum, and P in place of S
  __device__ __forceinline__ void scores(const PagedArgs& a, f32x4 (&p)[KS], int lane) {
    const int g = lane >> 4;
    absent = 0;
#pragma unroll
    for (int s = 0; s < KS; s++) {
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NC; c++) {
        u32x4 kk = k[s][c];
        if (c >= FIRST_TAIL && (4 * c + g) * E >= a.D) kk = u32x4{0u, 0u, 0u, 0u};
        if constexpr (BF) {
          acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kk), __builtin_bit_cast(bf16x8, q[c]),
                                                        acc, 0, 0, 0);
        } else {
#pragma unroll
          for (int e = 0; e < 4; e++)
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kk[e]), __uint_as_float(q[c][e]), acc, 0, 0, 0);
        }
      }
      const uint64_t good = __ballot(sl[s] >= 0);
      if ((good & 0xffffu) != 0xffffu) {
        absent |= ((uint32_t)(~good >> (4 * g)) & 15u) << (4 * s);
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (!((good >> (4 * g + i)) & 1)) acc[i] = -INFINITY;
      }
      p[s] = acc;
    }
    float t = -INFINITY;
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int i = 0; i < 4; i++) t = fmaxf(t, p[s][i]);
    t = fmaxf(t, __shfl_xor(t, 16, 64));
    t = fmaxf(t, __shfl_xor(t, 32, 64));
    const float mn = fmaxf(m, t);
    // no key with a share so far: the reference is 0, and every power 0.  The
    // difference first, then the scale: s * c - m * c in one fused step would
    // keep the rounding of m * c, at large scores more than the powers' range
    const float c = a.scale, ref = mn == -INFINITY ? 0.f : mn;
    const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - ref) * c);
    m = mn;
    float sum = 0.f;
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        p[s][i] = __builtin_amdgcn_exp2f((p[s][i] - ref) * c);
        sum += p[s][i];
      }
    l = l * alpha + sum;  // this lane's keys alone: joined in finish()
#pragma unroll
    for (int i = 0; i < NO; i++) o[i] *= alpha;
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
  __device__ __forceinline__ void sums(const bf16_t* tile, const f32x4 (&p)[KS], int lane) {
    if constexpr (BF) {
      const int g = lane >> 4, e = (lane >> 2) & 3, c4 = 4 * (lane & 3);
#pragma unroll
      for (int s = 0; s < KS; s += 2) {
        u32x4 ph, pl;
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const float x = p[s + h][2 * i], y = p[s + h][2 * i + 1];
            const uint32_t w = cvt2(x, y);
            ph[2 * h + i] = w;
            pl[2 * h + i] = cvt2(x - __uint_as_float(w << 16), y - __uint_as_float(w & 0xffff0000u));
          }
#pragma unroll
        for (int d = 0; d < NO; d++) {
          s16x4 r[2];
#pragma unroll
          for (int h = 0; h < 2; h++)
            r[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_s16x4*)(tile + (16 * (s + h) + 4 * g + e) * STRIDE + 16 * d + c4));
          const bf16x8 vt = __builtin_bit_cast(bf16x8, __builtin_shufflevector(r[0], r[1], 0, 1, 2, 3, 4, 5, 6, 7));
          o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt, __builtin_bit_cast(bf16x8, ph), o[d], 0, 0, 0);
          o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt, __builtin_bit_cast(bf16x8, pl), o[d], 0, 0, 0);
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
      for (int s = 0; s < KS; s++)
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int b = 0; b < NV; b++)
#pragma unroll
            for (int t = 0; t < VW; t++)
              o[b * VW + t] =
                  __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[4 * s + i][b][t]), p[s][i], o[b * VW + t], 0, 0, 0);
    }
  }
  // tiles t0, t0 + step, .. below t1 of the keys [lo, hi)
  __device__ __forceinline__ void run(const PagedArgs& a, const int32_t* pages, int kh, int lo, int hi, int t0, int t1,
                                      int step, bf16_t* tile, int lane) {
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
      f32x4 p[KS];
      scores(a, p, lane);
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
      sums(tile, p, lane);
      __builtin_amdgcn_wave_barrier();
      if constexpr (!BF) {
        if (next) load_v(a, V, lane);
      }
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
  }
  // four columns of this lane's query: i-th quad of the lane, its first column
  static constexpr int QUADS = DP / 16;
  __device__ __forceinline__ int quad(int i, int lane, f32x4& x) const {
    const int g = lane >> 4;
    if constexpr (BF) {
      x = o[i];
      return 16 * i + 4 * g;
    } else if constexpr (VW == 4) {
      const int b = i >> 2, e = i & 3;
#pragma unroll
      for (int t = 0; t < 4; t++) x[t] = o[4 * b + t][e];
      return 64 * b + 16 * g + 4 * e;
    } else {
#pragma unroll
      for (int t = 0; t < 4; t++) x[t] = o[t & 1][2 * i + (t >> 1)];
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

constexpr int direct_waves(int dc) { return dc == 8 ? 4 : 8; }  // 256 registers a lane at most hold 8

// The waves of a workgroup join what each summed of one walk: rows of sums in
// each wave's LDS part, maxima and sums of shares beside.  NW: as many waves
// as there can be, nw of them here.
struct Shares {
  float m[8][16], l[8][16];
};
template <typename T, int DC>
__device__ __forceinline__ void leave(const Walk<T, DC>& wk, Shares& sh, uint8_t* lds, int n, int w, int lane) {
  typedef Walk<T, DC> W;
  const int q = lane & 15;
  if (lane < 16) sh.m[w][lane] = wk.m, sh.l[w][lane] = wk.l;
  float* mine = (float*)(lds + w * W::LDS);
#pragma unroll
  for (int i = 0; i < W::QUADS; i++) {
    f32x4 x;
    const int d = wk.quad(i, lane, x);
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
template <typename T, int DC, int NW>
__device__ __forceinline__ Total joined(const PagedArgs& a, const Shares& sh, const uint8_t* lds, int nw, int r, int d) {
  typedef Walk<T, DC> W;
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
  SJ_REQUIRE(q != o || ldq == ldo || rows == 1, "paged attention: in place with strides %ld and %ld", ldq, ldo);
  const size_t need = sj_paged_attention_workspace_bytes(rows, hq, hk, head_dim);
  SJ_REQUIRE(((uintptr_t)workspace & 15) == 0, "paged attention: the workspace is not 16-byte aligned");
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
  a.G = (int)(hq / hk);
  a.QT = (a.G + 15) / 16;
  SJ_REQUIRE(rows <= (1L << 23) / (hk * a.QT), "paged attention: %ld rows of %ld heads", rows, hk);
  a.d_page = make_div((uint32_t)page_size);
  a.d_heads = make_div((uint32_t)(hk * a.QT));
  a.d_tiles = make_div((uint32_t)a.QT);
  a.d_quads = make_div((uint32_t)(head_dim / 4 > 0 ? head_dim / 4 : 1));
  long most = ldt * page_size;
  if (window > 0 && window < most) most = window;
  hipStream_t s = (hipStream_t)stream;
  if (int st = dtype == SJ_BF16 ? attend<bf16_t>(s, a, most, workspace) : attend<float>(s, a, most, workspace)) return st;
  SJ_LAUNCH_CHECK("paged attention");
  return SJ_OK;
}
