// Attention over the pages of requests that share the beginning of their
// sequences: beams of one prompt, several answers to it, a long document that
// many ask about (no counterpart in the reference, whose cache holds one
// sequence: model lib.rs:36-50).
#include <type_traits>

#include "paged_walk.h"

using namespace sj;

namespace {

//   o = (sum_shared + sum_own) / (l_shared + l_own), both relative to the
//   larger of the two maxima
//
// The keys that the rows of a group share are walked once for all of them: the
// query heads of a KV head of all the group's rows are columns.  Up to 32 of
// them are one walk (two MFMA tiles on one key's loads), whose waves take the
// key tiles in turn; more are blocks of 128, whose waves take 32 columns each
// of the same key tiles.  Every row's own keys are a walk of their own, as in
// paged.hip.  The shared walks lie in a line of places, and every workgroup
// takes an equal piece of it; the rows' own walks lie in another, and every wave
// takes an equal piece of that (these are short, and mostly waiting: a wave needs
// nobody to join with).  So few long prefixes and many short tails fill the chip
// alike.  What was summed of a walk goes to the workspace; a second launch joins
// the parts of each row's two walks.
//
// Small calls go through sj_paged_attention, each row by itself (FEW): together 4
// rows over 960 shared keys (6/2 heads of 64, bf16) take 14.8 us, 1.6 to launch,
// 3.3 for the lists, a walk's chain of page, keys and products, 4.5 for the join;
// alone 10.5.  24 groups of 5 rows over up to 6000 keys (16/4 heads of 64, fp32) take 36.5 us,
// 12 of them their 61 MB at a copy's rate: each wave waits for two or three tiles.
// 64 rows over 16384 keys (32/8 heads of 128, bf16) take 60 us, where their 91 MB
// are 18 and their products, P as two planes, 18: the walks' launch 50 (the lists
// 3, the shared walks 37 to 41, the multiplying waves' own instructions 21 of them,
// own walks 6), the join of 34 MB of parts 10.  One plane would round P to 8 bits,
// and took 2 us less.
//
// A group's prefix is walked whether or not any row shares it: within a window
// that begins behind position 0 no row does, and each walks its window alone (32
// rows over 16384 keys, 32/8 heads of 128, a window of 1024 48 us, by
// sj_paged_attention 23; of 8192 142 and 123).

constexpr int CT = 2, COLS = 16 * CT, BLOCK = 4 * COLS;
constexpr int WIDE_PLACE = 64;  // keys of a place of a walk whose waves go by columns
constexpr int MAX_ROWS = 2048, MAX_GROUPS = 256;  // what LDS lists beside two stages of tiles
constexpr int GROUPS_OF_WAVES = 512;  // workgroups, at most
// Elements of keys and values that the rows read of as long sequences as the table
// holds, if each reads its own: up to here they do (us, for the rows together and
// alone: 4 rows over 960 keys, 2 KV heads of 64, 1 M, 14.8 and 10.5; 128 rows of
// that, 34 M, 17.3 and 12.5; 16 rows over 1024, 8 heads of 128, 42 M, 18.6 and
// 23.2; 8 rows over 2048, 38 M, 21.4 and 23.0).  One number for both types, though
// fp32 would change later: 8 groups of 5 rows over up to 2000 keys, 4 heads of 64,
// 47 M, 20.5 and 15.6; 24 over 1000, 70 M, 23.7 each.
constexpr double FEW = 33554432.0;

struct SharedArgs {
  PagedArgs p;
  const int32_t *starts, *group_starts, *prefix;
  int groups;
  Div d_group;  // by G
  // left for the join by the first workgroup
  int4* row_info;    // first own key, group (-1: alone), first place in units of the row's walks, places of a walk
  int4* group_info;  // [2 * groups]: first place, places of a walk, columns of a block, first slot; first row, slots of
                     // a KV head, blocks, -
  int2* line;        // places of a workgroup's piece of the shared walks, of a wave's of the own ones
  float *lead_part, *own_part;  // slots: of 32 columns; of the heads of a row's walk
  int lead_slot, own_slot;
};

// index of the last of n <= 64 STEP ascending values that is at or below y (below
// 0 if none is): counted by STEPs, then within
template <int STEP>
__device__ __forceinline__ int last_at(const int* v, int n, int y, int lane) {
  const int far = STEP * lane;
  const int c = STEP * (__popcll(__ballot(far < n && v[min(far, n - 1)] <= y)) - 1);
  return c + __popcll(__ballot(lane < STEP && c + lane < n && v[max(min(c + lane, n - 1), 0)] <= y)) - 1;
}

// -------------------------------------------------------- staged key tiles
//
// 64 keys and their values go through LDS (two stages), and each wave
// multiplies all of them with its own 32 columns: a key is read once for 128
// columns, and with neighbouring lanes along its row.  (Operands loaded straight
// from memory have neighbouring lanes on different keys, each an access of its
// own to the first cache: 60 a load, which was all the time of 64 rows over
// 16384 keys.)  A key's chunk c of 16 bytes lies at position c ^ turn(key) of its
// row, so that the lanes of a read meet all banks: eight keys of one chunk (K)
// and the quarters of four rows (V, transposed by ds_read_b64_tr_b16).  The
// running maximum stays until a score passes it by 8 powers of two: the sums have
// the room, and the outputs are rarely scaled.
// over the four lanes that hold a column
__device__ __forceinline__ float column_max(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float column_sum(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

template <int DC>
struct Staged {
  static constexpr int POS = DC == 1 ? 4 : DC == 2 ? 8 : 16, RB = 16 * POS;  // chunks and bytes of a row in LDS
  static constexpr int KT = 64, KS = KT / 16, TILE = KT * RB, STAGE = 2 * TILE, LDS = 2 * STAGE;
  static constexpr int MINE = KT / 4, ROWS = 1024 / RB, LOADS = MINE / ROWS;  // keys a wave brings, rows of a load
  static constexpr int NO = 2 * DC;

  u32x4 q[CT][DC];
  f32x4 o[CT][NO];
  float m[CT], l[CT];
  u32x4 k[LOADS], v[LOADS];
  int pid, sl;

  static constexpr int QUADS = NO;
  __device__ __forceinline__ int quad(int ct, int i, int lane, f32x4& x) const {
    x = o[ct][i];
    return 16 * i + 4 * (lane >> 4);
  }
  static __device__ __forceinline__ int turn(int row) {
    return DC == 1   ? (((row >> 1) & 1) << 1) | ((row >> 2) & 1)
           : DC == 2 ? ((row & 3) << 1) | ((row >> 2) & 1)
                     : (((row >> 3) & 1) << 3) | ((row & 3) << 1) | ((row >> 2) & 1);
  }
  __device__ __forceinline__ void start(const PagedArgs& a, int ct, const bf16_t* x, bool has, int lane) {
    const int g = lane >> 4;
#pragma unroll
    for (int c = 0; c < DC; c++) {
      const int d = (4 * c + g) * 8;
      q[ct][c] = has && d < a.D ? load16(x + d) : u32x4{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int i = 0; i < NO; i++) o[ct][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    m[ct] = -INFINITY;
    l[ct] = 0.f;
  }
  // the page of one of the keys that this wave brings of tile t
  __device__ __forceinline__ void look(const PagedArgs& a, const int32_t* pages, int t, int hi, int w, int lane) {
    const uint32_t j = key_at(t * KT, MINE * w + (lane & (MINE - 1)));
    pid = is_key(j, hi) ? pages[div(j, a.d_page)] : -1;
  }
  __device__ __forceinline__ void place(const PagedArgs& a, int t, int w, int lane) {
    const uint32_t j = key_at(t * KT, MINE * w + (lane & (MINE - 1)));
    sl = (uint32_t)pid < (uint32_t)a.pages ? pid * a.P + in_page(j, a.d_page, a.P) : -1;
  }
  // a key without a slot reads slot 0
  __device__ __forceinline__ void load(const PagedArgs& a, const bf16_t* K, const bf16_t* V, int lane) {
#pragma unroll
    for (int i = 0; i < LOADS; i++) {
      const int row = ROWS * i + lane / POS, d = 8 * (lane % POS);
      const long at = (long)max(__shfl(sl, row, 64), 0) * a.ldkv + (d < a.D ? d : 0);
      k[i] = load16(K + at);
      v[i] = load16(V + at);
    }
  }
  // to a stage, columns past the head and values of keys without a slot as zeros
  // (whatever lies there counts 0 times 0); and which keys there are
  __device__ __forceinline__ void store(const PagedArgs& a, uint8_t* stage, uint32_t* valid, int w, int lane) {
    const uint32_t there = (uint32_t)__ballot(sl >= 0) & ((1u << MINE) - 1);
    if (lane == 0) valid[w] = there;
#pragma unroll
    for (int i = 0; i < LOADS; i++) {
      const int row = ROWS * i + lane / POS;
      uint8_t* to = stage + (MINE * w + row) * RB + 16 * ((lane % POS) ^ turn(MINE * w + row));
      *(u32x4*)to = 8 * (lane % POS) < a.D ? k[i] : u32x4{0u, 0u, 0u, 0u};
      *(u32x4*)(to + TILE) = (there >> row) & 1 ? v[i] : u32x4{0u, 0u, 0u, 0u};
    }
  }
  __device__ __forceinline__ void multiply(const PagedArgs& a, const uint8_t* stage, const uint32_t* valid, int nt, int lane) {
    const int g = lane >> 4, k15 = lane & 15, tk = turn(k15);
    const u32x4 there = *(const u32x4*)valid;
    const uint8_t* krow = stage + k15 * RB;
    f32x4 p[CT][KS];
    // the next 16 keys are on their way while these are multiplied
    u32x4 kk[2][DC];
    auto keys = [&](int s) {
#pragma unroll
      for (int c = 0; c < DC; c++) kk[s & 1][c] = *(const u32x4*)(krow + 16 * s * RB + 16 * ((4 * c + g) ^ tk));
    };
    keys(0);
#pragma unroll
    for (int s = 0; s < KS; s++) {
      if (s + 1 < KS) keys(s + 1);
      __builtin_amdgcn_sched_barrier(0);  // the compiler would put each read before its use
#pragma unroll
      for (int ct = 0; ct < CT; ct++) p[ct][s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < DC; c++)
#pragma unroll
        for (int ct = 0; ct < CT; ct++)
          p[ct][s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kk[s & 1][c]),
                                                             __builtin_bit_cast(bf16x8, q[ct][c]), p[ct][s], 0, 0, 0);
    }
    if ((there[0] & there[1] & there[2] & there[3]) != 0xffffu)
#pragma unroll
      for (int s = 0; s < KS; s++)
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (!((there[s] >> (4 * g + i)) & 1))
#pragma unroll
            for (int ct = 0; ct < CT; ct++) p[ct][s][i] = -INFINITY;
    const float c = a.scale;
    float top[CT];
    bool passed = false;
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
      float t = -INFINITY;
#pragma unroll
      for (int s = 0; s < KS; s++)
#pragma unroll
        for (int i = 0; i < 4; i++) t = fmaxf(t, p[ct][s][i]);
      top[ct] = column_max(t);
      passed |= (top[ct] - m[ct]) * c > 8.f;
    }
    if (__any(passed)) {
#pragma unroll
      for (int ct = 0; ct < CT; ct++) {
        const float mn = fmaxf(m[ct], top[ct]), ref = mn == -INFINITY ? 0.f : mn;
        const float alpha = m[ct] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m[ct] - ref) * c);
        m[ct] = mn;
        l[ct] *= alpha;
#pragma unroll
        for (int i = 0; i < NO; i++) o[ct][i] *= alpha;
      }
    }
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
      const float ref = m[ct] == -INFINITY ? 0.f : m[ct];
      float sum = 0.f;
#pragma unroll
      for (int s = 0; s < KS; s++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          p[ct][s][i] = __builtin_amdgcn_exp2f((p[ct][s][i] - ref) * c);
          sum += p[ct][s][i];
        }
      l[ct] += sum;  // this lane's keys alone: joined in run()
    }
    const int e = (lane >> 2) & 3, tv = turn(4 * g + e), half = 8 * (lane & 1), odd = (lane >> 1) & 1;
    const uint8_t* vrow = stage + TILE + (4 * g + e) * RB + half;
    bf16x8 vt[2];
    auto values = [&](int n) {  // n-th of the products: 32 keys, 16 columns
      const int s = 2 * (n / NO), d = n % NO;
      s16x4 r[2];
#pragma unroll
      for (int h = 0; h < 2; h++)
        r[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vrow + 16 * (s + h) * RB + 16 * ((2 * d + odd) ^ tv)));
      vt[n & 1] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(r[0], r[1], 0, 1, 2, 3, 4, 5, 6, 7));
    };
    values(0);
    u32x4 ph[CT], pl[CT];
#pragma unroll
    for (int n = 0; n < KS / 2 * NO; n++) {
      const int s = 2 * (n / NO), d = n % NO;
      if (d == 0) {
#pragma unroll
        for (int ct = 0; ct < CT; ct++)
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
      if (n + 1 < KS / 2 * NO) values(n + 1);
#pragma unroll
      for (int ct = 0; ct < CT; ct++)
        o[ct][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt[n & 1], __builtin_bit_cast(bf16x8, ph[ct]), o[ct][d], 0, 0, 0);
#pragma unroll
      for (int ct = 0; ct < CT; ct++)
        o[ct][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt[n & 1], __builtin_bit_cast(bf16x8, pl[ct]), o[ct][d], 0, 0, 0);
    }
  }
  // tiles t0 .. t1 - 1 of the keys [0, hi); every wave of the workgroup, those
  // without columns (nt 0) too.  valid: [2][4] words of LDS
  __device__ __forceinline__ void run(const PagedArgs& a, const int32_t* pages, int kh, int hi, int t0, int t1, uint8_t* lds,
                                      uint32_t (*valid)[4], int w, int lane, int nt) {
    const bf16_t* K = (const bf16_t*)a.k + (long)kh * a.D;
    const bf16_t* V = (const bf16_t*)a.v + (long)kh * a.D;
    auto fetch = [&](int t) {  // its pages have been asked for; asks for the next one's
      place(a, t, w, lane);
      load(a, K, V, lane);
      if (t + 1 < t1) look(a, pages, t + 1, hi, w, lane);
    };
    look(a, pages, t0, hi, w, lane);
    fetch(t0);
    __syncthreads();  // the walk before has read its tiles
    store(a, lds, valid[0], w, lane);
    if (t0 + 1 < t1) fetch(t0 + 1);
    __syncthreads();
    for (int t = t0; t < t1; t++) {
      const int now = (t - t0) & 1;
      if (nt) multiply(a, lds + now * STAGE, valid[now], nt, lane);
      if (t + 1 == t1) break;
      // the other stage was read before the last barrier
      store(a, lds + (now ^ 1) * STAGE, valid[now ^ 1], w, lane);
      if (t + 2 < t1) fetch(t + 2);
      __syncthreads();
    }
#pragma unroll
    for (int ct = 0; ct < CT; ct++) l[ct] = column_sum(l[ct]);
  }
};

// v, of which the compiler knows nothing: what comes of it is formed here, not
// before the loop, where it would hold registers through the other walks
__device__ __forceinline__ int here(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// workgroups a CU holds (by registers)
template <typename T>
constexpr int per_cu(int dc) { return dc == 8 || (dc == 4 && sizeof(T) == 4) ? 1 : 2; }

// whether blocks of columns go over staged tiles (else their waves load operands)
template <typename T, int DC>
constexpr bool STAGES = sizeof(T) == 2 && DC <= 4;
template <typename T, int DC>
constexpr int tile_bytes() {
  const int walks = 4 * Walk<T, DC>::LDS;
  if constexpr (STAGES<T, DC>)
    return Staged<DC>::LDS > walks ? Staged<DC>::LDS : walks;
  else
    return walks;
}

template <typename T, int DC>
__global__ __launch_bounds__(256, per_cu<T>(DC)) void k_shared_walks(SharedArgs s) {
  typedef Walk<T, DC, CT> WL;
  typedef Walk<T, DC> W;
  const PagedArgs& a = s.p;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ Shares sh;
  // requests, rows, places, slots and keys of the groups
  __shared__ int g_request[MAX_GROUPS + 1], g_row[MAX_GROUPS + 1], g_pre[MAX_GROUPS + 1], g_sub[MAX_GROUPS],
      g_keys[MAX_GROUPS];
  __shared__ int pre[MAX_ROWS + 1];  // the places before a row
  __shared__ __attribute__((aligned(16))) uint32_t valid[2][4];
  __shared__ int ws[2][4];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, nb = a.HK * a.QT, ng = s.groups;
  const int most = (int)(a.ldt * a.P);
  constexpr int PLACE = 4 * W::KT;  // keys of a place of a row's own walk: four tiles

  // the rows' positions and requests, asked for early (what row_range reads)
  constexpr int HELD = MAX_ROWS / 256;
  const int per_row = (a.rows + 255) / 256;
  int held_pos[HELD], held_owner[HELD];
#pragma unroll
  for (int i = 0; i < HELD; i++) {
    const int r = t * per_row + i;
    const bool in = i < per_row && r < a.rows;
    held_pos[i] = in ? a.positions[r] : -1;
    held_owner[i] = in && a.owners ? a.owners[r] : r;
  }
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
  struct Group {
    int cols, wide, block, blocks, places;  // wide: waves by columns; places: of a walk
  };
  auto group_of = [&](int g) {
    Group r = {0, 0, COLS, 0, 0};
    const int keys = g_keys[g];
    if (none || keys <= 0 || keys > most) return r;
    r.cols = (g_row[g + 1] - g_row[g]) * a.G;
    r.wide = r.cols > COLS;
    r.block = r.wide ? BLOCK : COLS;
    r.blocks = (r.cols + r.block - 1) / r.block;
    r.places = tiles_of(keys, r.wide ? WIDE_PLACE : 4 * WL::KT);
    return r;
  };
  auto slots_of = [](const Group& r) { return (r.cols + COLS - 1) / COLS; };  // of a KV head
  {
    constexpr int MOST = MAX_GROUPS / 256;
    const int per = (ng + 255) / 256;
    int places[MOST], slots[MOST], mine = 0, slot = 0;
#pragma unroll
    for (int i = 0; i < MOST; i++) {
      const int g = t * per + i;
      places[i] = slots[i] = 0;
      if (i < per && g < ng) {
        const Group r = group_of(g);
        slots[i] = a.HK * slots_of(r);
        places[i] = a.HK * r.blocks * r.places;
      }
      mine += places[i];
      slot += slots[i];
    }
    int at = (int)scan_add((uint32_t)mine), at_slot = (int)scan_add((uint32_t)slot);
    if (lane == 63) ws[0][w] = at, ws[1][w] = at_slot;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; i++)
      if (i < w) at += ws[0][i], at_slot += ws[1][i];
    if (t == 255) g_pre[ng] = at;
    at -= mine;
    at_slot -= slot;
#pragma unroll
    for (int i = 0; i < MOST; i++) {
      const int g = t * per + i;
      if (i < per && g < ng) {
        g_pre[g] = at;
        g_sub[g] = at_slot;
        at += places[i];
        at_slot += slots[i];
      }
    }
    __syncthreads();
  }
  const int lead = g_pre[ng];

  // Whether row r, of a request in group g, walks its group's keys: it sees all
  // of them.  Among groups without requests the last at or before the owner is
  // the one that has it.
  auto shares = [&](int g, int r, int owner, int lo, int hi) {
    return lo == 0 && owner >= g_request[g] && owner < g_request[g + 1] && r >= g_row[g] && r < g_row[g + 1] &&
           g_keys[g] > 0 && g_keys[g] <= hi;
  };
  // the rows: where their own keys begin
  {
    int n[HELD], group[HELD], from[HELD], mine = 0;
#pragma unroll
    for (int i = 0; i < HELD; i++) {
      n[i] = from[i] = 0;
      group[i] = -1;
      const int r = t * per_row + i;
      int lo, hi;
      if (i < per_row && r < a.rows && range_of(a, held_pos[i], held_owner[i], lo, hi)) {
        if (lead > 0) {
          int g = 0, e = ng;  // the last group that begins at or before the owner
          while (e - g > 1) {
            const int m = (g + e) >> 1;
            if (g_request[m] <= held_owner[i]) g = m; else e = m;
          }
          if (shares(g, r, held_owner[i], lo, hi)) group[i] = g, lo = g_keys[g];
        }
        from[i] = lo;
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
    for (int i = 0; i < HELD; i++) {
      const int r = t * per_row + i;
      if (i < per_row && r < a.rows) {
        pre[r] = at;
        if (blockIdx.x == 0) s.row_info[r] = make_int4(from[i], group[i], at, n[i]);
        at += n[i];
      }
    }
    __syncthreads();
  }
  // Every workgroup takes both, its shared places and then its waves' own ones,
  // or some take the ones and the others the others, whichever leaves the longest
  // with fewer places (24 groups of 5 fp32 rows: 39 us, apart 36; 48 groups 58 and
  // 50).  Where that is the same, few places and many own walks are better apart
  // (24 groups with up to 1000 own keys a row 44 and 37), else not (100 groups 93
  // and 109; 8 rows over 16384 keys 40 and 43).
  const int own = pre[a.rows] * nb, all = gridDim.x;
  auto each = [](long n, long of) { return (int)((n + of - 1) / of); };
  const int lead_each = each(lead, all), mixed = max(1, each((long)lead + each(own, 4), all));
  const int sum = lead_each + each(own, 4L * all);
  const bool fewer = mixed < sum || (mixed == sum && mixed <= 3 && 2 * (long)own >= all);
  const bool apart = fewer && (own == 0 || each(lead, mixed) < all);
  const int piece = max(1, apart ? mixed : lead_each);
  const int taken = apart ? each(lead, piece) : 0, own_groups = max(all - taken, 1), waves = 4 * own_groups;
  const int own_piece = max(1, each(own, waves));
  if (blockIdx.x == 0) {
    for (int g = t; g < ng; g += 256) {
      const Group r = group_of(g);
      s.group_info[2 * g] = make_int4(g_pre[g], r.places, r.block, g_sub[g]);
      s.group_info[2 * g + 1] = make_int4(g_row[g], slots_of(r), r.blocks, 0);
    }
    if (t == 0) *s.line = make_int2(piece, own_piece);
  }
  const int b = blockIdx.x;
  int x = (int)min((long)lead, (long)b * piece);
  const int e = (int)min((long)lead, (long)x + piece);
  const int quads = a.D / 4, lane0 = lane;
  while (x < e) {
    const int lane = here(lane0);
    const int g = __builtin_amdgcn_readfirstlane(last_at<4>(g_pre, ng, x, lane));
    const Group r = group_of(g);
    const int keys = __builtin_amdgcn_readfirstlane(g_keys[g]), places = r.places, in = x - g_pre[g];
    const int walk = __builtin_amdgcn_readfirstlane(in / places), c0 = in - walk * places, c1 = min(places, c0 + e - x);
    const int kh = walk / r.blocks, cb = walk - kh * r.blocks, r0 = g_row[g];
    const int32_t* pages = a.table + (long)g_request[g] * a.ldt;
    // the query of column c of the group, for this KV head
    auto query = [&](int c) {
      const int row = div(c, s.d_group);
      return (const T*)a.q + (long)(r0 + row) * a.ldq + ((long)kh * a.G + c - row * a.G) * a.D;
    };
    float* part = s.lead_part + (long)(g_sub[g] + kh * slots_of(r) + 4 * b) * s.lead_slot;
    const int first = cb * r.block + (r.wide ? w * COLS : 0), cols = min(max(r.cols - first, 0), COLS), nt = (cols + 15) / 16;
    auto begin = [&](auto& wk) {
#pragma unroll
      for (int ct = 0; ct < CT; ct++) {
        const int c = 16 * ct + (lane & 15);
        wk.start(a, ct, query(first + c), c < cols, lane);
      }
    };
    // a wave's own columns, straight from its registers
    auto put = [&](const auto& wk) {
      typedef std::remove_cv_t<std::remove_reference_t<decltype(wk)>> K;
      // 64 bits: a group's slots pass 2^31 floats at 8.3 M columns of 256; the same for the
      // whole wave, as a vector product cost 64 rows over 16384 keys 1.5 us
      part += (long)__builtin_amdgcn_readfirstlane(4 * cb + w) * s.lead_slot;
#pragma unroll
      for (int ct = 0; ct < CT; ct++) {
        const int c = 16 * ct + (lane & 15);
        if (c >= cols) continue;
        if (lane < 16) *(float2*)(part + 2 * c) = make_float2(wk.m[ct], wk.l[ct]);
#pragma unroll
        for (int i = 0; i < K::QUADS; i++) {
          f32x4 v;
          const int d = wk.quad(ct, i, lane, v);
          if (d < a.D) *(f32x4*)(part + 2 * COLS + c * a.D + d) = v;
        }
      }
    };
    bf16_t* tile = (bf16_t*)(lds + w * WL::LDS);
    const int tiles = tiles_of(keys, WL::KT);
    if (r.wide) {
      if constexpr (STAGES<T, DC>) {
        constexpr int PER = WIDE_PLACE / Staged<DC>::KT;
        Staged<DC> wk;
        begin(wk);
        wk.run(a, pages, kh, keys, PER * c0, min(PER * c1, tiles_of(keys, Staged<DC>::KT)), lds, valid, w, lane, nt);
        put(wk);
      } else {
        constexpr int PER = WIDE_PLACE / WL::KT;
        WL wk;
        begin(wk);
        if (nt) wk.run(a, pages, kh, 0, keys, PER * c0, min(PER * c1, tiles), 1, tile, lane, nt);
        put(wk);
      }
    } else {
      if constexpr (STAGES<T, DC>) __syncthreads();  // a staged walk's tiles have been read
      WL wk;
      begin(wk);
      wk.run(a, pages, kh, 0, keys, 4 * c0 + w, min(4 * c1, tiles), 4, tile, lane, nt);
      part += (long)cb * s.lead_slot;
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
    }
    x += c1 - c0;
  }
  __syncthreads();  // the waves' tiles lie elsewhere in the rows' own walks
  // a wave's piece; those of one workgroup lie apart, so that few walks go over all workgroups
  const int mine = (int)blockIdx.x - taken;
  if (mine < 0) return;
  const int wave = w * own_groups + mine;
  int y = (int)min((long)own, (long)wave * own_piece);
  const int ye = (int)min((long)own, (long)y + own_piece);
  while (y < ye) {
    const int lane = here(lane0);
    const int at = div(y, a.d_heads), row = __builtin_amdgcn_readfirstlane(last_at<32>(pre, a.rows, at, lane));
    const int first = __builtin_amdgcn_readfirstlane(pre[row]), places = __builtin_amdgcn_readfirstlane(pre[row + 1]) - first;
    const int in = y - first * nb, hb = __builtin_amdgcn_readfirstlane(in / places);
    const int c0 = in - hb * places, c1 = min(places, c0 + ye - y);
    const int kh = div(hb, a.d_tiles), qt = hb - kh * a.QT, n = min(16, a.G - qt * 16);
    int owner, lo, hi;
    row_range(a, row, owner, lo, hi);
    owner = __builtin_amdgcn_readfirstlane(owner);
    if (lead > 0) {
      const int g = max(__builtin_amdgcn_readfirstlane(last_at<4>(g_request, ng, owner, lane)), 0);
      if (shares(g, row, owner, lo, hi)) lo = g_keys[g];
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    W wk;
    wk.start(a, row, kh, qt, lane);
    wk.run(a, a.table + (long)owner * a.ldt, kh, lo, hi, 4 * c0, min(4 * c1, tiles_of(hi - lo, W::KT)), 1,
           (bf16_t*)(lds + w * W::LDS), lane);
    float* part = s.own_part + (long)(row * nb + hb + wave) * s.own_slot;
    const int c = lane & 15;
    if (c < n) {
      if (lane < 16) *(float2*)(part + 2 * c) = make_float2(wk.m[0], wk.l[0]);
#pragma unroll
      for (int i = 0; i < W::QUADS; i++) {
        f32x4 v;
        const int d = wk.quad(0, i, lane, v);
        if (d < a.D) *(f32x4*)(part + 32 + c * a.D + d) = v;
      }
    }
    y += c1 - c0;
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
  const int g = info.y;
  int4 group = make_int4(0, 0, 1, 0), more = group;
  if (g >= 0) group = s.group_info[2 * g], more = s.group_info[2 * g + 1];
  const int items = n * quads, span = min(items, 256), shares = 256 / span, t = threadIdx.x, gr = t / span;
  for (int u0 = 0; u0 < items; u0 += span) {
    const int u = u0 + t - gr * span, r = div(min(u, items - 1), a.d_quads), q = min(u, items - 1) - r * quads;
    const bool live = gr < shares && u < items;
    Total v;
    // the parts of a walk at x0 of its line: slot `first` and every `step` slots
    auto add = [&](const float* base, long slot, int first, int step, int piece, int x0, int places, int c, int ncols) {
      if (places == 0) return;
      const int p0 = x0 / piece, parts = (x0 + places - 1) / piece - p0 + 1;
      constexpr int MANY = 8;  // parts asked for at once
      for (int i = gr; i < parts; i += MANY * shares) {
        float2 m[MANY];
        f32x4 o[MANY];
#pragma unroll
        for (int k = 0; k < MANY; k++) {
          const float* p = base + (first + step * (p0 + min(i + k * shares, parts - 1))) * slot;
          m[k] = *(const float2*)(p + 2 * c);
          o[k] = *(const f32x4*)(p + 2 * ncols + c * a.D + 4 * q);
        }
#pragma unroll
        for (int k = 0; k < MANY; k++) v.add(m[k].x, i + k * shares < parts ? m[k].y : 0.f, o[k], a.scale);
      }
    };
    if (live) {
      if (g >= 0) {
        const int at = (row - more.x) * a.G + qt * 16 + r, walk = kh * more.z + at / group.z;
        add(s.lead_part, s.lead_slot, group.w + kh * more.y + at / COLS, 4, line.x, group.x + walk * group.y, group.y,
            at % COLS, COLS);
      }
      add(s.own_part, s.own_slot, row * nb + hb, 1, line.y, info.z * nb + hb * info.w, info.w, r, 16);
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
  // each group's last slot may hold fewer than COLS columns
  const size_t slots = (size_t)hk * (rows * G / COLS + groups);
  l.own = l.lead + 4 * (slots + 4 * GROUPS_OF_WAVES) * l.lead_slot;
  l.bytes = l.own + 4 * ((size_t)rows * hk * QT + 4 * GROUPS_OF_WAVES) * l.own_slot;
  return l;
}
// whether the prefixes are walked for their groups: by sizes alone, too
bool grouped(long rows, long head_dim, long groups) {
  return groups > 0 && groups <= MAX_GROUPS && rows <= MAX_ROWS && head_dim % 8 == 0;
}

template <typename T, int DC>
int launch_walks(hipStream_t st, const SharedArgs& s) {
  constexpr int lds = tile_bytes<T, DC>();
  static sj::OncePerDevice once;
  if (int e = sjh::once_per_device(once, [] {
        SJ_HIP(hipFuncSetAttribute((const void*)k_shared_walks<T, DC>, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
        return SJ_OK;
      }))
    return e;
  k_shared_walks<T, DC><<<256 * per_cu<T>(DC), 256, lds, st>>>(s);
  SJ_LAUNCH_CHECK("paged attention of groups");
  k_shared_join<T><<<(unsigned)((long)s.p.rows * s.p.HK * s.p.QT), 256, 0, st>>>(s);
  SJ_LAUNCH_CHECK("paged attention of groups");
  return SJ_OK;
}
template <typename T>
int launch(hipStream_t st, const SharedArgs& s) {
  const int D = s.p.D;
  if (D <= 32) return launch_walks<T, 1>(st, s);
  if (D <= 64) return launch_walks<T, 2>(st, s);
  if (D <= 96 && sizeof(T) == 2) return launch_walks<T, sizeof(T) == 2 ? 3 : 4>(st, s);
  if (D <= 128) return launch_walks<T, 4>(st, s);
  return launch_walks<T, 8>(st, s);
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
  const size_t need = sj_paged_attention_shared_workspace_bytes(rows, hq, hk, head_dim, groups);
  SJ_REQUIRE(((uintptr_t)workspace & 15) == 0, "paged attention of groups: the workspace is not 16-byte aligned");
  if (need > workspace_bytes || (need && !workspace))
    return sjh::fail(SJ_ERR_CAPACITY, "paged attention of groups workspace: required %zu bytes, available %zu bytes", need,
                     workspace ? workspace_bytes : 0);
  // all places of the line are counted in 31 bits
  const long most = ldt * page_size, seen = window > 0 && window < most ? window : most;
  const double places = ((double)rows * hk * (s.p.QT + s.p.G / (double)COLS) + (double)groups * hk) * (most / 64.0 + 1);
  if (!grouped(rows, head_dim, groups) || places >= 2147483647.0 || 2.0 * rows * hk * seen * head_dim <= FEW)
    return sj_paged_attention(stream, q, ldq, k_cache, v_cache, ldkv, dtype, pages, page_size, table, ldt, requests, owners,
                              positions, rows, hq, hk, head_dim, window, o, ldo, lse, workspace, workspace_bytes);
  const Layout l = layout_of(rows, hq, hk, head_dim, groups);
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
  return dtype == SJ_BF16 ? launch<bf16_t>(st, s) : launch<float>(st, s);
}
