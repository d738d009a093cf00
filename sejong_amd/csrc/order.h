// Entries of a row of logits in registers, their order as keys, and the places
// of a few keys among each other.
#pragma once
#include <math.h>

#include "lanes.h"

namespace sj {

constexpr float LOG2E = 1.4426950408889634f;

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
template <typename T, int EE>
struct Unit;
template <int EE>
struct Unit<float, EE> {
  static constexpr int E = EE;
  struct __attribute__((packed, aligned(4))) Raw { float v[E]; } r;
  __device__ __forceinline__ float get(int i) const { return r.v[i]; }
  __device__ __forceinline__ void set(int i, float x) { r.v[i] = x; }
};
template <int EE>
struct Unit<bf16_t, EE> {
  static constexpr int E = EE;
  struct __attribute__((packed, aligned(2))) Raw { uint32_t v[E / 2]; } r;
  __device__ __forceinline__ float get(int i) const {
    const uint32_t w = r.v[i >> 1];
    return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
  }
  __device__ __forceinline__ void set(int i, float x) {
    uint32_t& w = r.v[i >> 1];
    w = i & 1 ? (w & 0xffffu) | ((uint32_t)f2bf(x) << 16) : (w & 0xffff0000u) | f2bf(x);
  }
};
template <typename T>
constexpr int WIDE = 16 / (int)sizeof(T);  // entries of 16 bytes
__device__ __forceinline__ float at_f32(const float* x, long i) { return x[i]; }
__device__ __forceinline__ float at_f32(const bf16_t* x, long i) { return bf2f(x[i]); }

// The place of each of the n keys of `keys` (LDS) among them, f(place, key) for
// the first `top`: four lanes of a group's NT threads count for one key.
template <int NT, class F>
__device__ __forceinline__ void rank(const u64* keys, int n, int top, int t, F f) {
  for (int i = t >> 2; i < n; i += NT / 4) {
    const u64 k = keys[i];
    uint32_t place = 0;
#pragma unroll 4
    for (int c = t & 3; c < n; c += 4) place += keys[c] > k;
    place += dpp<0xB1>(place);
    place += dpp<0x4E>(place);
    if ((t & 3) == 0 && (int)place < top) f((int)place, k);
  }
}
__device__ __forceinline__ u64 larger_of(u64 a, u64 b) { return a > b ? a : b; }

}  // namespace sj
