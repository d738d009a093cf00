// Sums, maxima and scans over a wave with data-parallel moves (no LDS); the
// meeting of workgroups that each hold a part of a result.
#pragma once
#include "common.h"
#include "keys.h"

namespace sj {

// ------------------------------------------------ reductions and scans
// Four steps within rows of 16 lanes, then the four rows' values as scalars,
// in a fixed order.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true);
}
__device__ __forceinline__ float lane_of(float v, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int lane) {
  return (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
template <typename V, class F>
__device__ __forceinline__ V wave_all(V v, F f) {
  v = f(v, dpp<0xB1>(v));   // lanes 1, 0, 3, 2
  v = f(v, dpp<0x4E>(v));   // lanes 2, 3, 0, 1
  v = f(v, dpp<0x141>(v));  // mirrored within 8
  v = f(v, dpp<0x140>(v));  // mirrored within 16
  return f(f(lane_of(v, 0), lane_of(v, 16)), f(lane_of(v, 32), lane_of(v, 48)));
}
__device__ __forceinline__ float all_max(float v) {
  return wave_all(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float all_min(float v) {
  return wave_all(v, [](float a, float b) { return fminf(a, b); });
}
__device__ __forceinline__ float all_sum(float v) {
  return wave_all(v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ uint32_t all_max(uint32_t v) {
  return wave_all(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
__device__ __forceinline__ unsigned long long all_max(unsigned long long v) {
  const uint32_t hi = all_max((uint32_t)(v >> 32));
  const uint32_t lo = all_max((uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
  return ((unsigned long long)hi << 32) | lo;
}

// inclusive scans: within rows of 16 lanes, then the rows' last values into
// the rows behind
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_or0(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ uint32_t scan_add(uint32_t v) {
  v += dpp_or0<0x111, 0xf>(v);  // from 1, 2, 4, 8 lanes before
  v += dpp_or0<0x112, 0xf>(v);
  v += dpp_or0<0x114, 0xf>(v);
  v += dpp_or0<0x118, 0xf>(v);
  v += dpp_or0<0x142, 0xa>(v);  // lane 15 of rows 0 and 2 to rows 1 and 3
  v += dpp_or0<0x143, 0xc>(v);  // lane 31 to rows 2 and 3
  return v;
}
// of values >= 0
__device__ __forceinline__ int scan_max(int v) {
  v = max(v, dpp_or0<0x111, 0xf>(v));
  v = max(v, dpp_or0<0x112, 0xf>(v));
  v = max(v, dpp_or0<0x114, 0xf>(v));
  v = max(v, dpp_or0<0x118, 0xf>(v));
  v = max(v, dpp_or0<0x142, 0xa>(v));
  v = max(v, dpp_or0<0x143, 0xc>(v));
  return v;
}

// -------------------------------------------------------------- meeting
//
// Parts of a result pass between workgroups (on different XCDs, each with its
// own L2) through relaxed atomics at agent scope, which are coherent by
// themselves.  A part is complete (vmcnt 0) before its flag is set, and its
// flag (vmcnt 0 again) before its workgroup looks at the flags of the others;
// so the one whose flag is set last finds all of them.  Two may both find
// them: they write the same bits.  Nobody waits for anybody.  The workspace is
// the caller's and not cleared, so a set flag is a number of 64 bits that no
// other call has (sjh::call_number); whoever finds all flags clears them, and
// a replayed graph, which keeps its number, starts from cleared flags again.
__device__ __forceinline__ void part_put(unsigned long long* p, unsigned long long v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ unsigned long long part_get(const unsigned long long* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void part_put(float* p, float x, float y) {
  part_put((unsigned long long*)p, ((unsigned long long)__float_as_uint(y) << 32) | __float_as_uint(x));
}
__device__ __forceinline__ float2 part_get(const float* p) {
  const unsigned long long v = part_get((const unsigned long long*)p);
  return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}
// Every thread of the workgroup, after its part_put of part `mine`: whether
// all the parts are complete (then the flags are cleared, and part_get reads
// the others).  flag(i): part i's flag; complete: a word of LDS.
template <class F>
__device__ __forceinline__ bool meet(F flag, int mine, int parts, unsigned long long number, int* complete) {
  const int lane = threadIdx.x & 63;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x < 64) {
    if (lane == 0) part_put(flag(mine), number);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    bool set = true;
    for (int i = lane; i < parts; i += 64) set &= part_get(flag(i)) == number;
    set = __all(set);
    if (lane == 0) *complete = set;
  }
  __syncthreads();
  if (!*complete) return false;
  for (int i = threadIdx.x; i < parts; i += blockDim.x) part_put(flag(i), 0ull);
  return true;
}

}  // namespace sj

namespace sjh {
// a number that no other call has, as far as 64 bits go, and not 0 (capi.hip)
unsigned long long call_number();
}  // namespace sjh
