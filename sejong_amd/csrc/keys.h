// Places of keys in pages and tiles, right up to the last of 2^31 - 1 keys: a
// tile may reach past them, so places of keys are unsigned.  Host code too.
#pragma once
#include <stdint.h>

#ifdef __HIP__
#define SJ_ANYWHERE __host__ __device__ __forceinline__
#else
#define SJ_ANYWHERE inline
#endif

namespace sj {

// n / d for n < 2^31: mul = floor(2^32 (2^shift - d) / d) + 1 with 2^shift >=
// d; the added n is the 33rd bit of 2^32 + mul
struct Div {
  uint32_t mul, shift;
};
inline Div make_div(uint32_t d) {
  Div r = {0, 0};
  while ((1ul << r.shift) < d) r.shift++;
  r.mul = (uint32_t)((((1ul << r.shift) - d) << 32) / d + 1);
  return r;
}
SJ_ANYWHERE int div(uint32_t n, Div d) { return (int)(((uint32_t)(((uint64_t)d.mul * n) >> 32) + n) >> d.shift); }

// the tiles of `tile` keys that `keys` >= 0 of them take
SJ_ANYWHERE int tiles_of(int keys, int tile) { return (int)(((uint32_t)keys + (uint32_t)(tile - 1)) / (uint32_t)tile); }
// the i-th key of the tile that begins at base; below hi it is a key
SJ_ANYWHERE uint32_t key_at(int base, int i) { return (uint32_t)base + (uint32_t)i; }
SJ_ANYWHERE bool is_key(uint32_t j, int hi) { return j < (uint32_t)hi; }
// its place in its page
SJ_ANYWHERE int in_page(uint32_t j, Div d_page, int page_size) {
  return (int)(j - (uint32_t)div(j, d_page) * (uint32_t)page_size);
}

}  // namespace sj
