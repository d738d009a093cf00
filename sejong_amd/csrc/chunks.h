// How a pool's pages and its free list are dealt out to workgroups, where their
// counts lie in the workspace, and what rows of a page are copied as.  Host code
// alone, no HIP.
#pragma once
#include <stddef.h>

namespace sj {

// The workgroups of a launch over n entries: chunks of whole rounds.  Every
// workgroup adds up the counts of those before it, so there are at most
// CHUNKS.
constexpr long CHUNK_ROUND = 1024;  // entries of a workgroup's round
constexpr long CHUNKS = 4096;
struct Chunks {
  long chunk, count;
};
inline Chunks chunks_of(long n) {
  const long rounds = n > CHUNK_ROUND * CHUNKS ? (n + CHUNK_ROUND * CHUNKS - 1) / (CHUNK_ROUND * CHUNKS) : 1;
  return {rounds * CHUNK_ROUND, (n + rounds * CHUNK_ROUND - 1) / (rounds * CHUNK_ROUND)};
}
// The most chunks that n entries or any part of them take: the count falls to
// half where a workgroup begins to take a round more.
inline long chunks_most(long n) {
  const long rounds = (n + CHUNK_ROUND - 1) / CHUNK_ROUND;
  return rounds < CHUNKS ? rounds : CHUNKS;
}

// The compaction's workspace, in places of 4 bytes: where the high pages go, the
// free pages below, the workgroups' counts of those and of the pages that move
// (high pages are any part of the pool).
struct CompactSpace {
  size_t targets, below, moves, all;
};
inline CompactSpace compact_space(long pages, long free_count) {
  CompactSpace s;
  s.targets = (size_t)pages;
  s.below = s.targets + (size_t)free_count;
  s.moves = s.below + (size_t)chunks_of(free_count).count;
  s.all = s.moves + (size_t)chunks_most(pages);
  return s;
}

// A row of `width` elements of `size` bytes: 16-byte units, and elements behind
// them.  Rows may be longer than 2^31 bytes.
struct RowUnits {
  int units, tail;
};
inline RowUnits row_units(long width, long size) {
  const long units = width * size / 16;
  return {(int)units, (int)(width - units * (16 / size))};
}

}  // namespace sj
