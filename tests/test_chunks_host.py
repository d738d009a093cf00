"""How pages are dealt out to workgroups, where their counts lie, and what rows are
copied as (csrc/chunks.h, which needs no HIP), compiled here as host code that
traps on a signed overflow; and the workspace queries that go by it."""
import os
import subprocess

import pytest

from sejong_amd import _native as N

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROUND, CHUNKS = 1024, 4096
EDGE = ROUND * CHUNKS  # above this many entries a workgroup takes a round more

PROGRAM = r"""
#include <cstdio>
#include "chunks.h"

int main(int argc, char**) {
  long pages, after, listed;
  if (argc > 1) {
    long width, size;
    while (scanf("%ld %ld", &width, &size) == 2) {
      const sj::RowUnits r = sj::row_units(width, size);
      printf("%d %d\n", r.units, r.tail);
    }
    return 0;
  }
  while (scanf("%ld %ld %ld", &pages, &after, &listed) == 3) {
    const sj::Chunks high = sj::chunks_of(pages - after), list = sj::chunks_of(listed);
    const sj::CompactSpace s = sj::compact_space(pages, listed);
    printf("%ld %ld %ld %ld %zu %zu %zu %zu\n", high.chunk, high.count, list.chunk, list.count, s.targets, s.below, s.moves,
           s.all);
  }
}
"""

SIZES = [1, 2, 1023, 1024, 1025, 400001] + [k * EDGE + d for k in (1, 2, 3, 7, 511) for d in (-1024, -1, 0, 1, 5000, 10 ** 6)]


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    where = tmp_path_factory.mktemp("chunks")
    src, exe = where / "chunks.cpp", where / "chunks"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-ftrapv", "-I", os.path.join(ROOT, "sejong_amd", "csrc"), str(src), "-o",
                    str(exe)], check=True)
    return str(exe)


def test_every_array_of_a_compaction_has_room(program):
    """Pools around the sizes where a workgroup takes a round more, shrunk to any size: the high pages' marks, the list's
    targets and both counts end before the next array begins, and the last before the workspace does."""
    cases = [(pages, pages - high, listed) for pages in SIZES for high in SIZES + [0] if high <= pages
             for listed in (0, 1, pages // 3, pages)]
    out = subprocess.run([program], input="".join("%d %d %d\n" % c for c in cases), check=True, capture_output=True,
                         text=True, timeout=60).stdout.splitlines()
    assert len(out) == len(cases)
    for (pages, after, listed), line in zip(cases, out):
        high_chunk, high_count, list_chunk, list_count, targets, below, moves, end = map(int, line.split())
        for n, chunk, count in ((pages - after, high_chunk, high_count), (listed, list_chunk, list_count)):
            assert chunk % ROUND == 0 and count <= CHUNKS and (count - 1) * chunk < n <= count * chunk or n == count == 0
        assert pages - after <= targets and targets + listed <= below, (pages, after, listed)
        assert below + list_count <= moves and moves + high_count <= end, (pages, after, listed)
        assert N.load().sj_paged_compact_workspace_bytes(pages, listed) == 4 * end


def test_a_larger_pool_needs_no_less():
    """What holds a pool holds every part of it, which is what the high pages are."""
    lib = N.load()
    needs = [lib.sj_paged_compact_workspace_bytes(n, 100) for n in sorted(SIZES)]
    assert needs == sorted(needs)
    for pages in SIZES:
        for high in SIZES:
            if high <= pages:
                moves = -(-high // (-(-high // EDGE) * ROUND))  # workgroups that count the high pages
                assert lib.sj_paged_compact_workspace_bytes(pages, 0) >= 4 * (pages + moves)


def test_units_of_rows_of_any_length(program):
    """Rows of 2^31 bytes and more too: the units and the elements behind them are the row."""
    cases = [(w, size) for size in (2, 4) for w in list(range(1, 40)) + [k * 2 ** 29 + d for k in (1, 2, 3) for d in range(-9, 10)]
             + [2 ** 31 - 1 - d for d in range(9)]]
    out = subprocess.run([program, "rows"], input="".join("%d %d\n" % c for c in cases), check=True, capture_output=True,
                         text=True, timeout=60).stdout.splitlines()
    for (width, size), line in zip(cases, out, strict=True):
        assert line.split() == [str(width * size // 16), str(width * size % 16 // size)], (width, size)
