"""Places of keys in tiles and pages (csrc/keys.h, which needs no HIP) at the
largest sizes that the paged calls take, against whole numbers without a limit:
compiled here as host code that traps on a signed overflow."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INT_MAX = 2 ** 31 - 1

PROGRAM = r"""
#include <cstdio>
#include "keys.h"

int main() {
  int lo, hi, page, tile;
  while (scanf("%d %d %d %d", &lo, &hi, &page, &tile) == 4) {
    const sj::Div d = sj::make_div((uint32_t)page);
    const int tiles = sj::tiles_of(hi - lo, tile);
    printf("%d", tiles);
    if (tiles > 0) {  // the last tile's keys
      const int base = lo + (tiles - 1) * tile;
      for (int i = 0; i < tile; i++) {
        const uint32_t j = sj::key_at(base, i);
        if (sj::is_key(j, hi)) printf(" %d:%d", sj::div(j, d), sj::in_page(j, d, page));
      }
    }
    printf("\n");
  }
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    where = tmp_path_factory.mktemp("keys")
    src, exe = where / "keys.cpp", where / "keys"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-ftrapv", "-I", os.path.join(ROOT, "sejong_amd", "csrc"), str(src), "-o",
                    str(exe)], check=True)
    return str(exe)


@pytest.mark.parametrize("page", [1, 2, 7, 16, 24, 129, 2 ** 20, 2 ** 30, INT_MAX])
def test_places_of_the_last_keys(program, page):
    """No key past the table's last position, whatever is left of the last tile; every tile counted."""
    last = INT_MAX // page * page  # the table's positions
    cases = [(lo, hi, page, tile) for tile in (16, 32, 64, 128, 512) for hi in (0, 1, page, 1000, last - 1, last)
             for lo in {0, hi, max(hi - 1, 0), max(hi - 100, 0), max(hi - 3000, 0)} if 0 <= lo <= hi <= last]
    out = subprocess.run([program], input="".join("%d %d %d %d\n" % c for c in cases), check=True, capture_output=True,
                         text=True, timeout=60).stdout.splitlines()
    assert len(out) == len(cases)
    for (lo, hi, page, tile), line in zip(cases, out):
        tiles = -(-(hi - lo) // tile)
        keys = range(lo + (tiles - 1) * tile, hi) if tiles else ()
        assert line.split() == [str(tiles)] + ["%d:%d" % (j // page, j % page) for j in keys], (lo, hi, page, tile)
