"""The pages' calls at the largest sizes that they take."""
import ctypes

import numpy as np
import pytest

from tests import beam_util as BU
from tests import gpu_util as G
from tests import paged_util as PU
from tests.test_gpu_pages import native

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,width", [("f32", 2 ** 29 + 3), ("bf16", 2 ** 30 + 5)])
def test_copy_of_rows_past_32_bits(dtype, width):
    """A page whose one row is longer than 2^31 bytes: its beginning, its middle, what lies near 2^31 bytes, its end, and
    nothing behind it."""
    size, code, word = (4, 0, np.uint32) if dtype == "f32" else (2, 4, np.uint16)
    rng = np.random.default_rng(width)
    N = native()[0]
    ld = width + 4
    K = G.Dev(2 * ld, dtype)
    at = [0, width // 2, 2 ** 31 // size - 200, width - 40]  # 40 elements each
    parts = rng.integers(1, 2 ** 15, (len(at), 40)).astype(word)
    back = np.full(44, 77, word)

    def up(i, x):
        N.api.sj_upload(K.at(i), ctypes.c_void_p(x.ctypes.data), x.nbytes)

    up(ld + width - 40, back)  # the target's last elements and the four behind them
    for i, x in zip(at, parts):
        up(i, x)
    C = PU.ints([[0, 1, 1]])
    N.api.sj_paged_copy(None, K.p, K.p, ld, code, 1, 0, 2, 1, width, C.p, 1)
    for first in (0, ld):  # the source as it was, the target like it
        for i, x in zip(at, parts):
            got = np.empty_like(x)
            N.api.sj_download(ctypes.c_void_p(got.ctypes.data), K.at(first + i), got.nbytes)
            np.testing.assert_array_equal(got, x)
    N.api.sj_download(ctypes.c_void_p(back.ctypes.data), K.at(ld + width - 40), back.nbytes)
    np.testing.assert_array_equal(back[:40], parts[-1])
    assert (back[40:] == 77).all()


@pytest.mark.parametrize("count,layers", [(2 ** 22 - 1, 1), (2 ** 22 + 1, 1), (2 ** 23 + 5, 3), (2 ** 24, 1), (260_000, 40)])
def test_copies_of_long_lists(count, layers):
    """Lists with more places than one launch has workgroups for, few of them taken: the first, the last, some between."""
    rng = np.random.default_rng(count)
    N = native()[0]
    P, width, taken = 2, 8, 40
    pages = 2 * taken
    copies = np.tile([-1, -1, 0], (count, 1)).astype(np.int32)
    at = np.unique(np.concatenate([[0, count - 1], rng.integers(0, count, taken - 2)]))
    names = rng.permutation(pages)
    copies[at] = np.stack([names[:len(at)], names[taken:taken + len(at)], 1 + np.arange(len(at)) % P], 1)
    kv = [G.rnd((layers, pages * P, width), "bf16", rng) for _ in range(2)]
    K, V = (G.dev(x.ravel(), "bf16") for x in kv)
    C = PU.ints(copies)
    N.api.sj_paged_copy(None, K.p, V.p, width, 4, layers, pages * P * width, pages, P, width, C.p, count)
    for x, d in zip(kv, (K, V)):
        want = BU.copy(x.copy(), copies[at], P, width)
        np.testing.assert_array_equal(d.host(), want.ravel())


@pytest.mark.parametrize("requests", [2 ** 23 + 3, 2 ** 24])
def test_compaction_of_many_requests(requests):
    """As many requests as one launch has workgroups for, and as many as there can be: rows of one page that many share."""
    rng = np.random.default_rng(requests)
    N, lib = native()
    P, pages, after, used = 4, 300, 200, 150
    names = rng.permutation(pages)
    table = names[rng.integers(0, used, requests)].astype(np.int32)
    lengths = rng.integers(0, P + 1, requests).astype(np.int32)
    free = np.concatenate([np.full(used, -1), names[used:]]).astype(np.int32)
    below = free[used:][free[used:] < after]
    moved = np.setdiff1d(np.arange(after, pages), free[used:])
    to = np.arange(pages)
    to[moved] = below[:len(moved)]
    ins = [PU.ints(x) for x in (table, lengths, np.zeros(pages), free, [used])]
    out = PU.ints(np.full(requests + 1, 55))
    shared, listed, copies, summary = (PU.ints(np.full(n, 55)) for n in (pages, pages, 3 * 100, 4))
    need = lib.sj_paged_compact_workspace_bytes(pages, pages)
    ws = G.Dev(need, "u8")
    T, L, S, F, H = (b.p for b in ins)
    N.api.sj_paged_compact(None, T, 1, L, requests, P, pages, after, S, F, pages, H, out.p, shared.p, listed.p, copies.p, 100,
                           summary.p, ws.p, need)
    assert summary.host().tolist() == [len(moved), pages - len(below) + len(moved), 0, len(below) - len(moved)]
    got = out.host()
    assert got[-1] == 55
    np.testing.assert_array_equal(got[:-1], np.where(lengths > 0, to[table], -1))
