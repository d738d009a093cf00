"""Attention over shared prefixes of prompts (many tokens a request), and at the
largest sizes that it takes."""
import ctypes

import numpy as np
import pytest

from tests import gpu_util as G
from tests import paged_util as PU
from tests.test_gpu_paged import HALF_ULP, native
from tests.test_gpu_shared import Shared

pytestmark = pytest.mark.gpu


def bf16_bits(x):
    return (np.asarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint16)


def test_columns_of_a_group_past_32_bits_of_the_workspace():
    """2048 rows of 4096 query heads on one KV head of 256: the group's sums lie more than 2^31 floats apart."""
    rows, hq, D, P, prefix, some = 2048, 4096, 256, 16, 48, 64
    rng = np.random.default_rng(1)
    N, lib = native()
    shared = prefix // P
    table = np.concatenate([np.tile(np.arange(shared), (rows, 1)), shared + np.arange(rows)[:, None]], 1)
    pages = shared + rows
    k, v = (G.rnd((pages * P, 1, D), "bf16", rng) for _ in range(2))
    q = G.rnd((some, hq, D), "bf16", rng, 1.5)  # row r's is q[r % some]
    positions = np.full(rows, prefix)  # the prefix and one key of its own
    Q, O, L = G.Dev(rows * hq * D, "bf16"), G.Dev(rows * hq * D, "bf16"), G.Dev(rows * hq, "f32")
    raw = bf16_bits(q)
    for r in range(0, rows, some):
        N.api.sj_upload(Q.at(r * hq * D), ctypes.c_void_p(raw.ctypes.data), raw.nbytes)
    K, V = G.dev(k.ravel(), "bf16"), G.dev(v.ravel(), "bf16")
    T, Z, F, X = PU.ints(table), PU.ints(positions), PU.ints([0, rows]), PU.ints([prefix])
    need = lib.sj_paged_attention_shared_workspace_bytes(rows, hq, 1, D, 1)
    assert 4 * rows * hq * (D + 2) > 2 ** 33  # bytes of the group's sums
    ws = G.Dev(need, "u8")
    N.api.sj_paged_attention_shared(None, Q.p, hq * D, K.p, V.p, D, 4, pages, P, T.p, shared + 1, rows, None, Z.p, rows, None,
                                    F.p, X.p, 1, hq, 1, D, 0, O.p, hq * D, L.p, ws.p, need)
    for r in (0, 1000, 2031, 2032, 2047):  # the last ones' sums lie behind 2^31 floats
        got, lse = np.empty(hq * D, np.uint16), np.empty(hq, np.float32)
        N.api.sj_download(ctypes.c_void_p(got.ctypes.data), O.at(r * hq * D), got.nbytes)
        N.api.sj_download(ctypes.c_void_p(lse.ctypes.data), L.at(r * hq), lse.nbytes)
        got = (got.astype(np.uint32) << 16).view(np.float32).astype(np.float64).reshape(hq, D)
        (o, ls, mag, err), = PU.attention(q[r % some][None], k, v, table, P, pages, [r], positions[:1], hq, 1, D)
        # as for smaller calls: the score's rounding twice, 16 bits of the shares, one rounding to the storage type
        tol = (2 * err[:, None] + 2.0 ** -15) * mag + np.abs(o) * HALF_ULP["bf16"] * 1.01 + 1e-38
        assert (np.abs(got - o) <= tol).all(), r
        assert (np.abs(lse - ls) <= err * 2 + 2.0 ** -21 * (1 + np.abs(ls))).all(), r


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("groups,per,hq,hk,D,P,window", [([(96, [40, 17, 33]), (50, [64])], 17, 6, 2, 64, 16, 0),
                                                         ([(300, [128, 130])], 128, 4, 2, 64, 24, 0),
                                                         ([(64, [70] * 4)], 64, 8, 2, 128, 16, 0),
                                                         ([(1000, [200])], 200, 3, 1, 32, 7, 0),
                                                         ([(96, [40, 50])], 33, 6, 2, 64, 16, 60),
                                                         ([(96, [40, 50])], 33, 16, 1, 256, 16, 120)])
def test_prompts_over_a_shared_prefix(dtype, groups, per, hq, hk, D, P, window):
    """Requests with many tokens at once: every one sees the prefix and its request's tokens up to itself."""
    a = Shared(per + D, dtype, hq, hk, D, P, groups, alone=[per, per + 9], per=per, pad=2, window=window)
    a.upload().run().check()
    first = a.O.host().copy(), a.L.host().copy()
    for b in (a.O, a.L):
        b.upload(np.full(b.n, 55.0))
    a.run()
    assert all((x == y.host()).all() for x, y in zip(first, (a.O, a.L)))  # every output again, the same bits


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_more_rows_of_prompts_than_are_walked_together(dtype):
    """2048 rows in one group, and a few more, which attend alone."""
    for per in (256, 257):
        Shared(per, dtype, 2, 1, 32, 16, [(40, [per] * 8)], per=per).upload().run().check()
