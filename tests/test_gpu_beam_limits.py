"""The beam selection at the largest number of rows that it takes of a vocabulary."""
import ctypes

import numpy as np
import pytest

from tests import beam_util as BU
from tests import gpu_util as G
from tests import paged_util as PU
from tests.test_gpu_beam import logits, native

pytestmark = pytest.mark.gpu


def test_four_million_rows_of_more_than_one_slice():
    """2^22 rows of 4097 (34 GB of logits), the first, the last and some prompts between; nothing behind the last."""
    V, beams, keep, block = 4097, 4, 2, 2 ** 14
    rows = 2 ** 22
    groups = rows // beams
    rng = np.random.default_rng(1)
    N, lib = native()
    x = logits(rng, block, V, "bf16")  # row r's are x[r % block]
    raw = (x.astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)
    X = G.Dev(rows * V, "bf16")
    for r in range(0, rows, block):
        N.api.sj_upload(X.at(r * V), ctypes.c_void_p(raw.ctypes.data), raw.nbytes)
    scores = rng.normal(-20, 2, rows).astype(np.float32)
    S = G.dev(scores)
    parents, tokens = (PU.ints(np.full(groups * keep + 1, 55)) for _ in range(2))
    after = G.dev(np.full(groups * keep + 1, 55.0))
    need = lib.sj_beam_select_workspace_bytes(groups, beams, V, keep)
    ws = G.Dev(need + 64, "u8")
    guard = np.full(64, 0xA5, np.uint8)
    N.api.sj_upload(ws.at(need), ctypes.c_void_p(guard.ctypes.data), 64)
    N.api.sj_beam_select(None, X.p, 4, V, groups, beams, V, S.p, None, None, -1, 0.0, keep, parents.p, tokens.p, after.p, None,
                         None, ws.p, need)
    parents, tokens, after = parents.host(), tokens.host(), after.host()
    assert parents[-1] == 55 and tokens[-1] == 55 and after[-1] == 55
    for g in [0, 1, groups // 2 - 1, groups // 2, groups - 2, groups - 1] + rng.integers(0, groups, 20).tolist():
        r = g * beams
        want = BU.select(x[r % block:r % block + beams], scores[r:r + beams].astype(np.float64), beams, keep)
        at = slice(g * keep, (g + 1) * keep)
        np.testing.assert_array_equal(parents[at], want["parents"] + r)
        np.testing.assert_array_equal(tokens[at], want["tokens"])
        # totals of 64 bits, the sum's powers to 7.8e-13, rounded once to fp32
        assert (np.abs(after[at] - want["scores"]) <= np.abs(want["scores"]) * 2.0 ** -24 * 1.001 + 1e-12).all()
    N.api.sj_download(ctypes.c_void_p(guard.ctypes.data), ws.at(need), 64)
    assert (guard == 0xA5).all()
