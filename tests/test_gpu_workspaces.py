"""Calls write nothing behind the bytes that their workspace query names."""
import numpy as np
import pytest

from tests import gpu_util as G
from tests.test_gpu_beam import Select, logits
from tests.test_gpu_pages import Compact, Fork, state
from tests.test_gpu_paged import Attend
from tests.test_gpu_shared import Shared

pytestmark = pytest.mark.gpu
GUARD = 16384


class Guarded:
    """A call object's workspace, of just the bytes asked for, with a known pattern behind them."""

    def __init__(self, call):
        self.call, self.need = call, call.need
        call.ws = G.Dev(self.need + GUARD, "u8").upload(np.repeat([0xFF, 0xA5], [self.need, GUARD]).astype(np.uint8))

    def run(self):
        self.call.run()
        want = self.call.check()
        assert (self.call.ws.host()[self.need:] == 0xA5).all()
        return want


@pytest.mark.parametrize("pages,after", [(4_194_305, 64), (4_200_000, 10_000), (4_300_000, 500_000), (5_000_003, 1_000_000),
                                         (4_194_304, 64), (400_001, 300_001), (8193, 4000), (60, 40)])
def test_compaction(pages, after):
    """Pools in which a workgroup of the high pages' launch takes one round while one of the whole pool takes two."""
    rng = np.random.default_rng(after)
    R, P, cols = 4, 4, 7
    names = rng.permutation(pages)
    table, lengths = names[:R * cols].reshape(R, cols), np.full(R, P * cols)
    free = np.concatenate([np.full(R * cols, -1), names[R * cols:]])
    c = Compact(lengths, table, np.zeros(pages, int), free, R * cols, pages, P, after, 5000)
    assert Guarded(c).run()["status"] == 0


@pytest.mark.parametrize("groups,beams,P,hi,spare", [(1, 1, 16, 40, 4), (16, 4, 16, 900, 200), (300, 8, 16, 200, 20000),
                                                     (2000, 5, 16, 64, 12000), (2, 2, 16, 100, 4_194_305), (2, 2, 16, 100, 16400)])
def test_fork(groups, beams, P, hi, spare):
    rng = np.random.default_rng(groups)
    lengths, table, shared, free, head, pages = state(rng, groups, beams, P, hi, spare)
    parents = np.arange(groups)[:, None] * beams + rng.integers(0, beams, (groups, beams))
    assert Guarded(Fork(parents.ravel(), lengths, table, shared, free, head, pages, P)).run()["status"] == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V,groups,beams,keep", [(1, 1, 1, 1), (3, 2, 5, 64), (257, 7, 4, 4), (1000, 2, 33, 64), (4096, 3, 3, 8),
                                                 (4097, 1, 1, 1), (50001, 2, 4, 64), (8193, 70, 8, 5), (16385, 40, 8, 64)])
def test_selection(dtype, V, groups, beams, keep):
    rng = np.random.default_rng(V)
    rows = groups * beams
    Guarded(Select(logits(rng, rows, V, dtype), rng.normal(-20, 2, rows), beams, keep, dtype)).run()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("groups,alone,hq,hk,D,P", [([(40, [1, 2])], [], 2, 1, 8, 16), ([(200, [3] * 5)], [7], 6, 2, 64, 16),
                                                    ([(9000, [1] * 40)], [], 8, 2, 64, 16), ([(300, [20] * 70)], [1], 8, 1, 256, 16),
                                                    ([(100, [4] * 300)], [], 16, 2, 96, 16), ([(9, [1] * 8)] * 255, [5], 2, 2, 32, 4),
                                                    ([(16, [1] * 2047)], [], 33, 1, 16, 16), ([(600, [2, 3])] * 60, [], 17, 1, 128, 24)])
def test_shared_attention(dtype, groups, alone, hq, hk, D, P):
    Guarded(Shared(len(groups) + D, dtype, hq, hk, D, P, groups, alone=alone).upload()).run()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lengths,hq,hk,D", [([20000], 6, 2, 64), ([9000, 3], 8, 8, 128), ([3000, 4000, 1], 2, 1, 32),
                                             ([5000] * 5, 17, 1, 256), ([6000], 33, 1, 64)])
def test_attention(dtype, lengths, hq, hk, D):
    Guarded(Attend(D, dtype, hq, hk, D, 16, lengths).upload()).run()
