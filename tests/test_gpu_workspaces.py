"""Calls write nothing behind the bytes that their workspace query names."""
import numpy as np
import pytest

from tests import gpu_util as G
from tests.test_gpu_pages import Compact

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
