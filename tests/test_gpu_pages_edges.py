"""The pages' calls at the largest sizes that they take."""
import ctypes

import numpy as np
import pytest

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
