"""The sizes that the beam selection takes by its documentation: rows times vocab /
8192, rounded up, below 2^23.  Host code: a call that passes the checks of its sizes
asks for its workspace."""
import pytest

from sejong_amd import _native as N
from tests.test_beam_host import SELECT
from tests.test_paged_host import changed, refused


@pytest.mark.parametrize("rows,vocab", [(2 ** 23 - 1, 1), (2 ** 23 - 1, 4096), (2 ** 23 - 1, 4097), (2 ** 22, 4097),
                                        (2 ** 23 - 1, 8192), (2 ** 22 - 1, 8193), (2 ** 22 - 1, 16384), (2 ** 12 - 1, 2 ** 24)])
def test_sizes_that_are_taken(rows, vocab):
    need = N.load().sj_beam_select_workspace_bytes(rows, 1, vocab, 4)
    kw = dict(groups=rows, beams=1, vocab=vocab, ldx=vocab, keep=4, end_token=0)
    refused("sj_beam_select", changed(SELECT, workspace=None, **kw), 2, b"required %d bytes" % need)


@pytest.mark.parametrize("rows,vocab", [(2 ** 23, 1), (2 ** 23, 8192), (2 ** 22, 8193), (2 ** 12, 2 ** 24)])
def test_sizes_that_are_refused(rows, vocab):
    refused("sj_beam_select", changed(SELECT, groups=rows, beams=1, vocab=vocab, ldx=vocab, end_token=0), 1, b"beam selection")
