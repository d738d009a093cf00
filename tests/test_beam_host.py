"""Refusals of the beam selection, of the pages' fork, compaction and copy, and
of attention over shared prefixes: host code, no device is touched.  The plain
forms that the GPU tests compare with, against each other."""
import ctypes

import numpy as np
import pytest

from sejong_amd import _native as N
from tests import beam_util as BU
from tests.test_paged_host import ATTEND, INT_MAX, X, changed, refused

Y, Z = ctypes.c_void_p(0x2000), ctypes.c_void_p(0x3000)
BIG = 2 ** 40

SELECT = dict(stream=None, x=X, dtype=N.SJ_F32, ldx=264, groups=2, beams=4, vocab=257, scores=X, lengths=X, ended=X,
              end_token=1, length_power=0.6, keep=8, parents=Y, tokens=Y, scores_after=Y, lengths_after=Y, ended_after=Y,
              workspace=X, workspace_bytes=BIG)


@pytest.mark.parametrize("kw", [dict(dtype=N.SJ_F16), dict(groups=-1), dict(beams=0), dict(beams=65), dict(keep=0),
                                dict(keep=65), dict(vocab=0), dict(ldx=256), dict(vocab=2 ** 24 + 1, ldx=2 ** 25),
                                dict(groups=2 ** 21, beams=4, vocab=257), dict(groups=2 ** 18, vocab=70000, ldx=70000),
                                dict(end_token=-2), dict(end_token=257), dict(length_power=-0.5), dict(length_power=17.0),
                                dict(length_power=float("nan")), dict(x=None), dict(scores=None), dict(parents=None),
                                dict(tokens=None), dict(scores_after=None), dict(lengths=None),
                                dict(lengths=None, length_power=0.0), dict(scores_after=X), dict(lengths_after=X),
                                dict(ended_after=X), dict(workspace=ctypes.c_void_p(0x1008))])
def test_select_refusals(kw):
    refused("sj_beam_select", changed(SELECT, **kw), 1, b"beam selection")


def test_select_workspace():
    lib = N.load()
    for groups, beams, vocab, keep in ((2, 4, 257, 8), (1, 8, 131072, 16), (3, 1, 5, 64)):
        need = lib.sj_beam_select_workspace_bytes(groups, beams, vocab, keep)
        at = dict(groups=groups, beams=beams, vocab=vocab, ldx=vocab, keep=keep)
        assert need > 0
        refused("sj_beam_select", changed(SELECT, workspace_bytes=need - 1, **at), 2, b"required %d bytes" % need)
        refused("sj_beam_select", changed(SELECT, workspace=None, **at), 2, b"available 0 bytes")


FORK = dict(stream=None, parents=X, requests=4, table=X, ldt=4, lengths=X, requests_before=4, page_size=16, pages=8,
            shared=X, free_pages=X, free_count=8, free_head=X, table_after=Y, lengths_after=Y, shared_after=Y,
            free_after=Y, copies=Y, summary=Y, workspace=X, workspace_bytes=BIG)


@pytest.mark.parametrize("kw", [dict(requests=-1), dict(requests=16385), dict(requests_before=16385),
                                dict(requests_before=-1), dict(free_count=-1), dict(free_count=INT_MAX + 1),
                                dict(page_size=0), dict(pages=0), dict(ldt=0), dict(pages=INT_MAX), dict(ldt=INT_MAX),
                                dict(parents=None), dict(table=None), dict(lengths=None), dict(shared=None),
                                dict(free_pages=None), dict(table_after=None), dict(lengths_after=None),
                                dict(shared_after=None), dict(free_after=None), dict(copies=None), dict(summary=None),
                                dict(table_after=X), dict(lengths_after=X), dict(shared_after=X), dict(free_after=X),
                                dict(free_head=ctypes.c_void_p(0x2004)), dict(workspace=ctypes.c_void_p(0x1004))])
def test_fork_refusals(kw):
    refused("sj_paged_fork", changed(FORK, **kw), 1, b"paged fork")


COMPACT = dict(stream=None, table=X, ldt=4, lengths=X, requests=4, page_size=16, pages=8, pages_after=4, shared=X,
               free_pages=X, free_count=8, free_head=X, table_after=Y, shared_after=Y, free_after=Y, copies=Y, capacity=4,
               summary=Y, workspace=X, workspace_bytes=BIG)


@pytest.mark.parametrize("kw", [dict(requests=-1), dict(requests=2 ** 24 + 1), dict(free_count=-1), dict(capacity=-1),
                                dict(page_size=0), dict(pages=0), dict(ldt=0), dict(pages=INT_MAX), dict(ldt=INT_MAX),
                                dict(pages_after=-1), dict(pages_after=9), dict(table=None), dict(lengths=None),
                                dict(shared=None), dict(free_pages=None), dict(table_after=None), dict(shared_after=None),
                                dict(free_after=None), dict(copies=None), dict(summary=None), dict(table_after=X),
                                dict(shared_after=X), dict(free_after=X), dict(free_head=ctypes.c_void_p(0x2004)),
                                dict(workspace=ctypes.c_void_p(0x1004))])
def test_compact_refusals(kw):
    refused("sj_paged_compact", changed(COMPACT, **kw), 1, b"paged compact")


COPY = dict(stream=None, k_cache=X, v_cache=X, ldkv=128, dtype=N.SJ_BF16, layers=2, layer_stride=4096, pages=8,
            page_size=16, width=128, copies=X, count=4)


@pytest.mark.parametrize("kw", [dict(dtype=N.SJ_F64), dict(layers=-1), dict(layers=65537), dict(count=-1),
                                dict(count=2 ** 24 + 1), dict(count=2 ** 20, layers=1024), dict(width=0), dict(width=129),
                                dict(ldkv=INT_MAX + 1), dict(layer_stride=-1), dict(page_size=0), dict(pages=0),
                                dict(pages=INT_MAX), dict(k_cache=None), dict(v_cache=None), dict(copies=None)])
def test_copy_refusals(kw):
    refused("sj_paged_copy", changed(COPY, **kw), 1, b"paged copy")


def test_pages_workspaces():
    lib = N.load()
    need = lib.sj_paged_fork_workspace_bytes(4, 4, 8)
    assert need > 0
    refused("sj_paged_fork", changed(FORK, workspace_bytes=need - 1), 2, b"required %d bytes" % need)
    refused("sj_paged_fork", changed(FORK, workspace=None), 2, b"available 0 bytes")
    need = lib.sj_paged_compact_workspace_bytes(8, 8)
    assert need > 0
    refused("sj_paged_compact", changed(COMPACT, workspace_bytes=need - 1), 2, b"required %d bytes" % need)
    refused("sj_paged_compact", changed(COMPACT, workspace=None), 2, b"available 0 bytes")


SHARED = {}
for _n, _v in ATTEND.items():
    SHARED[_n] = _v
    if _n == "rows":
        SHARED.update(starts=X, group_starts=X, prefix=X, groups=2)
SHARED.update(workspace=X, workspace_bytes=BIG)


@pytest.mark.parametrize("kw", [dict(dtype=N.SJ_F16), dict(rows=-1), dict(requests=-1), dict(hq=3), dict(hk=0), dict(hq=0),
                                dict(head_dim=0), dict(head_dim=257, ldq=2048, ldo=2048, ldkv=2048), dict(window=-1),
                                dict(ldq=255), dict(ldo=255), dict(ldkv=127), dict(page_size=0), dict(pages=0),
                                dict(pages=INT_MAX), dict(ldt=0), dict(ldt=INT_MAX), dict(q=None), dict(k_cache=None),
                                dict(v_cache=None), dict(table=None), dict(positions=None), dict(o=None),
                                dict(owners=None, rows=5), dict(groups=-1), dict(groups=2 ** 24 + 1),
                                dict(group_starts=None), dict(prefix=None), dict(ldq=512, o=X),
                                dict(workspace=ctypes.c_void_p(0x1008))])
def test_shared_refusals(kw):
    refused("sj_paged_attention_shared", changed(SHARED, **kw), 1, b"paged attention")


def test_shared_workspace():
    lib = N.load()
    need = lib.sj_paged_attention_shared_workspace_bytes(4, 4, 2, 64, 2)
    assert need >= lib.sj_paged_attention_workspace_bytes(4, 4, 2, 64) > 0
    refused("sj_paged_attention_shared", changed(SHARED, workspace_bytes=need - 1), 2, b"required %d bytes" % need)
    refused("sj_paged_attention_shared", changed(SHARED, workspace=None), 2, b"available 0 bytes")


def test_no_rows_is_no_work():
    lib = N.load()
    assert lib.sj_beam_select(*changed(SELECT, groups=0)) == 0
    assert lib.sj_paged_copy(*changed(COPY, count=0)) == 0 and lib.sj_paged_copy(*changed(COPY, layers=0)) == 0
    assert lib.sj_paged_attention_shared(*changed(SHARED, rows=0)) == 0
    assert lib.sj_paged_attention_shared(*changed(SHARED, requests=0)) == 0


def test_plain_forks_keep_every_page():
    """A long random life of forks: no page is lost, held twice, or on the list while a row has it."""
    rng = np.random.default_rng(5)
    P, pages, R, W = 4, 60, 6, 8
    free, head, shared = rng.permutation(pages), 0, np.zeros(pages, int)
    table, lengths = np.full((R, W), -1), np.zeros(R, int)
    for step in range(200):
        for r in range(R):  # a token more, sometimes a page
            if lengths[r] < W * P - 1:
                if lengths[r] % P == 0:
                    table[r, lengths[r] // P], head = free[head], head + 1
                lengths[r] += 1
        parents = rng.integers(-1 if step % 10 == 0 else 0, R, R)
        f = BU.fork(parents, table, lengths, P, pages, shared, free, head)
        assert f["status"] == 0
        table, lengths, shared, free, head = f["table"], f["lengths"], f["shared"], f["free"], f["head"]
        rows = [table[r, :-(-lengths[r] // P)] for r in range(R)]
        held = np.bincount(np.concatenate(rows).astype(int), minlength=pages)
        np.testing.assert_array_equal(np.maximum(held - 1, 0), shared)
        assert sorted(free[head:]) == [p for p in range(pages) if held[p] == 0]
        tails = [row[-1] for row, n in zip(rows, lengths) if n % P]
        assert len(set(tails)) == len(tails) and all(held[p] == 1 for p in tails)
