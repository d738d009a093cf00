"""Refusals of the paged-cache, rotary and token-score calls: host code, no
device is touched."""
import ctypes

import numpy as np
import pytest

from sejong_amd import _native as N

X = ctypes.c_void_p(0x1000)  # never read: every call below is refused before a launch
INT_MAX = 2 ** 31 - 1


def refused(name, args, status=1, word=b""):
    lib = N.load()
    got = getattr(lib, name)(*args)
    assert got == status and word in lib.sj_last_error(), (name, got, lib.sj_last_error())


def changed(base, **kw):
    names, values = zip(*base.items())
    assert set(kw) <= set(names)
    return [kw.get(n, v) for n, v in base.items()]


PLAN = dict(stream=None, lengths=X, counts=X, requests=4, page_size=16, pages=8, table=X, ldt=4, free_pages=X,
            free_count=8, free_head=None, lengths_after=None, starts=X, positions=X, slots=X, owners=X, capacity=8,
            summary=ctypes.c_void_p(0x2000))


@pytest.mark.parametrize("kw", [dict(requests=-1), dict(page_size=0), dict(page_size=-16), dict(pages=0), dict(ldt=0),
                                dict(pages=INT_MAX), dict(ldt=INT_MAX // 16 + 1), dict(capacity=-1), dict(lengths=None),
                                dict(counts=None), dict(table=None), dict(free_pages=None), dict(starts=None),
                                dict(summary=None), dict(slots=None), dict(owners=None), dict(positions=None),
                                dict(lengths_after=X), dict(free_head=ctypes.c_void_p(0x2004)), dict(free_count=-1),
                                dict(capacity=INT_MAX + 1), dict(requests=2 ** 24 + 1)])
def test_plan_refusals(kw):
    refused("sj_paged_plan", changed(PLAN, **kw), 1, b"paged plan")


ROPE = dict(stream=None, x=X, ldx=128, y=X, ldy=128, dtype=N.SJ_BF16, rows=4, heads=2, head_dim=64, rotary_dim=64,
            layout=0, positions=X, turns=X, amplitude=1.0, inverse=0)


@pytest.mark.parametrize("kw", [dict(dtype=N.SJ_F16), dict(dtype=N.SJ_F64), dict(head_dim=63), dict(rotary_dim=66),
                                dict(rotary_dim=7), dict(rotary_dim=-2), dict(layout=2), dict(layout=-1), dict(rows=-1),
                                dict(heads=0), dict(rows=2 ** 24 + 1),
                                dict(heads=2 ** 14 + 1, ldx=2 ** 21, ldy=2 ** 21), dict(ldx=127), dict(ldy=127), dict(x=None), dict(y=None),
                                dict(positions=None), dict(turns=None), dict(head_dim=1026, ldx=4096, ldy=4096)])
def test_rope_refusals(kw):
    refused("sj_rope_rows", changed(ROPE, **kw), 1, b"rope rows")


def test_no_rows_is_no_work():
    lib = N.load()
    assert lib.sj_rope_rows(*changed(ROPE, rows=0, x=None, y=None)) == 0
    assert lib.sj_paged_append(*changed(APPEND, rows=0)) == 0
    assert lib.sj_paged_attention(*changed(ATTEND, rows=0)) == 0
    assert lib.sj_paged_attention(*changed(ATTEND, requests=0)) == 0
    assert lib.sj_token_logprobs(*changed(SCORE, rows=0)) == 0
    assert lib.sj_token_logprobs_bwd(*changed(BACK, rows=0)) == 0


@pytest.mark.parametrize("kw", [dict(theta=0.0), dict(theta=-1.0), dict(theta=float("nan")), dict(kind=4), dict(kind=-1),
                                dict(kind=1, factor=0.0), dict(kind=2, factor=float("inf")),
                                dict(kind=3, factor=2.0, context=0.0, fast=32.0, slow=1.0),
                                dict(kind=3, factor=2.0, context=100.0, fast=1.0, slow=1.0)])
def test_frequency_refusals(kw):
    s = N.RopeScaling(kw.get("theta", 1e4), kw.get("kind", 0), kw.get("factor", 1.0), kw.get("context", 0.0),
                      kw.get("fast", 0.0), kw.get("slow", 0.0))
    refused("sj_rope_frequencies", [None, X, 64, ctypes.byref(s)], 1, b"rope frequencies")


def test_frequency_argument_refusals():
    s = N.RopeScaling(1e4, 0, 1.0, 0.0, 0.0, 0.0)
    for args in ([None, None, 64, ctypes.byref(s)], [None, X, 0, ctypes.byref(s)], [None, X, 63, ctypes.byref(s)],
                 [None, X, 64, None], [None, X, 1026, ctypes.byref(s)]):
        refused("sj_rope_frequencies", args, 1, b"rope frequencies")


APPEND = dict(stream=None, q=X, ldq=256, k=X, ldk=128, v=X, ldv=128, dtype=N.SJ_BF16, rows=4, hq=4, hk=2, head_dim=64,
              rotary_dim=64, layout=1, positions=X, slots=X, turns=X, amplitude=1.0, q_out=X, ldqo=256, k_cache=X,
              v_cache=X, ldkv=128, cache_slots=32)


@pytest.mark.parametrize("kw", [dict(dtype=N.SJ_I32), dict(head_dim=65), dict(rotary_dim=128), dict(layout=3),
                                dict(rows=-1), dict(hk=0), dict(hq=-1), dict(ldq=255), dict(ldqo=255), dict(ldk=127),
                                dict(ldv=127), dict(ldkv=127), dict(cache_slots=-1), dict(k=None), dict(v=None),
                                dict(q=None), dict(q_out=None), dict(positions=None), dict(slots=None), dict(turns=None),
                                dict(k_cache=None), dict(v_cache=None)])
def test_append_refusals(kw):
    refused("sj_paged_append", changed(APPEND, **kw), 1, b"paged append")


ATTEND = dict(stream=None, q=X, ldq=256, k_cache=X, v_cache=X, ldkv=128, dtype=N.SJ_BF16, pages=8, page_size=16, table=X,
              ldt=4, requests=4, owners=X, positions=X, rows=4, hq=4, hk=2, head_dim=64, window=0, o=X, ldo=256,
              lse=None, workspace=None, workspace_bytes=0)


@pytest.mark.parametrize("kw", [dict(dtype=N.SJ_F16), dict(rows=-1), dict(requests=-1), dict(hq=3), dict(hk=0),
                                dict(hq=0), dict(head_dim=0), dict(head_dim=257, ldq=2048, ldo=2048, ldkv=2048),
                                dict(window=-1), dict(ldq=255), dict(ldo=255), dict(ldkv=127), dict(page_size=0),
                                dict(pages=0), dict(pages=INT_MAX), dict(ldt=0), dict(ldt=INT_MAX), dict(q=None),
                                dict(k_cache=None), dict(v_cache=None), dict(table=None), dict(positions=None),
                                dict(o=None), dict(owners=None, rows=5), dict(rows=2 ** 22 + 1)])
def test_attention_refusals(kw):
    refused("sj_paged_attention", changed(ATTEND, **kw), 1, b"paged attention")


SCORE = dict(stream=None, x=X, dtype=N.SJ_F32, ldx=264, rows=4, vocab=257, tokens=X, top=5, logprob=X, entropy=X,
             stats=X, top_ids=X, top_logprob=X, workspace=None, workspace_bytes=0)


@pytest.mark.parametrize("kw", [dict(dtype=N.SJ_F16), dict(rows=-1), dict(vocab=0), dict(ldx=256), dict(top=-1),
                                dict(top=65), dict(vocab=3, top=4), dict(x=None), dict(rows=2 ** 24 + 1),
                                dict(vocab=2 ** 24 + 1, ldx=2 ** 25), dict(vocab=100000, ldx=100000, rows=2 ** 21), dict(tokens=None), dict(top_ids=None),
                                dict(top_logprob=None)])
def test_score_refusals(kw):
    refused("sj_token_logprobs", changed(SCORE, **kw), 1, b"token log probabilities")


BACK = dict(stream=None, x=X, dtype=N.SJ_F32, ldx=264, rows=4, vocab=257, tokens=X, stats=X, entropy=X, dlogprob=X,
            dentropy=X, dx=X, dx_dtype=N.SJ_F32, lddx=264)


@pytest.mark.parametrize("kw", [dict(dtype=N.SJ_F64), dict(dx_dtype=N.SJ_I32), dict(rows=-1), dict(vocab=0),
                                dict(ldx=256), dict(lddx=256), dict(x=None), dict(stats=None), dict(dx=None),
                                dict(tokens=None), dict(entropy=None)])
def test_score_backward_refusals(kw):
    refused("sj_token_logprobs_bwd", changed(BACK, **kw), 1, b"token log probabilities backward")


def test_short_workspaces_are_refused():
    """A call that needs scratch says how much, and takes no less."""
    lib = N.load()
    need = lib.sj_paged_attention_workspace_bytes(4, 4, 2, 64)
    if need:
        refused("sj_paged_attention", changed(ATTEND, workspace=X, workspace_bytes=need - 1), 2, b"required %d bytes" % need)
        refused("sj_paged_attention", changed(ATTEND, workspace=None, workspace_bytes=need), 2, b"available 0 bytes")
        odd = ctypes.c_void_p(0x1008)
        refused("sj_paged_attention", changed(ATTEND, workspace=odd, workspace_bytes=need), 1, b"16-byte aligned")
    need = lib.sj_token_logprobs_workspace_bytes(4, 150000, 5)
    if need:
        big = dict(vocab=150000, ldx=150000)
        refused("sj_token_logprobs", changed(SCORE, workspace=X, workspace_bytes=need - 1, **big), 2,
                b"required %d bytes" % need)
        refused("sj_token_logprobs", changed(SCORE, workspace=ctypes.c_void_p(0x1004), workspace_bytes=need, **big), 1,
                b"16-byte aligned")


def test_the_gradient_formula_against_differences():
    """dx of sum dlp logprob + dent entropy, against central differences in 64 bits (their own error h^2 and eps / h)."""
    from tests import score_util as U
    rng = np.random.default_rng(3)
    x, tokens = rng.normal(0, 2, (4, 9)), np.array([0, 8, -1, 3])
    dlp, dent = rng.normal(size=4), rng.normal(size=4)
    got = U.gradient(x, tokens, dlp, dent)
    h = 1e-5
    for r in range(4):
        for v in range(9):
            e = np.zeros_like(x)
            e[r, v] = h
            f = [dlp @ s["logprob"] + dent @ s["entropy"] for s in (U.scores(x + e, tokens), U.scores(x - e, tokens))]
            assert abs((f[0] - f[1]) / (2 * h) - got[r, v]) < 1e-8


def test_limits_are_the_documented_ones():
    """Rows times tiles of 16 query heads up to 2^23; rows times slices of 8192 entries below 2^23 (the refusal that
    follows is the missing workspace's)."""
    wide = dict(hq=40, hk=2, ldq=40 * 64, ldo=40 * 64, requests=2 ** 23, workspace=X, workspace_bytes=2 ** 40)
    refused("sj_paged_attention", changed(ATTEND, rows=2 ** 21 + 1, **wide), 1, b"rows of 2 heads")
    refused("sj_paged_attention", changed(ATTEND, hq=65536, hk=65536, ldq=2 ** 22, ldo=2 ** 22, ldkv=2 ** 22), 1,
            b"paged attention")
    for slices in (3, 5, 7):
        most = (2 ** 23 - 1) // slices
        at = dict(vocab=slices * 8192, ldx=slices * 8192)
        refused("sj_token_logprobs", changed(SCORE, rows=most, **at), 2, b"required")
        refused("sj_token_logprobs", changed(SCORE, rows=most + 1, **at), 1, b"rows of")
        refused("sj_token_logprobs_bwd", changed(BACK, rows=most + 1, lddx=slices * 8192, **at), 1, b"rows of")


def test_in_place_calls_keep_their_rows_places():
    """The output may be the input only where each element stays in its own place: other strides or types would have
    rows overwritten before they are read."""
    refused("sj_rope_rows", changed(ROPE, ldx=128, ldy=136), 1, b"in place")
    refused("sj_rope_rows", changed(ROPE, ldx=256, ldy=128), 1, b"in place")
    refused("sj_paged_append", changed(APPEND, ldq=512, ldqo=256), 1, b"in place")
    refused("sj_paged_attention", changed(ATTEND, ldq=512, ldo=256), 1, b"in place")
    for kw in (dict(ldx=264, lddx=265), dict(dx_dtype=N.SJ_BF16), dict(dtype=N.SJ_BF16)):
        refused("sj_token_logprobs_bwd", changed(BACK, **kw), 1, b"in place")


def test_cut_walks_and_long_rows_need_a_workspace():
    lib = N.load()
    need = lib.sj_paged_attention_workspace_bytes(4, 4, 2, 64)
    assert need > 0
    refused("sj_paged_attention", changed(ATTEND, workspace=X, workspace_bytes=need - 1), 2, b"required %d bytes" % need)
    refused("sj_paged_attention", changed(ATTEND, workspace=None, workspace_bytes=need), 2, b"available 0 bytes")
    need = lib.sj_token_logprobs_workspace_bytes(4, 150000, 5)
    assert need > 0
    big = dict(vocab=150000, ldx=150000)
    refused("sj_token_logprobs", changed(SCORE, workspace=X, workspace_bytes=need - 1, **big), 2, b"required %d bytes" % need)
    refused("sj_token_logprobs", changed(SCORE, workspace=None, workspace_bytes=need, **big), 2, b"available 0 bytes")
