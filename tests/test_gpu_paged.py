"""The paged cache's calls: the step's plan, rotary positions and the append,
attention over the pages, and a run of them together."""
import ctypes
import math

import numpy as np
import pytest

from tests import gpu_util as G
from tests import paged_util as PU
from tests import score_util as SU

pytestmark = pytest.mark.gpu
CODE = {"f32": 0, "bf16": 4}
HALF_ULP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}


def native():
    from sejong_amd import _native as N
    return N, N.load()


# ------------------------------------------------------------------- plan

class Plan:
    def __init__(self, lengths, counts, P, pages, width, table, free, head, capacity):
        self.R, self.P, self.pages, self.width, self.cap = len(lengths), P, pages, width, capacity
        self.args = (np.asarray(lengths, np.int32), np.asarray(counts, np.int32), P, pages, np.asarray(table, np.int32),
                     np.asarray(free, np.int32), head, capacity)
        self.n, self.m = PU.ints(list(lengths) + [0]), PU.ints(list(counts) + [0])
        self.table, self.free = PU.ints(np.append(table, 7)), PU.ints(list(free) + [0])
        self.nfree, self.head = len(free), PU.ints([head])
        self.after, self.starts = PU.ints(np.full(self.R + 1, 5)), PU.ints(np.full(self.R + 2, 5))
        self.rows = [PU.ints(np.full(capacity + 1, 5)) for _ in range(3)]
        self.summary = PU.ints([5] * 5)

    def run(self, stream=None):
        native()[0].api.sj_paged_plan(stream, self.n.p, self.m.p, self.R, self.P, self.pages, self.table.p, self.width,
                                      self.free.p, self.nfree, self.head.p, self.after.p, self.starts.p, self.rows[0].p,
                                      self.rows[1].p, self.rows[2].p, self.cap, self.summary.p)

    def check(self):
        lengths, counts, P, pages, table, free, head, cap = self.args
        want = PU.plan(lengths, counts, P, pages, table.reshape(self.R, self.width), free, head, cap)
        s = self.summary.host()
        assert s[4] == 5 and s[2] == want["status"] and s[1] == want["head"] and s[0] == want["starts"][-1]
        if not s[2]:
            assert s[3] == (int((lengths.astype(np.int64) + counts).max()) if self.R else 0)
        for got, w in ((self.starts, want["starts"]), (self.after, want["after"]), (self.table, want["table"].ravel()),
                       *zip(self.rows, want["rows"])):
            h = got.host()
            np.testing.assert_array_equal(h[:len(w)], w)
            assert h[-1] == (7 if got is self.table else 5)  # nothing behind the rows
        return want


def pool(rng, lengths, counts, P, extra=8, width=None):
    """Tables of requests that hold `lengths` tokens, and the free pages, in a random order."""
    lengths, counts = np.asarray(lengths, np.int64), np.asarray(counts, np.int64)
    have, want = -(-lengths // P), -(-(lengths + counts) // P)
    width = width or max(int(want.max()) if len(want) else 0, 1)
    pages = max(int(want.sum()) + extra, 1)
    order = rng.permutation(pages)
    table = np.full((len(lengths), width), -1)
    table[np.arange(width)[None, :] < have[:, None]] = order[:have.sum()]
    return pages, width, table, order[have.sum():]


@pytest.mark.parametrize("R,P,hi,new,pad", [(0, 16, 1, 1, 3), (1, 1, 5, 3, 0), (1, 16, 40, 5000, 7), (5, 16, 100, 1, 0),
                                            (64, 16, 4000, 1, 5), (300, 24, 500, 40, 1000), (1024, 7, 90, 9, 1),
                                            (1500, 100, 3000, 60, 0), (5000, 16, 50, 3, 100), (3, 1000, 5000, 4000, 0)])
def test_plan(R, P, hi, new, pad):
    rng = np.random.default_rng(R + P)
    lengths, counts = rng.integers(0, hi + 1, R), rng.integers(0, new + 1, R)
    if R > 3:
        lengths[:3] = [0, P, 2 * P]  # empty and full pages
        counts[1] = 0
    pages, width, table, free = pool(rng, lengths, counts, P)
    p = Plan(lengths, counts, P, pages, width + 2, np.pad(table, ((0, 0), (0, 2)), constant_values=-1), free, 0,
             int(counts.sum()) + pad)
    p.run()
    p.check()
    p.run()  # the same inputs again: the same step
    p.check()


def test_plan_from_the_middle_of_the_free_list_and_bad_pages():
    rng = np.random.default_rng(1)
    lengths, counts = np.array([17, 3, 0, 31]), np.array([20, 1, 9, 1])
    pages, width, table, free = pool(rng, lengths, counts, 8)
    table[0, 2] = pages  # the page that holds the last tokens of request 0 is none
    free = np.concatenate([[-1, -1], free])
    free[3] = -5
    p = Plan(lengths, counts, 8, pages, width, table, free, 2, 40)
    p.run()
    want = p.check()
    assert (want["rows"][1][:31] == -1).sum() > 5


@pytest.mark.parametrize("status,change", [
    (1, dict(free=2)), (1, dict(head=-1)), (1, dict(head=100)), (2, dict(width=2)), (4, dict(cap=10)), (8, dict(bad=(1, -3, 0))),
    (8, dict(bad=(0, 5, -1))), (13, dict(free=1, cap=3, bad=(2, -1, 2)))])
def test_void_plans(status, change):
    """A step that cannot be leaves tables, lengths and the free list as they are, and every row empty."""
    rng = np.random.default_rng(2)
    lengths, counts = np.array([17, 30, 4, 0]), np.array([20, 1, 9, 11])
    pages, width, table, free = pool(rng, lengths, counts, 8)
    if "width" in change:
        table, width = table[:, :change["width"]], change["width"]
    if "bad" in change:
        r, n, m = change["bad"]
        lengths[r], counts[r] = n, m
    p = Plan(lengths, counts, 8, pages, width, table, free[:change.get("free", len(free))], change.get("head", 0),
             change.get("cap", 60))
    p.run()
    assert p.check()["status"] == status


def test_plan_lengths_past_31_bits_are_void():
    p = Plan([2 ** 31 - 5, 3], [10, 1], 2 ** 20, 2047, 2047, np.full((2, 2047), -1), np.arange(20), 0, 40)
    p.run()
    assert p.summary.host()[2] & 8 and (p.rows[0].host()[:40] == -1).all()


# ----------------------------------------------------------------- rotary

SCALINGS = [dict(), dict(kind=1, factor=4.0), dict(kind=2, factor=8.0, theta=5000.0),
            dict(kind=3, factor=8.0, context=4096.0, fast=32.0, slow=1.0)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("rows,heads,D,rot,scaling,inverse,amp,inplace", [
    (1, 1, 2, 2, 0, 0, 1.0, False), (7, 3, 16, 16, 1, 0, 1.0, True), (65, 6, 64, 64, 3, 0, 1.2, False),
    (33, 2, 96, 40, 2, 1, 1.0, False), (300, 5, 80, 20, 3, 1, 0.7, True), (5, 40, 128, 128, 0, 1, 1.0, False),
    (3, 2, 256, 256, 2, 0, 1.0, True), (4, 2, 1024, 1024, 0, 0, 1.0, False), (9, 2, 30, 6, 1, 0, 1.0, False),
    (6, 3, 64, 0, 0, 0, 1.0, False), (2000, 4, 64, 32, 3, 0, 1.0, False)])
def test_rope_rows(dtype, layout, rows, heads, D, rot, scaling, inverse, amp, inplace):
    """An angle's cosine and sine are off by 2^-22 at any position, two products and a sum by 2^-23 of |a| + |b|."""
    N, lib = native()
    rng = np.random.default_rng(rows + D)
    ldx, off = heads * D + (3 if rows % 2 else 8), rows % 3
    x = G.rnd((rows, ldx), dtype, rng)
    pos = rng.integers(0, 1 << 20, rows)
    pos[0] = 0
    if rows > 2:
        pos[1], pos[2] = 2 ** 31 - 1, -7
    X = G.dev(np.concatenate([np.zeros(off), x.ravel()]), dtype)
    ldy = ldx if inplace else heads * D + 1
    Y = X if inplace else G.dev(np.full(off + rows * ldy, 55.0), dtype)
    sc = SCALINGS[scaling]
    T = PU.turns(rot, **sc) if rot else None
    Z = PU.ints(pos)
    N.api.sj_rope_rows(None, X.at(off), ldx, Y.at(off), ldy, CODE[dtype], rows, heads, D, rot, layout, Z.p, T and T.p,
                       ctypes.c_float(amp), inverse)
    got = Y.host()[off:].reshape(rows, ldy)
    amp = float(np.float32(amp))
    want = PU.rotate(x[:, :heads * D], heads, D, rot, layout, pos, PU.frequencies(rot, **sc), amp, bool(inverse))
    mag = np.abs(x[:, :heads * D]).reshape(rows, heads, D).max(2, keepdims=True).repeat(D, 2).reshape(rows, -1)
    # a frequency formed in double is off by some 2^-50 of itself, on both sides, and its angle by that times the position
    far = np.abs(pos.astype(np.float64))[:, None] * 2.0 ** -49
    tol = 2 * amp * mag * (2.0 ** -21 + far) + np.abs(want) * HALF_ULP[dtype] * 1.01
    assert (np.abs(got[:, :heads * D] - want) <= tol).all(), np.max(np.abs(got[:, :heads * D] - want) / tol)
    rest = got[:, heads * D:]
    np.testing.assert_array_equal(rest, x[:, heads * D:] if inplace else np.full_like(rest, 55.0))
    if rot < D:  # columns past the rotary width are copied
        cols = np.arange(heads * D).reshape(heads, D)[:, rot:].ravel()
        np.testing.assert_array_equal(got[:, cols], x[:, cols])


def test_rope_rows_agrees_with_the_whole_head_rope():
    """Interleaved, unscaled, counting positions: sj_rope's rotation."""
    N, lib = native()
    rng = np.random.default_rng(5)
    rows, heads, D = 40, 3, 64
    x = G.rnd((rows, heads * D), "f32", rng)
    X, A, B, T = G.dev(x), G.empty(x.size), G.empty(x.size), PU.turns(D)
    N.api.sj_rope(None, X.p, A.p, 0, rows, heads * D, rows, heads, D, 9, ctypes.c_float(1e4), 0)
    Z = PU.ints(9 + np.arange(rows))
    N.api.sj_rope_rows(None, X.p, heads * D, B.p, heads * D, 0, rows, heads, D, D, 0, Z.p, T.p,
                       ctypes.c_float(1.0), 0)
    np.testing.assert_allclose(B.host(), A.host(), rtol=0, atol=2.0 ** -20 * 5)


def test_rope_gradient_is_the_adjoint():
    """<dy, R x> = <R' dy, x> for the inverse call, row by row, and the forward's differences along a direction."""
    N, lib = native()
    rng = np.random.default_rng(6)
    rows, heads, D, rot = 20, 4, 96, 48
    x, d, dy = (rng.normal(size=(rows, heads * D)).astype(np.float32) for _ in range(3))
    T, Z = PU.turns(rot, **SCALINGS[3]), PU.ints(rng.integers(0, 100000, rows))

    def call(v, inverse, layout):
        X, Y = G.dev(v), G.empty(v.size)
        N.api.sj_rope_rows(None, X.p, heads * D, Y.p, heads * D, 0, rows, heads, D, rot, layout, Z.p, T.p,
                           ctypes.c_float(1.3), inverse)
        return Y.host().reshape(v.shape)
    for layout in (0, 1):
        y, dx = call(x, 0, layout), call(dy, 1, layout)
        bound = (np.abs(dy) * 1.3).sum(1) * 5 * 2.0 ** -20
        assert (np.abs((dy * y).sum(1) - (dx * x).sum(1)) <= bound).all()
        step = (call(x + d, 0, layout) - call(x - d, 0, layout)) / 2
        assert (np.abs((dy * step).sum(1) - (dx * d).sum(1)) <= 3 * bound).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,hq,hk,D,rot,layout", [(1, 6, 2, 64, 64, 0), (37, 4, 4, 96, 32, 1), (600, 3, 1, 20, 10, 0),
                                                     (9, 0, 2, 64, 64, 1), (130, 8, 2, 128, 128, 1)])
def test_append(dtype, rows, hq, hk, D, rot, layout):
    N, lib = native()
    rng = np.random.default_rng(rows)
    ld = (hq + 2 * hk) * D + 2
    x = G.rnd((rows, ld), dtype, rng)
    total, ldkv = 2 * rows + 5, hk * D + 4
    slots = rng.permutation(total)[:rows]
    if rows > 4:
        slots[1], slots[3], slots[-1] = -1, total, 2 ** 31 - 1  # padded, and outside the cache
    pos = rng.integers(0, 5000, rows)
    X, K, V = G.dev(x, dtype), G.dev(np.full((total + 1) * ldkv, 7.0), dtype), G.dev(np.full((total + 1) * ldkv, 7.0), dtype)
    ldo = hq * D + 1
    Q = G.dev(np.full(rows * ldo, 7.0), dtype)
    T, Z, S = PU.turns(rot), PU.ints(pos), PU.ints(slots)
    N.api.sj_paged_append(None, X.p, ld, X.at(hq * D), ld, X.at((hq + hk) * D), ld, CODE[dtype], rows, hq, hk, D, rot,
                          layout, Z.p, S.p, T.p, ctypes.c_float(1.0), Q.p, ldo, K.p, V.p, ldkv, total)
    f = PU.frequencies(rot)
    q = PU.rotate(x[:, :hq * D], hq, D, rot, layout, pos, f) if hq else np.zeros((rows, 0))
    k = PU.rotate(x[:, hq * D:(hq + hk) * D], hk, D, rot, layout, pos, f)
    gq, gk, gv = Q.host().reshape(rows, ldo), K.host().reshape(-1, ldkv), V.host().reshape(-1, ldkv)
    live = (slots >= 0) & (slots < total)
    tol = np.abs(x).max() * 2.0 ** -20 + HALF_ULP[dtype] * 1.01 * np.abs(x).max() * 1.5
    assert np.abs(gq[live, :hq * D] - q[live]).max(initial=0) <= tol
    assert (gq[~live] == 7.0).all() and (gq[:, hq * D:] == 7.0).all()
    assert np.abs(gk[slots[live], :hk * D] - k[live]).max() <= tol
    np.testing.assert_array_equal(gv[slots[live], :hk * D], x[live, (hq + hk) * D:(hq + 2 * hk) * D])
    other = np.setdiff1d(np.arange(total + 1), slots[live])
    assert (gk[other] == 7.0).all() and (gv[other] == 7.0).all()
    assert (gk[:, hk * D:] == 7.0).all() and (gv[:, hk * D:] == 7.0).all()


# -------------------------------------------------------------- attention

class Attend:
    """Requests in a random pool whose unused slots hold NaN."""

    def __init__(self, seed, dtype, hq, hk, D, P, lengths, window=0, per=1, pad=0, owners=True, ldkv=0, off=0, q_scale=1.5):
        rng = self.rng = np.random.default_rng(seed)
        self.dtype, self.hq, self.hk, self.D, self.P, self.window = dtype, hq, hk, D, P, window
        lengths = np.asarray(lengths)
        self.pages, self.width, self.tab, _ = pool(rng, lengths, np.zeros_like(lengths), P)
        slots = self.pages * P
        self.k, self.v = (np.full((slots, hk, D), np.nan) for _ in range(2))
        for r, n in enumerate(lengths):
            j = np.arange(n)
            s = self.tab[r][j // P] * P + j % P
            self.k[s], self.v[s] = G.rnd((n, hk, D), dtype, rng), G.rnd((n, hk, D), dtype, rng)
        self.pos = np.concatenate([np.maximum(lengths - per + i, -1) for i in range(per)] + [np.full(pad, -1)])
        self.own = np.concatenate([np.arange(len(lengths)) for _ in range(per)] + [np.full(pad, -1)])
        self.q = G.rnd((len(self.pos), hq, D), dtype, rng, q_scale)
        self.use_owners, self.ldkv, self.off = owners, ldkv or hk * D, off

    def upload(self):
        N, lib = native()
        o, ld, n = self.off, self.ldkv, len(self.pos)
        wide = np.full((2, len(self.k), ld), 3e38)
        wide[0, :, :self.hk * self.D], wide[1, :, :self.hk * self.D] = (t.reshape(len(t), -1) for t in (self.k, self.v))
        with np.errstate(over="ignore"):
            self.K, self.V = (G.dev(np.concatenate([np.zeros(o), w.ravel()]), self.dtype) for w in wide)
        self.ldq = self.hq * self.D + (o and 5)
        q = np.zeros((n, self.ldq))
        q[:, :self.hq * self.D] = self.q.reshape(n, -1)
        self.Q = G.dev(np.concatenate([np.zeros(o), q.ravel()]), self.dtype)
        self.O, self.L = G.dev(np.full(o + n * self.ldq + 8, 55.0), self.dtype), G.dev(np.full(n * self.hq + 4, 55.0))
        self.T, self.Z, self.W = PU.ints(self.tab), PU.ints(self.pos), PU.ints(self.own)
        need = lib.sj_paged_attention_workspace_bytes(n, self.hq, self.hk, self.D)
        self.ws = G.Dev(max(need, 16), "u8").upload(np.full(max(need, 16), 0xFF))  # NaN: nothing is kept there
        self.need = need
        return self

    def run(self, stream=None, lse=True):
        native()[0].api.sj_paged_attention(stream, self.Q.at(self.off), self.ldq, self.K.at(self.off), self.V.at(self.off),
                                           self.ldkv, CODE[self.dtype], self.pages, self.P, self.T.p, self.width,
                                           len(self.tab), self.W.p if self.use_owners else None, self.Z.p, len(self.pos),
                                           self.hq, self.hk, self.D, self.window, self.O.at(self.off), self.ldq,
                                           self.L.p if lse else None, self.ws.p, self.need)
        return self

    def check(self, lse=True):
        n = len(self.pos)
        own = self.own if self.use_owners else np.arange(n)
        want = PU.attention(self.q, self.k, self.v, self.tab, self.P, self.pages, own, self.pos, self.hq, self.hk, self.D,
                            self.window)
        o, l = self.O.host()[self.off:], self.L.host()
        assert (o[n * self.ldq:] == 55.0).all() and (l[-4:] == 55.0).all()
        o, l = o[:n * self.ldq].reshape(n, self.ldq), l[:-4].reshape(n, self.hq)
        assert (o[:, self.hq * self.D:] == 55.0).all()
        for r, w in enumerate(want):
            g = o[r, :self.hq * self.D].reshape(self.hq, self.D)
            if w is None:
                assert (g == 55.0).all() and (l[r] == 55.0).all()
                continue
            ref, ls, mag, err = w
            # shares are off by the score's rounding, twice (numerator and sum), and by the 16 bits that two bf16
            # planes keep of them; the sums over the keys are counted in err; one rounding to the storage type
            tol = (2 * err[:, None] + (2.0 ** -15 if self.dtype == "bf16" else 2.0 ** -21)) * mag
            tol = tol + np.abs(ref) * HALF_ULP[self.dtype] * 1.01 + 1e-38
            assert (np.abs(g - ref) <= tol).all(), (r, np.nanmax(np.abs(g - ref) / tol), g[0, :4], ref[0, :4])
            if lse:
                fin = np.isfinite(ls)
                assert (l[r][~fin] == ls[~fin]).all()
                assert (np.abs(l[r][fin] - ls[fin]) <= err[fin] * 2 + 2.0 ** -21 * (1 + np.abs(ls[fin]))).all()
        return want


LENGTHS = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 200, 1000]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("hq,hk,D,P", [(6, 2, 64, 16), (4, 4, 64, 24), (16, 1, 64, 1), (40, 2, 64, 64), (3, 1, 16, 5),
                                       (8, 2, 32, 100), (8, 4, 80, 16), (14, 2, 96, 7), (8, 1, 128, 16), (32, 8, 128, 64),
                                       (5, 5, 256, 32), (18, 1, 256, 16), (2, 2, 8, 16), (3, 3, 7, 16), (4, 2, 20, 256)])
def test_attention(dtype, hq, hk, D, P):
    a = Attend(hq * D + P, dtype, hq, hk, D, P, LENGTHS, pad=2).upload().run()
    a.check()
    first = a.O.host().copy(), a.L.host().copy()
    a.run()
    assert all((x == y.host()).all() for x, y in zip(first, (a.O, a.L)))  # the same bits again


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window", [1, 2, 17, 64, 100, 5000])
def test_attention_windows(dtype, window):
    Attend(window, dtype, 6, 2, 64, 16, LENGTHS + [700], window=window).upload().run().check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lengths,hq,hk,D,P", [([20000], 6, 2, 64, 16), ([9000, 3], 8, 8, 128, 64), ([1] * 500, 4, 2, 64, 16),
                                               ([5000] + [40] * 60, 16, 4, 64, 24), ([3000, 3001], 2, 1, 32, 16),
                                               ([70000], 2, 1, 16, 256), (list(range(0, 900, 9)), 6, 2, 64, 16),
                                               ([3] * 2100 + [200], 2, 1, 32, 16), ([700] + [9] * 2047, 1, 1, 16, 16),
                                               ([600] * 12, 68, 2, 64, 16)])
def test_attention_long_and_ragged_batches(dtype, lengths, hq, hk, D, P):
    """Few long rows are split over the workgroups and joined; many short ones share them."""
    Attend(len(lengths) + D, dtype, hq, hk, D, P, lengths).upload().run().check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_of_several_tokens_a_request(dtype):
    Attend(7, dtype, 6, 2, 64, 16, [5, 64, 130, 1, 2], per=4, pad=3).upload().run().check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D,ldkv,off", [(64, 136, 0), (64, 131, 3), (32, 72, 8), (128, 260, 1), (80, 161, 5)])
def test_attention_strides_and_alignment(dtype, D, ldkv, off):
    Attend(D + off, dtype, 4, 2, D, 16, [3, 100, 33, 64], owners=False, ldkv=max(ldkv, 2 * D), off=off).upload().run().check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 96])
def test_attention_bad_pages_and_empty_rows(dtype, D):
    """Entries that are no pages have no keys; a row of nothing else is 0 and -inf; owners past the requests are left."""
    a = Attend(3, dtype, 6, 2, D, 16, [40, 40, 100, 64, 10])
    a.tab[0, 0] = -1
    a.tab[1, :3] = [-1, a.pages, 2 ** 31 - 1]  # no page at all
    a.tab[2, 2] = -2 ** 31
    a.pos[3] = 2 ** 31 - 1  # further than the table is wide: the table's own positions
    a.tab[3, 4:] = -1
    a.own[4] = len(a.tab)
    want = a.upload().run().check()
    assert want[4] is None and (want[1][1] == -np.inf).all() and (want[1][0] == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lengths,D", [([40, 70, 20], 64), ([40, 7000, 20, 3000], 64), ([40, 70, 20], 20)])
def test_attention_windows_past_the_table(dtype, lengths, D):
    """A position so far past its table that the window holds none of its keys: 0 and -inf, in every form."""
    a = Attend(2, dtype, 6, 2, D, 16, lengths, window=2000 if max(lengths) > 2000 else 30)
    a.pos[0] = 100000
    a.pos[-1] = a.width * 16 + 5
    want = a.upload().run().check()
    assert (want[0][0] == 0).all() and (want[0][1] == -np.inf).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_scores_without_a_share(dtype):
    """Keys whose score is -inf, some of a row's or all of them; scores near the type's limits."""
    a = Attend(4, dtype, 4, 2, 64, 16, [70, 70, 130])
    a.q[:, :, 0] = G.O.round_to(np.abs(a.q[:, :, 0]) + 0.5, dtype)
    for r, picked in ((0, np.arange(0, 70, 3)), (1, np.arange(70)), (2, np.arange(64, 130))):
        a.k[a.tab[r][picked // 16] * 16 + picked % 16, :, 0] = -np.inf
    want = a.upload().run().check()
    assert (want[1][0] == 0).all()
    b = Attend(5, dtype, 4, 2, 64, 16, [90, 20])
    b.k *= np.where(np.arange(len(b.k)) % 5 == 0, 2.0 ** 40, 1.0)[:, None, None]
    b.upload().run()
    o = b.O.host()[:2 * 256]
    assert np.isfinite(o).all() and np.abs(o).max() < 6


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_nan_reaches_its_own_rows_alone(dtype):
    a = Attend(6, dtype, 4, 2, 64, 16, [70, 70, 30])
    a.v[a.tab[1][0] * 16 + 3, 0, 5] = np.nan  # a visible value of request 1, KV head 0
    a.k[a.tab[2][1] * 16 + 2, 1, 0] = np.nan  # a visible key of request 2, KV head 1
    a.upload().run()
    o = a.O.host()[:3 * 256].reshape(3, 2, 2, 64)
    assert np.isfinite(o[0]).all() and np.isnan(o[1, 0, :, 5]).all() and np.isfinite(o[1, 1]).all()
    assert np.isnan(o[2, 1]).all() and np.isfinite(o[2, 0]).all()


def test_attention_without_lse():
    Attend(8, "bf16", 6, 2, 64, 16, [300, 5]).upload().run(lse=False).check(lse=False)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_slots_past_32_bits(dtype):
    """Cache rows whose first element lies past 2^31 elements."""
    N, lib = native()
    ld, P, far = 4096, 16, 600000
    a = Attend(9, dtype, 4, 2, 64, P, [50, 20])
    k, v, pages = a.k, a.v, a.pages
    a.pages = far // P + pages
    K, V = (G.empty(a.pages * P * ld, dtype) for _ in range(2))
    for s in range(len(k)):
        for b, t in ((K, k), (V, v)):
            f = np.nan_to_num(t[s].ravel()).astype(np.float32)
            raw = f if dtype == "f32" else (f.view(np.uint32) >> 16).astype(np.uint16)
            N.api.sj_upload(b.at((far + s) * ld), raw.ctypes.data, raw.nbytes)
    a.k, a.v = a.k[:1], a.v[:1]
    a.upload()
    a.K, a.V, a.ldkv = K, V, ld
    shift = far // P
    a.T = PU.ints(np.where(a.tab >= 0, a.tab + shift, -1))
    a.run()
    a.k, a.v, a.pages = k, v, pages
    a.check()


def test_attention_agrees_with_the_contiguous_cache():
    """Pages in order are sj_attention_fwd_cached's cache."""
    N, lib = native()
    for dtype, D in (("bf16", 64), ("f32", 32)):
        a = Attend(10, dtype, 6, 2, D, 16, [333])
        a.tab[0] = np.arange(a.width)
        a.k, a.v = (G.rnd(t.shape, dtype, a.rng) for t in (a.k, a.v))
        a.upload().run()
        O = G.empty(6 * D, dtype)
        N.api.sj_attention_fwd_cached(None, a.Q.p, 6 * D, a.K.p, a.V.p, 2 * D, 333, CODE[dtype], 1, 332, 6, 2, D, 0, O.p,
                                      6 * D)
        got, want = a.O.host()[:6 * D], O.host()
        assert np.abs(got - want).max() <= np.abs(want).max() * (2.0 ** -7 if dtype == "bf16" else 2.0 ** -18)


def test_two_streams_and_two_graphs_of_one_workspace():
    """Calls on two streams with a workspace each at once; two captured graphs that share one, replayed in turn."""
    N, lib = native()
    a = Attend(11, "bf16", 6, 2, 64, 16, [5000, 700, 1]).upload()
    b = Attend(12, "bf16", 8, 4, 128, 16, [3000, 10]).upload()
    ga, gb = PU.Graph(a.run), PU.Graph(b.run)
    for _ in range(3):
        for x in (a, b):
            x.O.upload(np.full(x.O.n, 55.0))
        ga.do(ga.hip.hipGraphLaunch(ga.exe, ga.stream))
        gb.do(gb.hip.hipGraphLaunch(gb.exe, gb.stream))
        G.sync()
        a.check()
        b.check()
    ga.close()
    gb.close()
    need = max(a.need, b.need, 16)
    shared = G.Dev(need, "u8").upload(np.full(need, 0xFF))
    a.ws = b.ws = shared
    ga, gb = PU.Graph(a.run), PU.Graph(b.run)
    for _ in range(2):
        for g, x in ((ga, a), (gb, b)):
            x.O.upload(np.full(x.O.n, 55.0))
            g.replay()
            x.check()
    ga.close()
    gb.close()


# ---------------------------------------------------------- a run of them

def test_decoding_many_requests_together():
    """A layer's decoding loop as a server runs it, captured once per parity of its double-buffered lengths: plan, QKV
    product, append, attention, output head, token scores, for requests that join with prompts of their own and grow
    over page borders.  Every step against 64 bits from the values that the step itself stored."""
    N, lib = native()
    api = N.api
    rng = np.random.default_rng(21)
    R, P, hq, hk, D, V, steps = 5, 8, 4, 2, 64, 257, 6
    W, J = hq * D, hk * D
    lengths = np.array([0, 7, 8, 15, 30])
    pages, width, table, free = pool(rng, lengths, np.full(R, steps + 2), P)
    total, cap = pages * P, 2 * R  # prompts of 2 tokens in the first step, then one each: the rows behind are padded
    wqkv = G.rnd((W, W + 2 * J), "bf16", rng, W ** -0.5)
    wout = G.rnd((W, V), "f32", rng, W ** -0.5)
    WQ, WO = G.dev(wqkv.T.copy(), "bf16"), G.dev(wout)
    X = G.empty(cap * W, "bf16")
    QKV, Q, O = G.empty(cap * (W + 2 * J), "bf16"), G.zeros(cap * W, "bf16"), G.zeros(cap * W, "bf16")
    k0, v0 = (G.rnd((total, J), "bf16", rng) for _ in range(2))
    K, Vc = G.dev(k0, "bf16"), G.dev(v0, "bf16")
    T, table_d, free_d = PU.turns(D), PU.ints(table), PU.ints(free)
    lens = [PU.ints(lengths), PU.ints(np.zeros(R))]
    heads = [PU.ints([0, 0, 0, 0]), PU.ints([0, 0, 0, 0])]  # two summaries: each step reads the other's list position
    counts, starts = PU.ints(np.full(R, 2)), PU.ints(np.zeros(R + 1))
    pos, slots, own = (PU.ints(np.zeros(cap)) for _ in range(3))
    logits, targets = G.zeros(cap * V), PU.ints(np.zeros(cap))
    lp, ent, stats, ids, alt = G.zeros(cap), G.zeros(cap), G.zeros(2 * cap), PU.ints(np.zeros(3 * cap)), G.zeros(3 * cap)
    need = lib.sj_paged_attention_workspace_bytes(cap, hq, hk, D)
    ws = G.empty(max(need, 16), "u8")
    sn = lib.sj_token_logprobs_workspace_bytes(cap, V, 3)
    sw = G.empty(max(sn, 16), "u8")
    one = ctypes.c_float(1.0)

    def step(i):
        def record(s):
            a, b = i % 2, 1 - i % 2
            api.sj_paged_plan(s, lens[a].p, counts.p, R, P, pages, table_d.p, width, free_d.p, len(free), heads[a].at(1),
                              lens[b].p, starts.p, pos.p, slots.p, own.p, cap, heads[b].p)
            api.sj_qkv_fwd_t(s, X.p, W, cap, W, WQ.p, W, W, J, QKV.p, W + 2 * J, None, 0, D, None, 0)
            api.sj_paged_append(s, QKV.p, W + 2 * J, QKV.at(W), W + 2 * J, QKV.at(W + J), W + 2 * J, 4, cap, hq, hk, D, D,
                                1, pos.p, slots.p, T.p, one, Q.p, W, K.p, Vc.p, J, total)
            api.sj_paged_attention(s, Q.p, W, K.p, Vc.p, J, 4, pages, P, table_d.p, width, R, own.p, pos.p, cap, hq, hk, D,
                                   0, O.p, W, None, ws.p, need)
            api.sj_gemm(s, 0, 0, cap, V, W, O.p, 4, W, WO.p, 0, V, logits.p, 0, V, 0, None, 0)
            api.sj_token_logprobs(s, logits.p, 0, V, cap, V, targets.p, 3, lp.p, ent.p, stats.p, ids.p, alt.p, sw.p, sn)
        return record
    graphs = [PU.Graph(step(0)), PU.Graph(step(1))]
    have, freq, kc, vc, tab, head = lengths.copy(), PU.frequencies(D), k0.copy(), v0.copy(), table.copy(), 0
    for i in range(steps):
        m = np.full(R, 2 if i == 0 else 1)
        if i == 3:
            m[2] = 0  # a request that waits
        x = G.rnd((cap, W), "bf16", rng)
        tg = rng.integers(0, V, cap)
        X.upload(x)
        counts.upload(m)
        targets.upload(tg)
        graphs[i % 2].replay()
        want = PU.plan(have.astype(np.int32), m.astype(np.int32), P, pages, tab, free, head, cap)
        p, s, o = want["rows"]
        for got, w in zip((pos, slots, own), want["rows"]):
            np.testing.assert_array_equal(got.host(), w)
        np.testing.assert_array_equal(table_d.host().reshape(R, width), want["table"])
        np.testing.assert_array_equal(lens[1 - i % 2].host(), want["after"])
        tab, head, have = want["table"], want["head"], have + m
        live = s >= 0
        qkv = QKV.host().reshape(cap, -1)
        G.assert_stored_close(qkv[live], (x @ wqkv)[live], "bf16", "qkv", terms=(np.abs(x) @ np.abs(wqkv))[live])
        q = PU.rotate(qkv[:, :W], hq, D, D, 1, p, freq)
        k = PU.rotate(qkv[:, W:W + J], hk, D, D, 1, p, freq)
        gq, gk, gv = Q.host().reshape(cap, W), K.host().reshape(total, J), Vc.host().reshape(total, J)
        G.assert_stored_close(gq[live], q[live], "bf16", "q", terms=np.full(q[live].shape, 4.0))
        G.assert_stored_close(gk[s[live]], k[live], "bf16", "k", terms=np.full(k[live].shape, 4.0))
        kc[s[live]], vc[s[live]] = gk[s[live]], qkv[live, W + J:]
        np.testing.assert_array_equal(gk, kc)
        np.testing.assert_array_equal(gv, vc)
        go = O.host().reshape(cap, W)
        for r, w in enumerate(PU.attention(gq.reshape(cap, hq, D), kc.reshape(total, hk, D), vc.reshape(total, hk, D), tab, P,
                                           pages, o, p, hq, hk, D)):
            if w is None:
                continue
            tol = (2 * w[3][:, None] + 2.0 ** -15) * w[2] + np.abs(w[0]) * 2.0 ** -8 * 1.01
            assert (np.abs(go[r].reshape(hq, D) - w[0]) <= tol).all()
        lg = logits.host().reshape(cap, V)
        sc = SU.scores(lg, tg, 3)
        np.testing.assert_array_equal(ids.host().reshape(cap, 3), sc["ids"])
        assert np.abs(lp.host() - sc["logprob"]).max() < 2.0 ** -18 and np.abs(ent.host() - sc["entropy"]).max() < 2.0 ** -17
        assert np.abs(alt.host().reshape(cap, 3) - sc["alt"]).max() < 2.0 ** -18
    for g in graphs:
        g.close()


# 129 x 16647160 = 2^31 - 8: the last tile of a walk to the table's end reaches past 2^31
FAR_PAGE, FAR_WIDTH = 129, 16647160


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D,window", [(16, 100), (32, 3000), (64, 100), (64, 3000), (128, 100), (128, 3000), (20, 100)])
def test_attention_at_the_last_positions(dtype, D, window):
    """Tables of nearly 2^31 positions (whose pages are few and shared), windows that end with them, in every form.  A
    key past the first request's table would be in the second's first page, which holds large values."""
    a = Attend(D, dtype, 6, 2, D, FAR_PAGE, [FAR_PAGE] * 4, window=window)
    a.k, a.v = (G.rnd(t.shape, dtype, a.rng) for t in (a.k, a.v))
    far = FAR_PAGE * FAR_WIDTH - 1
    a.tab = np.tile(np.arange(FAR_WIDTH, dtype=np.int32) % 4 + 1, (2, 1))
    a.tab[1, 0] = 0
    a.v[:FAR_PAGE] = 2.0 ** 60
    a.width = FAR_WIDTH
    a.pos, a.own = np.array([far, far - 40, 5]), np.array([0, 0, 1])
    a.q = a.q[:3]
    a.upload().run().check()


def test_attention_over_2_to_the_31_keys():
    """A whole walk of 2^31 - 8 keys, each of four pages as often as the others: o and lse are those of one copy of
    the pages, lse + ln(copies).  A lane adds 4096 tiles' sums one after another and a matrix tile four times as many
    products of two planes: relative 2^-24 each, in the shares' sum and in the values'."""
    a = Attend(31, "bf16", 2, 1, 16, FAR_PAGE, [FAR_PAGE] * 4)
    a.k, a.v = (G.rnd(t.shape, "bf16", a.rng) for t in (a.k, a.v))
    a.tab = (np.arange(FAR_WIDTH, dtype=np.int32) % 4)[None]
    a.width = FAR_WIDTH
    a.pos, a.own, a.q = np.array([FAR_PAGE * FAR_WIDTH - 1]), np.array([0]), a.q[:1]
    a.upload().run()
    k, v, q = a.k[:4 * FAR_PAGE, 0], a.v[:4 * FAR_PAGE, 0], a.q[0]
    s = q @ k.T / 4.0
    e = np.exp(s - s.max(1, keepdims=True))
    o, lse = e @ v / e.sum(1, keepdims=True), s.max(1) + np.log(e.sum(1)) + math.log(FAR_WIDTH // 4)
    mag = e @ np.abs(v) / e.sum(1, keepdims=True)
    steps = 2.0 ** -24 * (4096 + 2 * 4 * 4096 + 1024)
    assert (np.abs(a.O.host()[:32].reshape(2, 16) - o) <= mag * (2 * steps + 2.0 ** -14) + np.abs(o) * 2.0 ** -8).all()
    assert (np.abs(a.L.host()[:2] - lse) <= steps + 2.0 ** -16).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lengths,D", [([20, 1, 7], 64), ([20000, 300], 64), ([20, 1, 7], 20)])
def test_attention_in_place(dtype, lengths, D):
    """o over q, in every form (one workgroup a walk, walks cut into pieces, narrow heads): the same bits as apart."""
    a = Attend(13, dtype, 6, 2, D, 16, lengths).upload().run()
    a.check()
    apart = a.O.host()[:len(lengths) * a.ldq]
    guard = G.dev(np.full(len(lengths) * a.ldq + 8, 55.0), dtype)
    q = np.concatenate([a.q.ravel(), np.full(8, 55.0)])
    a.Q = a.O = guard.upload(q)
    a.run().check()
    np.testing.assert_array_equal(a.O.host()[:len(apart)], apart)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lengths,hq,hk,D", [(LENGTHS, 6, 2, 64), ([20000, 3000, 1], 6, 2, 64), ([9000, 3], 8, 8, 128),
                                             ([4000, 50], 3, 1, 16), ([400, 30], 6, 2, 20), ([5000, 700], 2, 1, 256)])
def test_attention_writes_every_output_again(dtype, lengths, hq, hk, D):
    """The workspace as the last call left it, the outputs refilled: each call writes all of o and lse, the same bits."""
    a = Attend(14, dtype, hq, hk, D, 16, lengths, pad=1).upload().run()
    a.check()
    first = a.O.host(), a.L.host()
    for _ in range(3):
        a.O.upload(np.full(a.O.n, 55.0))
        a.L.upload(np.full(a.L.n, 55.0))
        a.run().check()
        for x, y in zip(first, (a.O, a.L)):
            np.testing.assert_array_equal(y.host()[:len(x)], x)


def test_replays_of_one_workspace_write_every_output():
    """Two graphs that share a workspace, replayed in turn with o and lse refilled, their captured calls' numbers kept."""
    a = Attend(15, "bf16", 6, 2, 64, 16, [5000, 700, 1]).upload()
    b = Attend(16, "f32", 4, 2, 32, 16, [3000, 10]).upload()
    need = max(a.need, b.need)
    a.ws = b.ws = G.Dev(need, "u8").upload(np.full(need, 0xFF))
    graphs = [PU.Graph(x.run) for x in (a, b)]
    for _ in range(3):
        for g, x in zip(graphs, (a, b)):
            x.O.upload(np.full(x.O.n, 55.0))
            x.L.upload(np.full(x.L.n, 55.0))
            g.replay()
            x.check()
    for g in graphs:
        g.close()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lengths,hq,hk,D", [([700] * 70, 6, 2, 64), ([5, 30, 64, 1, 0] * 40, 16, 4, 64),
                                             ([900] + [10] * 300, 8, 4, 128), ([100] * 2100, 2, 1, 32), ([60] * 9, 6, 2, 20)])
def test_attention_of_short_requests_in_wide_tables(dtype, lengths, hq, hk, D):
    """Tables for 131072 tokens, as a server that allows so many keeps them: the form for long walks, whatever the
    lengths."""
    a = Attend(17, dtype, hq, hk, D, 16, lengths)
    a.tab = np.pad(a.tab, ((0, 0), (0, 131072 // 16 - a.width)), constant_values=-1)
    a.width = a.tab.shape[1]
    a.upload().run().check()
