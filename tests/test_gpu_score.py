"""sj_token_logprobs and its gradient against the 64-bit definitions.

Tolerances: a term e^(x - m) is off by its argument's rounding, 2^-24 |x - m|,
and expf's 2^-23; a sum of V of them in fp32, over threads and then a tree, by
at most (V / 64 + 32) 2^-24 of itself."""
import numpy as np
import pytest

from tests import gpu_util as G
from tests import paged_util as PU
from tests import score_util as U

pytestmark = pytest.mark.gpu
ULP = 2.0 ** -24


def native():
    from sejong_amd import _native as N
    return N, N.load()


CODE = {"f32": 0, "bf16": 4}


class Score:
    """One call's buffers, each with guard values behind it."""

    def __init__(self, x, dtype, tokens, top, ld=None, offset=0):
        N, lib = native()
        self.n, self.V, self.top, self.dtype = x.shape[0], x.shape[1], top, dtype
        self.ld = ld or self.V
        wide = np.full((self.n, self.ld), 777.0)  # columns past the vocabulary are never read
        wide[:, :self.V] = x
        flat = np.concatenate([np.zeros(offset), wide.ravel()])
        self.off = offset
        self.x = G.dev(flat, dtype)
        self.tokens = PU.ints(tokens)
        self.lp, self.ent, self.stats = (G.dev(np.full(k * self.n + 4, 55.0)) for k in (1, 1, 2))
        self.ids = PU.ints(np.full(self.n * top + 4, 99))
        self.alt = G.dev(np.full(self.n * top + 4, 55.0))
        self.need = lib.sj_token_logprobs_workspace_bytes(self.n, self.V, top)
        self.ws = G.Dev(max(self.need, 16), "u8").upload(np.full(max(self.need, 16), 0xFF))  # nothing is kept there

    def forward(self, stream=None):
        native()[0].api.sj_token_logprobs(stream, self.x.at(self.off), CODE[self.dtype], self.ld, self.n, self.V,
                                          self.tokens.p, self.top, self.lp.p, self.ent.p, self.stats.p, self.ids.p,
                                          self.alt.p, self.ws.p, self.need)

    def host(self):
        out = [b.host() for b in (self.lp, self.ent, self.stats, self.ids, self.alt)]
        assert all((b[-4:] == (99 if b.dtype == np.int32 else 55.0)).all() for b in out)  # nothing behind the rows
        lp, ent, stats, ids, alt = (b[:-4] for b in out)
        return dict(lp=lp, ent=ent, stats=stats.reshape(-1, 2), ids=ids.reshape(self.n, -1), alt=alt.reshape(self.n, -1))

    def backward(self, dlp, dent, dx_dtype, lddx=None, stream=None):
        lddx = lddx or self.V
        dx = G.dev(np.full(self.n * lddx + 4, 55.0), dx_dtype)
        a = G.dev(dlp) if dlp is not None else None
        b = G.dev(dent) if dent is not None else None
        native()[0].api.sj_token_logprobs_bwd(stream, self.x.at(self.off), CODE[self.dtype], self.ld, self.n, self.V,
                                              self.tokens.p, self.stats.p, self.ent.p, a and a.p, b and b.p, dx.p,
                                              CODE[dx_dtype], lddx)
        h = dx.host()
        assert (h[-4:] == 55.0).all()
        h = h[:-4].reshape(self.n, lddx)
        assert (h[:, self.V:] == 55.0).all()  # columns past the vocabulary are left
        return h[:, :self.V]


def check_forward(got, x, tokens, top):
    want = U.scores(x, tokens, top)
    V = x.shape[1]
    np.testing.assert_array_equal(got["ids"], want["ids"])
    with np.errstate(invalid="ignore"):
        spread = np.abs(x - want["ref"][:, None])
        e_lp = np.where(np.isfinite(want["lp"]), ULP * (8 + 2 * spread + (V / 64 + 32)), 0.0)
    row = ULP * (16 + V / 64 + 32) * (1 + want["ll"])
    tok = np.where(want["ok"], e_lp[np.arange(len(x)), want["at"]], 0.0)
    for name, g, w, tol in (("logprob", got["lp"], want["logprob"], tok),
                            ("alternatives", got["alt"], want["alt"], np.take_along_axis(e_lp, want["ids"], 1)),
                            ("max", got["stats"][:, 0], want["ref"], 0.0), ("log sum", got["stats"][:, 1], want["ll"], row)):
        same = (g == w)  # infinities among them
        with np.errstate(invalid="ignore"):
            assert (same | (np.abs(g - w) <= tol)).all(), (name, np.nanmax(np.abs(g - w) - tol))
    with np.errstate(invalid="ignore"):
        mean = np.where(want["p"] > 0, want["p"] * spread, 0.0).sum(1)
        part = np.where(want["p"] > 0, want["p"] * spread * spread, 0.0).sum(1)
    tol = row * (1 + mean) + ULP * part + 8 * ULP * (want["ll"] + mean)
    assert (np.abs(got["ent"] - want["entropy"]) <= tol).all(), np.max(np.abs(got["ent"] - want["entropy"]) - tol)
    return want


def check_backward(dx, x, tokens, dlp, dent, dtype):
    want, s = U.gradient(x, tokens, dlp, dent), U.scores(x, tokens)
    V = x.shape[1]
    with np.errstate(invalid="ignore"):
        e = ULP * (40 + V / 64 + 2 * np.abs(x - s["ref"][:, None]) + 2 * s["ll"][:, None])
        a = np.abs(dlp)[:, None] if dlp is not None else 0.0
        b = np.abs(dent)[:, None] if dent is not None else 0.0
        lpH = np.where(s["p"] > 0, np.abs(s["lp"]) + s["entropy"][:, None], 0.0)
        tol = np.where(s["p"] > 0, s["p"] * e * (a + b * (1 + lpH)) + s["p"] * b * ULP * (V / 64 + 64) * (2 + lpH), 0.0)
    tol = tol + np.abs(want) * (2.0 ** -8 if dtype == "bf16" else 4 * ULP) + 1e-37
    assert (np.abs(dx - want) <= tol).all(), np.max(np.abs(dx - want) / tol)


def logits(rng, n, V, dtype, spread=2.0):
    x = rng.normal(0, spread, (n, V))
    x[np.arange(n), rng.integers(0, V, n)] += rng.random(n) * 15
    return G.O.round_to(x, dtype)


@pytest.mark.parametrize("n,V,top,dtype,ld,offset", [
    (1, 1, 1, "f32", 0, 0), (3, 2, 2, "bf16", 0, 0), (5, 63, 5, "f32", 64, 1), (70, 257, 5, "f32", 264, 0),
    (33, 257, 20, "bf16", 257, 3), (9, 1000, 64, "f32", 1001, 0), (7, 4099, 8, "bf16", 0, 1), (4, 8193, 32, "f32", 8200, 2),
    (3, 32768, 20, "bf16", 0, 0), (1030, 8300, 3, "bf16", 8301, 0), (690, 16400, 9, "f32", 0, 0), (2, 50001, 1, "bf16", 50008, 0), (2, 131072, 64, "f32", 0, 0), (17, 5000, 0, "f32", 0, 0),
    (1, 200001, 33, "f32", 0, 1), (600, 300, 3, "bf16", 301, 0), (1030, 16, 4, "f32", 0, 0)])
def test_scores_and_gradient(n, V, top, dtype, ld, offset):
    rng = np.random.default_rng(V + n)
    x = logits(rng, n, V, dtype)
    tokens = rng.integers(0, V, n)
    tokens[::3] = x.argmax(1)[::3]
    tokens[1::7] = -1
    tokens[2::7] = V
    s = Score(x, dtype, tokens, top, ld or None, offset)
    s.forward()
    got = s.host()
    check_forward(got, x, tokens, top)
    dlp, dent = rng.normal(size=n).astype(np.float32), rng.normal(size=n).astype(np.float32)
    for a, b, d in ((dlp, dent, dtype), (dlp, None, "f32"), (None, dent, "bf16")):
        check_backward(s.backward(a, b, d, V + (3 if d == "f32" else 0)), x, tokens, a, b, d)
    s.forward()  # the same again: equal bits
    again = s.host()
    assert all((again[k] == got[k]).all() for k in got)


@pytest.mark.parametrize("V", [5, 64, 257, 1000, 9000, 40000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_equal_and_ordered_rows(V, dtype):
    """Ties go to the lowest index; rows sorted either way, constant rows, rows of two values."""
    i = np.arange(V)
    x = np.stack([np.zeros(V), i // 3 * 0.5, (V - i) // 4 * 0.25, i % 2, np.where(i < V // 2, 1.0, -1.0), -(i % 7) * 1.0,
                  np.where(i == V - 1, -0.0, 0.0)])
    x = G.O.round_to(np.clip(x, -60, 60), dtype)
    tokens = np.arange(len(x)) % V
    top = min(V, 48)
    s = Score(x, dtype, tokens, top)
    s.forward()
    check_forward(s.host(), x, tokens, top)


@pytest.mark.parametrize("V", [6, 257, 5000, 33000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_masked_vocabularies(V, dtype):
    """Entries of -inf and of the type's lowest value, rows that hold little or nothing else."""
    rng = np.random.default_rng(V)
    low = float(G.O.round_to(np.array([-3.38e38]), dtype)[0])
    x = logits(rng, 6, V, dtype)
    x[0, ::2] = -np.inf
    x[1] = -np.inf
    x[2] = -np.inf
    x[2, V - 2] = 3.0
    x[3, 1:] = low
    x[4] = low
    x[5, 2:] = -np.inf
    tokens = np.array([1, 0, V - 2, 0, V - 1, 0])
    s = Score(x, dtype, tokens, 5)
    s.forward()
    check_forward(s.host(), x, tokens, 5)
    dlp, dent = np.ones(6, np.float32), np.ones(6, np.float32)
    dx = s.backward(dlp, dent, "f32")
    keep = [0, 2, 3, 4, 5]
    check_backward(dx[keep], x[keep], tokens[keep], dlp[keep], dent[keep], "f32")
    assert np.isfinite(dx).all()


def test_nan_stays_in_its_row_and_ranks_last():
    for V in (40, 300, 20000):
        x = logits(np.random.default_rng(1), 3, V, "f32")
        x[1, 7] = np.nan
        s = Score(x, "f32", np.array([0, 1, 2]), 4)
        s.forward()
        got = s.host()
        assert np.isnan(got["lp"][1]) and np.isnan(got["ent"][1]) and np.isnan(got["alt"][1]).all()
        y = x.copy()
        y[1, 7] = -np.inf
        np.testing.assert_array_equal(got["ids"], U.scores(y, [0, 1, 2], 4)["ids"])
        for r in (0, 2):
            check_forward({k: v[r:r + 1] for k, v in got.items()}, x[r:r + 1], [r], 4)
        dx = s.backward(np.ones(3, np.float32), np.ones(3, np.float32), "f32")
        assert np.isnan(dx[1]).all() and np.isfinite(dx[[0, 2]]).all()


def test_peaked_rows_keep_what_is_beside_the_peak():
    """ln p of the peak is -rest, of the order 1e-8: a sum that holds the peak's 1 would lose it."""
    x = np.zeros((2, 4))
    x[0] = [18.0, 0, -1, -2]
    x[1] = [0, 25.0, 25.0 - 16.0, 3.0]
    tokens = np.array([0, 1])
    s = Score(x, "f32", tokens, 2)
    s.forward()
    got, want = s.host(), U.scores(x, tokens, 2)
    np.testing.assert_allclose(got["lp"], want["logprob"], rtol=1e-5)
    np.testing.assert_allclose(got["ent"], want["entropy"], rtol=1e-5)
    dx = s.backward(np.ones(2, np.float32), np.zeros(2, np.float32), "f32")
    np.testing.assert_allclose(dx, U.gradient(x, tokens, np.ones(2), np.zeros(2)), rtol=1e-5, atol=1e-30)


def test_gradient_against_differences_of_the_forward():
    """The forward's own outputs at x +- h d: the difference is off by h^2 / 6 |f'''| (|f'''| < 8 max|d|^3 sum|w|
    for the log-sum and the entropy's fourth moment) and by the outputs' rounding over h."""
    rng = np.random.default_rng(11)
    n, V, h = 6, 700, 2.0 ** -5
    x = G.O.round_to(rng.normal(0, 1, (n, V)), "bf16")  # x +- h d is exact in fp32
    d = np.sign(rng.normal(size=(n, V)))
    tokens = rng.integers(0, V, n)
    dlp, dent = rng.normal(size=n).astype(np.float32), rng.normal(size=n).astype(np.float32)
    f = []
    for sign in (1, -1):
        s = Score(x + sign * h * d, "f32", tokens, 0)
        s.forward()
        g = s.host()
        f.append(float(dlp.astype(np.float64) @ g["lp"] + dent.astype(np.float64) @ g["ent"]))
    s = Score(x, "f32", tokens, 0)
    s.forward()
    dx = s.backward(dlp, dent, "f32")
    weight = np.abs(dlp).sum() + np.abs(dent).sum() * 10
    assert abs((f[0] - f[1]) / (2 * h) - (dx * d).sum()) < weight * (8 * h * h / 6 + 50 * ULP * 10 / h)


def test_rows_past_32_bits():
    """Rows whose first element lies past 2^31 elements."""
    N, lib = native()
    ld, V = 1 << 30, 300
    x = G.empty(2 * ld + V, "bf16")
    rng = np.random.default_rng(4)
    rows = logits(rng, 3, V, "bf16")
    for r in range(3):
        raw = (rows[r].astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)
        N.api.sj_upload(x.at(r * ld), raw.ctypes.data, raw.nbytes)
    s = Score(rows, "bf16", np.array([5, 6, 7]), 3)
    s.x, s.ld = x, ld
    s.forward()
    check_forward(s.host(), rows, np.array([5, 6, 7]), 3)
    check_backward(s.backward(np.ones(3, np.float32), np.ones(3, np.float32), "f32"), rows, np.array([5, 6, 7]), np.ones(3),
                   np.ones(3), "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [257, 5001])
def test_gradient_in_place(V, dtype):
    N, lib = native()
    rng = np.random.default_rng(V)
    x, tokens = logits(rng, 5, V, dtype), rng.integers(0, V, 5)
    s = Score(x, dtype, tokens, 0)
    s.forward()
    dlp, dent = G.dev(np.ones(5)), G.dev(np.full(5, -0.25))
    want = s.backward(np.ones(5, np.float32), np.full(5, -0.25, np.float32), dtype)
    N.api.sj_token_logprobs_bwd(None, s.x.p, CODE[dtype], V, 5, V, s.tokens.p, s.stats.p, s.ent.p, dlp.p, dent.p, s.x.p,
                                CODE[dtype], V)
    np.testing.assert_array_equal(s.x.host().reshape(5, V), want)


def crowded(n, V, seed):
    """Rows whose largest entries all lie with a few threads: more than LDS holds at the threshold."""
    rng = np.random.default_rng(seed)
    x = rng.normal(0, 1, (n, V))
    at = np.arange(V)
    x[:, (at // 4) % 64 < 40] += 50.0  # of each 64 units of 16 bytes (fp32), 40 tower over the rest
    return G.O.round_to(x, "f32")


@pytest.mark.parametrize("V,top", [(4000, 50), (8192, 64), (30000, 64)])
def test_crowded_rows(V, top):
    x = crowded(2, V, V)
    s = Score(x, "f32", np.array([1, 2]), top)
    s.forward()
    check_forward(s.host(), x, np.array([1, 2]), top)


def test_two_graphs_of_one_workspace():
    """Rows of several slices meet in a workspace that two captured graphs share, replayed in turn."""
    rng = np.random.default_rng(5)
    both = [Score(logits(rng, n, V, "f32"), "f32", rng.integers(0, V, n), 7) for n, V in ((5, 20000), (2, 50000))]
    need = max(s.need for s in both)
    shared = G.Dev(need, "u8").upload(np.full(need, 0xFF))
    for s in both:
        s.ws = shared
    graphs = [PU.Graph(s.forward) for s in both]
    for _ in range(3):
        for g, s in zip(graphs, both):
            x = logits(rng, s.n, s.V, "f32")
            s.x.upload(x)
            g.replay()
            check_forward(s.host(), x, s.tokens.host(), 7)
    for g in graphs:
        g.close()


def test_crowded_slices():
    """Many slices of a long row with 63 large entries each, one fewer than the alternatives asked for."""
    V = 40 * 8192 - 100
    x = np.tile(np.random.default_rng(0).normal(0, 1, V), (2, 1))
    for s in range(40):
        x[:, s * 8192 + np.arange(63) * 120] += 30.0
    x = G.O.round_to(x, "f32")
    s = Score(x, "f32", np.array([5, V - 1]), 64)
    s.forward()
    check_forward(s.host(), x, np.array([5, V - 1]), 64)


@pytest.mark.parametrize("V", [8193, 8200, 16390])
def test_a_last_slice_of_few_entries(V):
    x = logits(np.random.default_rng(V), 3, V, "f32")
    x[1, -3:] = 99.0
    s = Score(x, "f32", np.array([0, V - 1, 7]), 30)
    s.forward()
    check_forward(s.host(), x, np.array([0, V - 1, 7]), 30)


@pytest.mark.parametrize("n,V", [(40, 257), (3, 60000)])
def test_captured_scores_replay(n, V):
    """Forward and backward in one graph; new logits between the replays, every replay against the definitions."""
    rng = np.random.default_rng(9)
    x = logits(rng, n, V, "f32")
    tokens = rng.integers(0, V, n)
    s = Score(x, "f32", tokens, 6)
    N, lib = native()
    dlp, dent, dx = G.dev(np.ones(n)), G.dev(np.full(n, 0.5)), G.empty(n * V)

    def record(stream):
        s.forward(stream)
        N.api.sj_token_logprobs_bwd(stream, s.x.p, 0, s.ld, n, V, s.tokens.p, s.stats.p, s.ent.p, dlp.p, dent.p, dx.p, 0, V)
    g = PU.Graph(record)
    for k in range(3):
        x = logits(rng, n, V, "f32")
        s.x.upload(x)
        g.replay()
        check_forward(s.host(), x, tokens, 6)
        check_backward(dx.host().reshape(n, V), x, tokens, np.ones(n), np.full(n, 0.5), "f32")
    g.close()


@pytest.mark.parametrize("n,V,top,ld,offset", [
    (530, 16384, 64, 16385, 3), (1030, 8200, 40, 8203, 0), (350, 24601, 5, 24601, 1), (520, 16377, 0, 16379, 7),
    (260, 32768, 64, 32768, 8)])
def test_many_long_rows_of_bf16(n, V, top, ld, offset):
    """Many long rows that begin at any of the 8 places of 16 bytes; masked ends and beginnings, equal entries, a row
    of nothing, NaN."""
    rng = np.random.default_rng(V)
    x = logits(rng, n, V, "bf16")
    for r in range(9, n, 10):
        x[r, :rng.integers(1, 40)] = -np.inf
        x[r, V - rng.integers(1, 40):] = -np.inf
    for r in range(16):  # each place twice: entries that count only at the ends, and equal ones
        x[16 + r] = -np.inf
        x[16 + r, 0] = x[16 + r, V - 1] = 1.0
        x[32 + r] = -2.5
        x[48 + r, :9] = x[48 + r, V - 9:] = 30.0
    x[5] = -np.inf
    x[6] = G.O.round_to(np.array([-3.38e38]), "bf16")[0]
    tokens = rng.integers(0, V, n)
    tokens[::2], tokens[1::4] = 0, V - 1
    s = Score(x, "bf16", tokens, top, ld, offset)
    s.forward()
    check_forward(s.host(), x, tokens, top)
    y = x[:8].copy()
    y[3, 0], y[4, V - 1] = np.nan, np.nan
    y = np.concatenate([y, x[8:]])
    s = Score(y, "bf16", tokens, top, ld, offset)
    s.forward()
    got = s.host()
    assert np.isnan(got["lp"][3:5]).all() and np.isnan(got["ent"][3:5]).all()
    keep = np.r_[0:3, 5:n]
    check_forward({k: v[keep] for k, v in got.items()}, x[keep], tokens[keep], top)


@pytest.mark.parametrize("n,V,dtype", [(3, 1025, "bf16"), (2, 1025, "f32"), (300, 4096, "bf16"), (2, 8192, "f32"),
                                       (3, 50001, "f32"), (530, 16390, "f32")])
def test_long_lists(n, V, dtype):
    """33, 48 and 64 alternatives, with entries of -inf that leave fewer than those, and -inf almost everywhere."""
    rng = np.random.default_rng(n + V)
    x = logits(rng, n, V, dtype)
    x[0, 20:] = -np.inf
    x[1, rng.permutation(V)[:V - 64]] = -np.inf
    tokens = rng.integers(0, V, n)
    for top in (33, 48, 64):
        s = Score(x, dtype, tokens, top)
        s.forward()
        check_forward(s.host(), x, tokens, top)


def check_long_rows(got, x, tokens, top):
    """As check_forward, with the sums counted as they are formed: a term is off by 2 |x - m| + 5 units (its argument's
    two roundings, the power, the factor back to the maximum), and again 2 |m_s - m| + 4 from its slice's maximum to
    the row's; a thread adds 64 terms, then 8 levels, 8 slices at most and 8 levels: 100 + 4 |x - m| in all."""
    want = U.scores(x, tokens, top)
    np.testing.assert_array_equal(got["ids"], want["ids"])
    with np.errstate(invalid="ignore"):
        spread = np.abs(x - want["ref"][:, None])
        mean = np.where(want["p"] > 0, want["p"] * spread, 0.0).sum(1)
        part = np.where(want["p"] > 0, want["p"] * spread * spread, 0.0).sum(1)
    total = ULP * (100 + 4 * mean)
    log = total + 2 * ULP * (want["ll"] + 2)
    assert (got["stats"][:, 0] == want["ref"]).all()
    assert (np.abs(got["stats"][:, 1] - want["ll"]) <= log).all()

    def close(g, w, d, tol):
        with np.errstate(invalid="ignore"):
            near = np.isfinite(w) & (np.abs(g - w) <= tol + 2 * ULP * (d + np.abs(w)))
            assert (near | (g == w)).all(), np.nanmax(np.abs(g - w))
    rows = np.arange(len(x))
    close(got["lp"], want["logprob"], spread[rows, want["at"]], log)
    close(got["alt"], want["alt"], np.take_along_axis(spread, want["ids"], 1), log[:, None])
    tol = log + ULP * (104 * mean + 4 * part) + total * mean + 8 * ULP * (want["ll"] + mean)
    assert (np.abs(got["ent"] - want["entropy"]) <= tol).all(), np.max(np.abs(got["ent"] - want["entropy"]) / tol)


def many_slices(n, V, dtype, seed):
    """Rows of very many slices: the largest value twice, 256 slices of 8192 or 16384 apart; nothing but -inf in most
    slices or in all; equal entries; the largest at either end."""
    x = logits(np.random.default_rng(seed), n, V, dtype)
    i = np.arange(V)
    for at in (3 * 8192 + 5, 259 * 8192 + 7, 3 * 16384 + 9, 259 * 16384 + 11):
        if at < V:
            x[0, at] = 24.0
    if n > 1:
        x[1, (i // 8192) % 50 != 7] = -np.inf
    if n > 2:
        x[2] = -np.inf
        x[2, [V - 1, V // 2, 12345]] = [1.0, 2.0, 1.0]
    if n > 3:
        x[3] = -np.inf
    if n > 4:
        x[4] = -1.5
    if n > 5:
        x[5, 0] = x[5, V - 1] = 30.0
    return x


@pytest.mark.parametrize("n,V,dtype,top", [
    (6, 70 * 8192 - 77, "f32", 20), (6, 70 * 8192 - 77, "f32", 64), (15, 70 * 8192, "f32", 1), (15, 70 * 8192, "f32", 64),
    (3, 300 * 8192 - 8191, "f32", 64), (3, 300 * 8192 - 1, "f32", 1), (4, 300 * 8192 - 77, "f32", 20),
    (4, 270 * 8192 - 77, "f32", 64), (2, 300 * 8192 - 3, "bf16", 20), (1, 600 * 8192 - 77, "bf16", 64),
    (2, 300 * 16384 - 77, "bf16", 1), (2, 300 * 16384 - 77, "bf16", 64), (16, 70 * 16384 - 5, "bf16", 20),
    (1, 1 << 24, "f32", 64), (1, 1 << 24, "bf16", 5)])
def test_rows_of_many_slices(n, V, dtype, top):
    """More than 64 slices and more than 256, met within the launch (up to 1024 in all) and joined by a second one."""
    x = many_slices(n, V, dtype, V + n)
    tokens = np.random.default_rng(n).integers(0, V, n)
    tokens[0] = 3 * 8192 + 5
    s = Score(x, dtype, tokens, top)
    s.forward()
    check_long_rows(s.host(), x, tokens, top)


def refill(s):
    """Guard values in every output of a call."""
    for b, v in ((s.lp, 55.0), (s.ent, 55.0), (s.stats, 55.0), (s.ids, 99), (s.alt, 55.0)):
        b.upload(np.full(b.n, v))


@pytest.mark.parametrize("n,V,dtype,top", [(5, 257, "f32", 5), (3, 4099, "bf16", 8), (4, 50001, "f32", 20),
                                           (2, 131072, "bf16", 64), (600, 16400, "f32", 3), (300, 40000, "bf16", 0)])
def test_scores_write_every_output_again(n, V, dtype, top):
    """The workspace as the last call left it, the outputs refilled: each call writes all of them, the same bits."""
    rng = np.random.default_rng(V)
    x, tokens = logits(rng, n, V, dtype), rng.integers(0, V, n)
    s = Score(x, dtype, tokens, top)
    s.forward()
    first = s.host()
    check_forward(first, x, tokens, top)
    for _ in range(3):
        refill(s)
        s.forward()
        again = s.host()
        for k in first:
            np.testing.assert_array_equal(again[k], first[k])


def test_scores_on_two_streams_at_once():
    """Rows of several slices on two streams with a workspace each, several times, outputs refilled."""
    rng = np.random.default_rng(8)
    both = [Score(logits(rng, n, V, d), d, rng.integers(0, V, n), 9) for n, V, d in ((12, 60000, "f32"), (5, 131072, "bf16"))]
    graphs = [PU.Graph(s.forward) for s in both]
    for _ in range(3):
        data = []
        for s in both:
            refill(s)
            data.append(logits(rng, s.n, s.V, s.dtype))
            s.x.upload(data[-1])
        for g in graphs:
            g.do(g.hip.hipGraphLaunch(g.exe, g.stream))
        G.sync()
        for s, x in zip(both, data):
            check_forward(s.host(), x, s.tokens.host(), 9)
    for g in graphs:
        g.close()
