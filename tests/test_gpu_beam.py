"""Beam search's selection against 64 bits, and a search over the paged cache
with all its calls together."""
import ctypes

import numpy as np
import pytest

from tests import beam_util as BU
from tests import gpu_util as G
from tests import paged_util as PU

pytestmark = pytest.mark.gpu
CODE = {"f32": 0, "bf16": 4}


def native():
    from sejong_amd import _native as N
    return N, N.load()


class Select:
    def __init__(self, x, scores, beams, keep, dtype="f32", lengths=None, ended=None, end=-1, power=0.0, ld=0, off=0):
        self.x, self.scores = x, np.asarray(scores, np.float32)
        if dtype == "f32":  # the oracle reads what the device holds
            with np.errstate(over="ignore"):
                self.x = x = x.astype(np.float32).astype(np.float64)
        self.rows, self.V = x.shape
        self.beams, self.keep, self.dtype, self.end, self.power = beams, keep, dtype, end, power
        self.lengths, self.ended, self.off = lengths, ended, off
        self.ld = ld or self.V
        wide = np.full((self.rows, self.ld), 77.0)
        wide[:, :self.V] = x
        self.X = G.dev(np.concatenate([np.zeros(off), wide.ravel()]), dtype)
        self.S = G.dev(self.scores)
        self.L = None if lengths is None else PU.ints(lengths)
        self.E = None if ended is None else PU.ints(ended)
        self.groups = self.rows // beams
        m = self.groups * keep
        self.ints = [PU.ints(np.full(m + 1, 55)) for _ in range(4)]
        self.out = G.dev(np.full(m + 1, 55.0))
        need = native()[1].sj_beam_select_workspace_bytes(self.groups, beams, self.V, keep)
        self.need = need
        self.ws = G.Dev(max(need, 16), "u8").upload(np.full(max(need, 16), 0xFF))

    def run(self, stream=None):
        p, t, n, e = self.ints
        native()[0].api.sj_beam_select(stream, self.X.at(self.off), CODE[self.dtype], self.ld, self.groups, self.beams, self.V,
                                       self.S.p, self.L and self.L.p, self.E and self.E.p, self.end, self.power, self.keep,
                                       p.p, t.p, self.out.p, n.p if self.L else None, e.p, self.ws.p, self.need)
        return self

    def clear(self):
        for b in self.ints + [self.out]:
            b.upload(np.full(b.n, 55))

    def check(self):
        want = BU.select(self.x, self.scores.astype(np.float64), self.beams, self.keep, self.lengths, self.ended, self.end,
                         self.power)
        for got, key in zip(self.ints, ("parents", "tokens", "lengths", "ended")):
            h = got.host()
            assert h[-1] == 55
            if key != "lengths" or self.L:
                np.testing.assert_array_equal(h[:-1], want[key], key)
        s = self.out.host()
        assert s[-1] == 55
        s, w = s[:-1], want["scores"]
        none = w == -np.inf
        assert (s[none] == -np.inf).all()
        # totals of 64 bits, the sum's powers to 7.8e-13: one rounding to fp32; and one of the logarithm on each side,
        # which has the size of its row's largest logit
        large = np.abs(np.nan_to_num(self.x.max(1), nan=0.0, neginf=0.0))[want["parents"][~none]]
        assert (np.abs(s[~none] - w[~none]) <= np.abs(w[~none]) * 2.0 ** -24 * 1.001 + 1e-12 + large * 2.0 ** -52).all()
        return want


def logits(rng, rows, V, dtype, likely=6):
    x = rng.normal(0, 2, (rows, V))
    for _ in range(likely):
        x[np.arange(rows), rng.integers(0, V, rows)] += rng.uniform(0, 12, rows)
    return G.O.round_to(x, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V,groups,beams,keep", [(1, 3, 2, 4), (2, 3, 1, 2), (7, 5, 3, 8), (257, 9, 4, 4), (257, 2, 33, 64),
                                                 (511, 1, 1, 64), (512, 3, 5, 5), (513, 4, 2, 40), (1024, 2, 4, 8),
                                                 (1025, 3, 4, 8), (4096, 2, 3, 64), (4097, 2, 4, 6), (8192, 2, 2, 33),
                                                 (8193, 2, 3, 16), (20000, 3, 8, 8), (50001, 2, 4, 64), (131072, 1, 3, 16),
                                                 (70000, 1, 64, 64)])
def test_select(dtype, V, groups, beams, keep):
    rng = np.random.default_rng(V + beams)
    rows = groups * beams
    s = Select(logits(rng, rows, V, dtype), rng.normal(-20, 2, rows), beams, keep, dtype, lengths=rng.integers(1, 50, rows))
    s.run().check()
    first = [b.host().copy() for b in s.ints + [s.out]]
    s.clear()
    s.run()
    assert all((a == b.host()).all() for a, b in zip(first, s.ints + [s.out]))  # every output again, the same bits


@pytest.mark.parametrize("beams,slices,keep", [(1, 1, 11), (5, 1, 11), (31, 2, 11), (63, 2, 11), (64, 2, 11), (43, 3, 11),
                                               (17, 11, 11), (51, 5, 11), (64, 4, 11), (37, 7, 11), (1, 1, 40), (5, 1, 64),
                                               (17, 11, 33), (64, 4, 64), (37, 7, 64)])
def test_select_lists_of_any_number(beams, slices, keep):
    """As many lists as threads of the workgroup that takes them together, half as many, a few more, a few less."""
    rng = np.random.default_rng(beams)
    x = logits(rng, beams, 4096 * slices - 5, "f32")
    Select(x, rng.normal(-20, 2, beams), beams, keep, "f32", lengths=np.full(beams, 3)).run().check()


@pytest.mark.parametrize("V", [5, 257, 3000, 9000])
@pytest.mark.parametrize("power", [0.0, 0.6, 1.0, 16.0])
def test_select_with_ended_beams(V, power):
    """Ended beams compete with their own score and length; the rows of their logits hold NaN."""
    rng = np.random.default_rng(V)
    groups, beams, keep = 12, 4, 6
    rows = groups * beams
    x = logits(rng, rows, V, "f32")
    ended = (rng.random(rows) < 0.4).astype(int)
    ended[:4] = 1  # a prompt whose beams have all ended: fewer candidates than places
    x[ended == 1] = np.nan
    x[:, 3] += 6.0  # ending is likely
    lengths = rng.integers(0, 30, rows)
    want = Select(x, rng.normal(-8, 3, rows), beams, keep, "f32", lengths, ended, 3, power).run().check()
    assert (want["tokens"][:6] == [3, 3, 3, 3, -1, -1]).all() and want["ended"].sum() > 6


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [257, 2000, 30000])
def test_select_first_step(dtype, V):
    """One live beam of each prompt, the others' scores -inf; and prompts without any."""
    rng = np.random.default_rng(V)
    scores = np.full((4, 5), -np.inf)
    scores[:3, 0] = 0.0
    s = Select(logits(rng, 20, V, dtype), scores.ravel(), 5, 5, dtype).run()
    want = s.check()
    assert (want["parents"][:15].reshape(3, 5) == np.arange(3)[:, None] * 5).all() and (want["parents"][15:] == -1).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [300, 900, 5000, 200000])
@pytest.mark.parametrize("size", [3e2, 1e6, 2.0 ** 33, 1e30])
def test_select_large_logits(dtype, V, size):
    """Differences past every power's range, at sizes where fp32 cannot hold the maximum less a few hundred."""
    rng = np.random.default_rng(V)
    x = rng.normal(0, 1, (8, V)) * size
    x[:, 7] = x[:, 11] = np.abs(x).max(1)  # two tokens have all of the row
    Select(G.O.round_to(x, dtype), rng.normal(-8, 3, 8), 4, 7, dtype, lengths=np.full(8, 5)).run().check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [300, 900, 5000])
@pytest.mark.parametrize("size", [-1000.0, 1100.0, -7e4, 1e6, 2.0 ** 40, 1e30, -1e30])
def test_select_logits_near_a_large_one(dtype, V, size):
    """All logits lie near one far from 0, at the largest sizes on it."""
    rng = np.random.default_rng(V)
    x = G.O.round_to(size + rng.normal(0, 2, (8, V)), dtype)
    Select(x, rng.normal(-8, 3, 8), 4, 7, dtype, lengths=np.full(8, 5)).run().check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [40, 900, 5000, 40000])
def test_select_masked_entries(dtype, V):
    """Rows whose mask leaves a few tokens, one, or none; masks of the type's lowest value, which are candidates still."""
    rng = np.random.default_rng(V)
    x = logits(rng, 8, V, dtype)
    x[0, 3:] = -np.inf
    x[1, :] = -np.inf
    x[2, :-1] = -np.inf
    x[3, rng.random(V) < 0.9] = -np.inf
    x[4, 2:] = G.O.round_to(np.array([-3.3e38]), dtype)[0]
    x[5, :] = -np.inf
    Select(x, np.zeros(8), 2, 16, dtype, lengths=np.zeros(8, int)).run().check()


@pytest.mark.parametrize("V", [257, 5000, 20000])
def test_select_rows_that_are_not_finite(V):
    """NaN or +inf in a row, scores of NaN and +inf: such beams have no candidates, the others of the prompt do."""
    rng = np.random.default_rng(V)
    x = logits(rng, 15, V, "f32")
    x[0, V // 2] = np.nan
    x[4, V - 1] = np.inf
    x[6:9, 7] = np.nan  # no candidate at all
    scores = rng.normal(-5, 1, 15)
    scores[10], scores[11], scores[13] = np.nan, np.inf, -np.inf
    want = Select(x, scores, 3, 4).run().check()
    assert (want["parents"][8:12] == -1).all() and 0 not in want["parents"] and 4 not in want["parents"]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [100, 257, 3000, 9000, 60000])
def test_select_ties_go_to_the_lowest_index(dtype, V):
    """Equal logits within a row, whole rows of one value, and beams that are copies of each other."""
    rng = np.random.default_rng(V)
    x = G.O.round_to(np.round(rng.normal(0, 1, (12, V))), dtype)
    x[3:6] = 1.25
    x[7] = x[6]
    x[8] = x[6]
    scores = np.repeat([-3.0, -1.0, -2.0, -4.0], 3)
    want = Select(x, scores, 3, 20, dtype).run().check()
    assert (want["tokens"][20:40] == np.arange(20)).all()


@pytest.mark.parametrize("values", [1, 2, 40])
@pytest.mark.parametrize("V,beams,keep", [(100, 8, 64), (300, 8, 32), (9000, 6, 64), (5000, 3, 64)])
def test_select_many_entries_of_few_ranks(values, V, beams, keep):
    """Hundreds of candidates at the threshold, all of one rank or of few."""
    rng = np.random.default_rng(V)
    x = rng.integers(0, values, (2 * beams, V)) * 0.25
    x[:] = np.sort(x[:1], 1)[:, rng.permutation(V)]  # every row has the same sum
    Select(x, np.full(2 * beams, -4.0), beams, keep, "f32", lengths=np.full(2 * beams, 3)).run().check()


def test_select_totals_next_to_each_other():
    """Beams whose totals differ by less than fp32 holds of them: the order is that of 64 bits."""
    rng = np.random.default_rng(1)
    V, beams = 5000, 4
    x = logits(rng, 40, V, "f32")
    scores = np.zeros(40, np.float32)
    for g in range(0, 40, 4):
        x[g + 1:g + 4] = x[g]
        v = np.abs(x[g] + 2.0).argmin()
        for b in range(1, 4):  # one small entry is a little less: the sum moves by some 1e-7 of itself
            x[g + b, v] = np.float32(x[g, v] - 0.3 * b)
        scores[g:g + 4] = -40.0
    want = BU.select(x, scores.astype(float), beams, 16)
    gaps = -np.diff(want["ranks"].reshape(10, 16))
    assert ((gaps > 1e-11) & (gaps < 2e-6)).sum() > 20  # an fp32 total of 40 is good to 4e-6
    Select(x, scores, beams, 16).run().check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V,ld,off", [(257, 260, 1), (257, 257, 3), (3001, 3003, 5), (9001, 9001, 1), (20003, 20011, 7)])
def test_select_strides_and_alignment(dtype, V, ld, off):
    rng = np.random.default_rng(V)
    Select(logits(rng, 12, V, dtype), rng.normal(-9, 1, 12), 4, 7, dtype, ld=ld, off=off).run().check()


@pytest.mark.parametrize("V,beams", [(257, 4), (20000, 3), (60000, 8)])
def test_select_two_streams_and_replays(V, beams):
    """Two captured calls at once with a workspace each, then two that share one in turn; every replay writes every
    output again."""
    rng = np.random.default_rng(beams)
    a, b = (Select(logits(rng, 5 * beams, V, "bf16"), rng.normal(-9, 1, 5 * beams), beams, beams, "bf16",
                   lengths=np.full(5 * beams, 4), power=0.5) for _ in range(2))
    ga, gb = PU.Graph(a.run), PU.Graph(b.run)
    for _ in range(3):
        a.clear(), b.clear()
        ga.do(ga.hip.hipGraphLaunch(ga.exe, ga.stream))
        gb.do(gb.hip.hipGraphLaunch(gb.exe, gb.stream))
        G.sync()
        a.check(), b.check()
    ga.close(), gb.close()
    b.ws = a.ws
    ga, gb = PU.Graph(a.run), PU.Graph(b.run)
    for _ in range(2):
        for g, s in ((ga, a), (gb, b)):
            s.clear()
            g.replay()
            s.check()
    ga.close(), gb.close()


# ---------------------------------------------------------- a run of them

def test_a_search_over_the_paged_cache():
    """Beam search as a server runs it, a step captured once per parity of its double-buffered state: the plan of the
    live beams, QKV product, append, attention over the shared prompt, output head, selection, fork, copies.  Every step
    against the plain forms, from the values that the step itself stored."""
    N, lib = native()
    api = N.api
    rng = np.random.default_rng(9)
    groups, B, P, hq, hk, D, V, steps, END = 3, 4, 8, 4, 2, 64, 257, 7, 5
    R, W, J = groups * B, hq * D, hk * D
    prompt = np.array([21, 8, 40])
    # wide tables: attention walks the shared prefixes for all of a prompt's beams together
    width = max(int(-(-(prompt.max() + steps + 2) // P)), 2 ** 24 // (R * hk * D) // P + 1)
    pages = 80
    order = rng.permutation(pages)
    table, shared, made = np.full((R, width), -1), np.zeros(pages, int), 0
    for g in range(groups):  # the prompts' whole pages are shared, what is left of them each beam has
        full, cols = prompt[g] // P, -(-prompt[g] // P)
        for b in range(B):
            r = g * B + b
            if b == 0:
                table[r, :full] = order[made:made + full]
                made += full
            else:
                table[r, :full] = table[g * B, :full]
                shared[table[r, :full]] += 1
            if cols > full:
                table[r, full] = order[made]
                made += 1
    free = np.concatenate([np.full(made, -1), order[made:]])
    total = pages * P
    kc, vc = (G.rnd((total, J), "bf16", rng) for _ in range(2))
    for g in range(groups):  # copies of the prompt's last page hold the same
        for b in range(1, B):
            full = prompt[g] // P
            if prompt[g] % P:
                s, d = table[g * B, full] * P, table[g * B + b, full] * P
                kc[d:d + P], vc[d:d + P] = kc[s:s + P], vc[s:s + P]
    wqkv, wout = G.rnd((W, W + 2 * J), "bf16", rng, W ** -0.5), G.rnd((W, V), "f32", rng, 1.0)
    emb = G.rnd((V, W), "bf16", rng)
    WQ, WO, EMB = G.dev(wqkv.T.copy(), "bf16"), G.dev(wout), G.dev(emb, "bf16")
    X, QKV, Q, O = G.empty(R * W, "bf16"), G.empty(R * (W + 2 * J), "bf16"), G.zeros(R * W, "bf16"), G.zeros(R * W, "bf16")
    K, Vc, T = G.dev(kc, "bf16"), G.dev(vc, "bf16"), PU.turns(D)

    def two(a):
        return [PU.ints(a), PU.ints(a)]

    tables, lens = two(table), two(np.repeat(prompt, B))
    planned = PU.ints(np.zeros(R))
    holders, lists, heads = two(shared), two(free), two([0, made, 0, 0])
    mid = PU.ints([0, made, 0, 0])
    scores = [G.dev(np.tile([0.0, -np.inf, -np.inf, -np.inf], groups)), G.zeros(R)]
    gen, ended = two(np.zeros(R)), two(np.zeros(R))
    ids, parents, copies = PU.ints(np.zeros(R)), PU.ints(np.zeros(R)), PU.ints(np.zeros(3 * R))
    counts, starts = PU.ints(np.ones(R)), PU.ints(np.zeros(R + 1))
    pos, slots, own = (PU.ints(np.zeros(R)) for _ in range(3))
    gs, prefix, logit = PU.ints(np.arange(groups + 1) * B), PU.ints(prompt // P * P), G.zeros(R * V)
    sizes = [lib.sj_paged_attention_shared_workspace_bytes(R, hq, hk, D, groups),
             lib.sj_beam_select_workspace_bytes(groups, B, V, B), lib.sj_paged_fork_workspace_bytes(R, R, pages)]
    need = max(sizes)
    ws = G.Dev(need, "u8").upload(np.full(need, 0xFF))  # one workspace for all calls

    def step(i):
        def record(s):
            a, b = i % 2, 1 - i % 2
            api.sj_paged_plan(s, lens[a].p, counts.p, R, P, pages, tables[a].p, width, lists[a].p, pages, heads[a].at(1),
                              planned.p, starts.p, pos.p, slots.p, own.p, R, mid.p)
            api.sj_embedding_fwd(s, EMB.p, 4, ids.p, X.p, 4, R, W)
            api.sj_qkv_fwd_t(s, X.p, W, R, W, WQ.p, W, W, J, QKV.p, W + 2 * J, None, 0, D, None, 0)
            api.sj_paged_append(s, QKV.p, W + 2 * J, QKV.at(W), W + 2 * J, QKV.at(W + J), W + 2 * J, 4, R, hq, hk, D, D, 1,
                                pos.p, slots.p, T.p, ctypes.c_float(1.0), Q.p, W, K.p, Vc.p, J, total)
            api.sj_paged_attention_shared(s, Q.p, W, K.p, Vc.p, J, 4, pages, P, tables[a].p, width, R, own.p, pos.p, R,
                                          starts.p, gs.p, prefix.p, groups, hq, hk, D, 0, O.p, W, None, ws.p, need)
            api.sj_gemm(s, 0, 0, R, V, W, O.p, 4, W, WO.p, 0, V, logit.p, 0, V, 0, None, 0)
            api.sj_beam_select(s, logit.p, 0, V, groups, B, V, scores[a].p, gen[a].p, ended[a].p, END, 0.7, B, parents.p,
                               ids.p, scores[b].p, gen[b].p, ended[b].p, ws.p, need)
            api.sj_paged_fork(s, parents.p, R, tables[a].p, width, planned.p, R, P, pages, holders[a].p, lists[a].p, pages,
                              mid.at(1), tables[b].p, lens[b].p, holders[b].p, lists[b].p, copies.p, heads[b].p, ws.p, need)
            api.sj_paged_copy(s, K.p, Vc.p, J, 4, 1, 0, pages, P, J, copies.p, R)
        return record
    graphs = [PU.Graph(step(0)), PU.Graph(step(1))]
    have, head, freq = np.repeat(prompt, B), made, PU.frequencies(D)
    sc, gl, en, tok = np.tile([0.0, -np.inf, -np.inf, -np.inf], groups), np.zeros(R, int), np.zeros(R, int), np.zeros(R, int)
    moved = 0
    for i in range(steps):
        a, b = i % 2, 1 - i % 2
        graphs[i % 2].replay()
        plan = PU.plan(have.astype(np.int32), np.ones(R, np.int32), P, pages, table.astype(np.int32), free, head, R)
        assert plan["status"] == 0
        p, s, o = plan["rows"]
        np.testing.assert_array_equal(slots.host(), s)
        table, head, have = plan["table"], plan["head"], have + 1
        qkv = QKV.host().reshape(R, -1)
        x = emb[tok]
        G.assert_stored_close(qkv, x @ wqkv, "bf16", "qkv", terms=np.abs(x) @ np.abs(wqkv))
        kr = PU.rotate(qkv[:, W:W + J], hk, D, D, 1, p, freq)
        kc[s], vc[s] = G.O.round_to(kr, "bf16"), qkv[:, W + J:]
        gq, gk = Q.host().reshape(R, W), K.host().reshape(total, J)
        # the copies behind the selection have changed the cache already: compare after them, below
        lg = logit.host().reshape(R, V)
        want = BU.select(lg, sc, B, B, gl, en, END, 0.7)
        for got, key in ((parents, "parents"), (ids, "tokens"), (gen[b], "lengths"), (ended[b], "ended")):
            np.testing.assert_array_equal(got.host(), want[key], key)
        w32 = want["scores"].astype(np.float32).astype(float)
        fin = np.isfinite(w32)
        gs_ = scores[b].host()
        assert (gs_[~fin] == w32[~fin]).all() and (np.abs(gs_ - w32)[fin] <= np.abs(w32[fin]) * 2.0 ** -23).all()
        go = O.host().reshape(R, W)
        # the step's own key, as it was stored (a copy does not touch it: its page is written by its row alone)
        live = np.array([r for r in range(R) if np.isfinite(sc[r])])
        for r, w in enumerate(PU.attention(gq.reshape(R, hq, D), kc.reshape(total, hk, D), vc.reshape(total, hk, D), table, P,
                                           pages, o, p, hq, hk, D)):
            if r not in live:
                continue
            # a key that the product stored as its neighbour in bf16 moves a score by up to 2^-8 of its terms
            step_key = (np.abs(gq[r].reshape(hq, D)) @ np.ones(D)).max() * np.abs(kr[r]).max() * 2.0 ** -8 * D ** -0.5
            tol = (2 * w[3][:, None] + 2 * step_key + 2.0 ** -15) * w[2] + np.abs(w[0]) * 2.0 ** -8 * 1.01
            assert (np.abs(go[r].reshape(hq, D) - w[0]) <= tol).all()
        f = BU.fork(want["parents"], table, have, P, pages, shared, free, head)
        assert f["status"] == 0 and f["head"] == heads[b].host()[1]
        for got, key in ((tables[b], "table"), (lens[b], "lengths"), (holders[b], "shared"), (lists[b], "free"),
                         (copies, "copies")):
            np.testing.assert_array_equal(got.host(), f[key].ravel(), key)
        gv = Vc.host().reshape(total, J)
        moved += f["taken"]
        BU.copy(kc[None], f["copies"], P, J), BU.copy(vc[None], f["copies"], P, J)
        np.testing.assert_array_equal(gv, vc)
        G.assert_stored_close(gk, kc, "bf16", "k", terms=np.full(kc.shape, 4.0))
        kc = gk.copy()
        table, have, shared, free, head = f["table"], f["lengths"], f["shared"], f["free"], f["head"]
        sc, gl, en, tok = gs_, want["lengths"], want["ended"], want["tokens"]
        assert (tok >= 0).all()
    assert moved > 5
    for g in graphs:
        g.close()
