"""Attention of requests that share the beginning of their sequences: against
64 bits through every request's own table row."""
import numpy as np
import pytest

from tests import gpu_util as G
from tests import paged_util as PU
from tests.test_gpu_paged import CODE, Attend, native

pytestmark = pytest.mark.gpu


class Shared(Attend):
    """groups: (prefix, own tokens of each request); alone: lengths of requests in no group.  Prefixes' whole pages are
    shared, the rest of a prefix lies in each request's own page; unused slots hold NaN."""

    def __init__(self, seed, dtype, hq, hk, D, P, groups, alone=(), per=1, **kw):
        own = [prefix + n for prefix, tails in groups for n in tails]
        super().__init__(seed, dtype, hq, hk, D, P, own + list(alone), per=per, **kw)
        n = len(own) + len(alone)
        self.prefix = np.array([prefix for prefix, _ in groups], np.int64)
        self.first = np.concatenate([[0], np.cumsum([len(tails) for _, tails in groups])]).astype(np.int64)
        for g, (prefix, tails) in enumerate(groups):
            lead = self.tab[self.first[g]]
            for r in range(self.first[g] + 1, self.first[g + 1]):
                self.tab[r, :prefix // P] = lead[:prefix // P]
                for j in range(prefix // P * P, prefix):
                    s, d = lead[j // P] * P + j % P, self.tab[r, j // P] * P + j % P
                    self.k[d], self.v[d] = self.k[s], self.v[s]
        # rows in the order of their requests, as the plan gives them
        pad = len(self.pos) - n * per
        order = np.concatenate([np.arange(n)[:, None] + n * np.arange(per)[None, :]]).ravel()
        order = np.concatenate([order, np.arange(n * per, n * per + pad)]).astype(int)
        self.pos, self.own, self.q = self.pos[order], self.own[order], self.q[order]
        self.starts = np.arange(n + 1) * per
        self.use_starts = True

    # calls on small tables go through sj_paged_attention: with empty columns these are large ones
    wide = True

    def upload(self):
        n = len(self.pos)
        if self.wide:
            keys = 2 ** 24 // (n * self.hk * self.D) + 1
            more = np.full((len(self.tab), max(keys // self.P + 1 - self.width, 0)), -1)
            self.tab = np.concatenate([self.tab, more], 1)
            self.width = self.tab.shape[1]
        super().upload()
        self.need = native()[1].sj_paged_attention_shared_workspace_bytes(n, self.hq, self.hk, self.D, len(self.prefix))
        self.ws = G.Dev(max(self.need, 16), "u8").upload(np.full(max(self.need, 16), 0xFF))
        self.S, self.F, self.X = PU.ints(self.starts), PU.ints(self.first), PU.ints(np.append(self.prefix, 0))
        return self

    def run(self, stream=None, lse=True):
        native()[0].api.sj_paged_attention_shared(
            stream, self.Q.at(self.off), self.ldq, self.K.at(self.off), self.V.at(self.off), self.ldkv, CODE[self.dtype],
            self.pages, self.P, self.T.p, self.width, len(self.tab), self.W.p if self.use_owners else None, self.Z.p,
            len(self.pos), self.S.p if self.use_starts else None, self.F.p, self.X.p, len(self.prefix), self.hq, self.hk,
            self.D, self.window, self.O.at(self.off), self.ldq, self.L.p if lse else None, self.ws.p, self.need)
        return self


GROUPS = [(40, [1, 2, 30]), (0, [5, 5]), (64, [1]), (130, [17, 64, 65, 3, 1, 1, 9]), (16, [1, 0]), (1, [4, 4])]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("hq,hk,D,P", [(6, 2, 64, 16), (4, 4, 64, 24), (16, 1, 64, 1), (40, 2, 64, 64), (3, 1, 16, 5),
                                       (8, 2, 32, 100), (8, 4, 80, 16), (14, 2, 96, 7), (8, 1, 128, 16), (32, 8, 128, 64),
                                       (5, 5, 256, 32), (18, 1, 256, 16), (2, 2, 8, 16), (3, 3, 7, 16), (4, 2, 20, 256),
                                       (68, 2, 16, 16)])
def test_shared(dtype, hq, hk, D, P):
    a = Shared(hq * D + P, dtype, hq, hk, D, P, GROUPS, alone=[0, 1, 77], pad=2).upload().run()
    a.check()
    first = a.O.host().copy(), a.L.host().copy()
    for b in (a.O, a.L):
        b.upload(np.full(b.n, 55.0))
    a.run()
    assert all((x == y.host()).all() for x, y in zip(first, (a.O, a.L)))  # every output again, the same bits


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("groups,hq,hk,D,P", [([(9000, [1] * 40)], 8, 2, 64, 16), ([(5000, [300] * 5), (20, [900] * 3)], 8, 8, 128, 64),
                                              ([(600, [2, 3])] * 60, 4, 2, 64, 24), ([(30, [2, 3])] * 256, 2, 2, 64, 8), ([(9, [1] * 8)] * 255, 2, 2, 32, 4), ([(70000, [5, 9])], 2, 1, 16, 256),
                                              ([(100, [4] * 300)], 16, 2, 64, 16), ([(2000, [1])], 6, 2, 64, 16),
                                              ([(17, [1, 1])] * 1000, 2, 1, 32, 16), ([(500, [3] * 3), (3, [6000])], 6, 2, 64, 16),
                                              ([(300, [20] * 70)], 8, 1, 256, 16), ([(256, [1] * 64)], 4, 4, 96, 32)])
def test_shared_long_and_many(dtype, groups, hq, hk, D, P):
    Shared(len(groups) + D, dtype, hq, hk, D, P, groups).upload().run().check()


@pytest.mark.parametrize("rows", [1, 3, 9])
@pytest.mark.parametrize("places", [509, 511, 512, 1021, 1023, 1024])
def test_shared_and_own_walks_of_just_so_many_workgroups(places, rows):
    """As many places of 128 keys as leave few workgroups, one or none for the rows' own keys: the parts of those that
    nobody took would be what lies in the workspace, NaN."""
    Shared(places + rows, "f32", 1, 1, 64, 256, [(128 * places, [1] * rows)]).upload().run().check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_shared_several_tokens_a_request(dtype):
    """Drafted tokens: those that do not see the whole prefix attend alone."""
    Shared(7, dtype, 6, 2, 64, 16, [(48, [4, 9, 2]), (90, [1, 3])], alone=[5, 64], per=4, pad=3).upload().run().check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window", [1, 20, 64, 100, 150, 5000])
def test_shared_windows(dtype, window):
    Shared(window, dtype, 6, 2, 64, 16, GROUPS + [(300, [1, 50])], alone=[400], window=window).upload().run().check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window", [100, 150])
def test_shared_windows_of_many_rows(dtype, window):
    """As many rows as the groups are walked for within such windows."""
    Shared(window, dtype, 16, 16, 128, 16, GROUPS * 4, alone=[400] * 4, window=window).upload().run().check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("hq,hk,D,P", [(6, 2, 64, 16), (14, 2, 96, 7), (5, 5, 256, 32), (3, 3, 7, 16), (40, 2, 64, 64)])
def test_shared_small_calls(dtype, hq, hk, D, P):
    """Every row by itself: the bits of sj_paged_attention."""
    a = Shared(hq * D + P, dtype, hq, hk, D, P, GROUPS, alone=[0, 1, 77], pad=2)
    a.wide = False
    a.upload().run().check()
    first = a.O.host().copy(), a.L.host().copy()
    for b in (a.O, a.L):
        b.upload(np.full(b.n, 55.0))
    Attend.run(a)
    assert all((x == y.host()).all() for x, y in zip(first, (a.O, a.L)))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D,ldkv,off", [(64, 136, 0), (64, 131, 3), (32, 72, 8), (128, 260, 1), (80, 161, 5)])
def test_shared_strides_and_alignment(dtype, D, ldkv, off):
    a = Shared(D + off, dtype, 4, 2, D, 16, [(33, [3, 70]), (16, [1, 2, 3])], owners=False, ldkv=max(ldkv, 2 * D), off=off)
    a.use_starts = False
    a.upload().run().check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_shared_reads_the_first_requests_pages(dtype):
    """In a large call the prefix is read through the first request's row: another row's entries there are not looked at."""
    a = Shared(3, dtype, 6, 2, 64, 16, [(64, [5, 6, 7])])
    a.upload()
    a.T.upload(np.where((np.arange(len(a.tab))[:, None] > 0) & (np.arange(a.width)[None, :] < 4), -1, a.tab))
    a.run().check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_shared_prefixes_that_are_none(dtype):
    """Prefixes below 0, past the table or past a row's position; groups past the requests, out of order, or whose rows
    are not where the starts say: every row attends alone."""
    for change in range(7):
        a = Shared(change, dtype, 6, 2, 64, 16, [(64, [5, 6]), (40, [7, 3, 1])], alone=[20])
        if change == 0:
            a.prefix[:] = [-5, 10 ** 6]
        if change == 1:
            a.prefix[:] = [2 ** 31 - 1, -2 ** 31]
        if change == 2:
            a.pos[0], a.pos[3] = 62, 38  # these two do not see all of it
        if change == 3:
            a.first = np.array([4, 2, 5])
        if change == 4:
            a.first = np.array([-3, 2, 900])
            a.prefix[1] = 0
        if change == 5:
            a.starts = np.array([0, 1, 4, 3, 4, 3, 6])
        if change == 6:
            a.starts = np.zeros(7, int)
        a.upload().run().check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 96])
def test_shared_bad_pages(dtype, D):
    """Pages that are none in the prefix and behind it; a prefix of nothing else; owners past the requests."""
    a = Shared(3, dtype, 6, 2, D, 16, [(80, [5, 20]), (48, [1, 2]), (32, [3, 3])])
    a.tab[0:2, 2], a.tab[1, 5] = -1, a.pages
    a.tab[2:4, :3] = [-1, a.pages, 2 ** 31 - 1]
    a.tab[2, 3] = -4  # no key at all
    a.own[5] = len(a.tab)
    want = a.upload().run().check()
    assert want[5] is None and (want[2][1] == -np.inf).all() and (want[2][0] == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_shared_scores_without_a_share_and_nan(dtype):
    """Keys of the prefix whose score is -inf, all of them for one group; a NaN in one reaches its group's rows alone."""
    a = Shared(4, dtype, 4, 2, 64, 16, [(70, [3, 4]), (50, [2, 2])])
    a.q[:, :, 0] = G.O.round_to(np.abs(a.q[:, :, 0]) + 0.5, dtype)
    for r, picked in ((0, np.arange(0, 70, 3)), (1, np.arange(64, 70, 2)), (2, np.arange(50)), (3, np.arange(48, 50))):
        a.k[a.tab[r][picked // 16] * 16 + picked % 16, :, 0] = -np.inf
    # positions 64 .. 69 lie in a page of each request's own: the same keys there
    for j in range(64, 70):
        a.k[a.tab[1][4] * 16 + j % 16] = a.k[a.tab[0][4] * 16 + j % 16]
    a.upload().run().check()
    b = Shared(6, dtype, 4, 2, 64, 16, [(64, [3, 4]), (64, [2, 2])])
    b.v[b.tab[0][1] * 16 + 3, 0, 5] = np.nan
    b.k[b.tab[2][2] * 16 + 2, 1, 0] = np.nan
    b.upload().run()
    o = b.O.host()[:4 * 256].reshape(4, 2, 2, 64)
    assert np.isnan(o[:2, 0, :, 5]).all() and np.isfinite(o[:2, 1]).all() and np.isfinite(o[:2, 0, :, 6:]).all()
    assert np.isnan(o[2:, 1]).all() and np.isfinite(o[2:, 0]).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_shared_in_place_and_without_lse(dtype):
    a = Shared(5, dtype, 6, 2, 64, 16, [(200, [1, 2, 3]), (40, [1])], alone=[9])
    a.upload()
    keep = a.Q.host().copy()
    a.O = a.Q
    a.run(lse=False)
    got = a.Q.host()
    b = Shared(5, dtype, 6, 2, 64, 16, [(200, [1, 2, 3]), (40, [1])], alone=[9]).upload().run()
    n = len(a.pos) * a.ldq
    np.testing.assert_array_equal(got[:n], b.O.host()[:n])
    assert (keep == b.Q.host()).all()


def test_shared_no_groups_and_more_than_are_walked_together():
    """No group at all; more than 2048 rows and more than 256 groups attend alone."""
    Shared(1, "bf16", 6, 2, 64, 16, [], alone=[5, 300]).upload().run().check()
    Shared(2, "bf16", 2, 1, 32, 16, [(32, [1] * 2100)]).upload().run().check()
    Shared(3, "bf16", 2, 1, 32, 16, [(16, [1])] * 1100).upload().run().check()


def test_shared_two_streams_and_two_graphs_of_one_workspace():
    a = Shared(11, "bf16", 6, 2, 64, 16, [(3000, [5, 70, 1]), (64, [9] * 20)]).upload()
    b = Shared(12, "bf16", 8, 4, 128, 16, [(900, [3, 10])] * 3, alone=[700]).upload()
    for one in (False, True):
        if one:
            need = max(a.need, b.need)
            a.ws = b.ws = G.Dev(need, "u8").upload(np.full(need, 0xFF))
        graphs = [PU.Graph(a.run), PU.Graph(b.run)]
        for _ in range(3):
            for x in (a, b):
                x.O.upload(np.full(x.O.n, 55.0))
                x.L.upload(np.full(x.L.n, 55.0))
            for g in graphs:
                if one:
                    g.replay()
                else:
                    g.do(g.hip.hipGraphLaunch(g.exe, g.stream))
            G.sync()
            a.check()
            b.check()
        for g in graphs:
            g.close()
