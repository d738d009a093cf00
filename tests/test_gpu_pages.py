"""The pages' fork, compaction and copy against their plain forms."""
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


def state(rng, groups, beams, P, hi, spare, lo=0, kept=True):
    """Rows whose groups share their first pages, as forks leave them: (lengths, table, shared, free list, position, pages)."""
    lengths = np.repeat(rng.integers(lo, hi + 1, groups), beams)
    width = max(-(-hi // P), 1) + 1
    table, made = np.full((groups * beams, width), -1), 0
    for r, n in enumerate(lengths):
        full, cols, same = n // P, -(-n // P), 0
        if r % beams:
            same = int(rng.integers(0, full + 1))
            table[r, :same] = table[r - 1 - int(rng.integers(0, r % beams)), :same]
        table[r, same:cols] = np.arange(made, made + cols - same)
        made += cols - same
    pages = max(made + spare, 1)
    names = rng.permutation(pages)
    held = table >= 0
    table[held] = names[table[held]]
    shared = np.maximum(np.bincount(table[held].astype(int), minlength=pages) - 1, 0)
    if kept and groups > 2:
        shared[table[0][:lengths[0] // P]] += 1
    free = np.concatenate([np.full(made, -1), names[made:]])
    return lengths, table, shared, free, made, pages


class Fork:
    def __init__(self, parents, lengths, table, shared, free, head, pages, P):
        self.args = (np.asarray(parents), np.asarray(table), np.asarray(lengths), P, pages, np.asarray(shared),
                     np.asarray(free), head)
        self.R, self.before, self.width = len(parents), len(lengths), table.shape[1]
        self.inputs = [PU.ints(np.append(a, 9)) for a in (parents, table, lengths, shared, free)] + [PU.ints([head])]
        self.outs = dict(table=PU.ints(np.full(self.R * self.width + 1, 55)), lengths=PU.ints(np.full(self.R + 1, 55)),
                         shared=PU.ints(np.full(pages + 1, 55)), free=PU.ints(np.full(len(free) + 1, 55)),
                         copies=PU.ints(np.full(3 * self.R + 1, 55)))
        self.summary = PU.ints([55] * 5)
        need = self.need = native()[1].sj_paged_fork_workspace_bytes(self.R, self.before, pages)
        self.ws = G.Dev(need, "u8").upload(np.full(need, 0xFF))

    def run(self, stream=None):
        p, t, n, s, f, h = (b.p for b in self.inputs)
        o = self.outs
        native()[0].api.sj_paged_fork(stream, p, self.R, t, self.width, n, self.before, self.args[3], self.args[4], s, f,
                                      len(self.args[6]), h, o["table"].p, o["lengths"].p, o["shared"].p, o["free"].p,
                                      o["copies"].p, self.summary.p, self.ws.p, self.need)
        return self

    def check(self):
        want = BU.fork(*self.args)
        for key, b in self.outs.items():
            h = b.host()
            np.testing.assert_array_equal(h[:-1], np.asarray(want[key]).ravel(), key)
            assert h[-1] == 55
        np.testing.assert_array_equal(self.summary.host(), [want["taken"], want["head"], want["status"], want["back"], 55])
        return want


@pytest.mark.parametrize("groups,beams,P,hi,spare", [(0, 1, 16, 5, 3), (1, 1, 16, 0, 4), (1, 1, 16, 40, 4), (3, 4, 8, 100, 20),
                                                     (16, 4, 16, 900, 200), (5, 3, 1, 60, 50), (40, 5, 24, 3000, 3000),
                                                     (300, 8, 16, 200, 20000), (2000, 5, 16, 64, 12000), (2, 2, 1000, 5000, 8),
                                                     (3, 64, 7, 400, 40000)])
def test_fork(groups, beams, P, hi, spare):
    rng = np.random.default_rng(groups + P)
    lengths, table, shared, free, head, pages = state(rng, groups, beams, P, hi, spare)
    parents = np.arange(groups)[:, None] * beams + rng.integers(0, beams, (groups, beams))
    parents[rng.random(groups) < 0.2] = -1
    f = Fork(parents.ravel(), lengths, table, shared, free, head, pages, P).run()
    f.check()
    f.run()  # the same state again: the same step
    assert f.check()["status"] == 0


@pytest.mark.parametrize("R,before", [(7, 12), (30, 12), (0, 12), (12, 0)])
def test_fork_to_another_number_of_requests(R, before):
    rng = np.random.default_rng(R)
    lengths, table, shared, free, head, pages = state(rng, before // 4, 4, 8, 90, 60)
    parents = rng.integers(-1, before, R) if before else np.full(R, -1)
    if before == 0:
        table, lengths = np.zeros((0, 4), int), np.zeros(0, int)
    Fork(parents, lengths, table, shared, free, head, pages, 8).run().check()


def test_fork_frees_requests_in_place():
    """Requests that stay where they are cost no page; those that end give theirs back, shared ones with the last."""
    rng = np.random.default_rng(2)
    lengths, table, shared, free, head, pages = state(rng, 4, 4, 8, 100, 10, kept=False)
    parents = np.arange(16)
    parents[[1, 4, 5, 6, 7]] = -1
    want = Fork(parents, lengths, table, shared, free, head, pages, 8).run().check()
    assert want["taken"] == 0 and want["back"] >= -(-lengths[4] // 8)


def test_fork_of_a_page_that_others_hold():
    """A last page that is not full and that somebody else holds: every child gets a copy."""
    table, lengths, shared = np.array([[3, 1, -1], [5, 2, -1]]), np.array([11, 9]), np.zeros(8, int)
    shared[1], shared[3] = 1, 1
    want = Fork([0, 0, 1], lengths, table, shared, [-1, -1, -1, -1, 0, 4, 6, 7], 4, 8, 8).run().check()
    assert want["taken"] == 2 and want["copies"].tolist() == [[1, 0, 3], [1, 4, 3], [-1, -1, 0]] and want["back"] == 0


@pytest.mark.parametrize("status,change", [(1, "short"), (1, "head"), (1, "far"), (8, "parent"), (8, "negative"), (8, "long"),
                                           (9, "both")])
def test_void_forks(status, change):
    """A step that cannot be leaves the pages, the list and its position; all requests after it are empty."""
    rng = np.random.default_rng(3)
    lengths, table, shared, free, head, pages = state(rng, 3, 4, 8, 90, 12, lo=10)
    lengths = lengths // 8 * 8 + 3
    table = np.where(table < 0, pages, table)
    parents = np.repeat(np.arange(3) * 4, 4)
    if change == "short":
        free = free[:head + 2]
    if change in ("head", "both"):
        head = -1
    if change == "far":
        head = len(free) + 1
    if change in ("parent", "both"):
        parents[5] = 12
    if change == "negative":
        lengths[2] = -1
    if change == "long":
        lengths[3] = 8 * table.shape[1] + 1
    if change == "short":
        table = np.where(table == pages, 0, table)
    want = Fork(parents, lengths, table, shared, free, head, pages, 8).run().check()
    assert want["status"] == status and (want["lengths"] == 0).all()


@pytest.mark.parametrize("groups,beams,P,hi,spare", [(300, 4, 16, 60, 900), (256, 4, 16, 60, 900), (64, 3, 16, 60, 900),
                                                     (193, 1, 16, 60, 900), (60, 8, 4, 300, 0), (1, 1, 4, 9, 16000),
                                                     (1, 1, 4, 9, 17000), (7, 3, 16, 40000, 99), (7, 3, 16, 25000, 99)])
def test_fork_in_one_launch_and_in_several(groups, beams, P, hi, spare):
    """Sizes around those that one launch takes: requests, pages, entries of the tables."""
    rng = np.random.default_rng(groups)
    lengths, table, shared, free, head, pages = state(rng, groups, beams, P, hi, spare + groups * beams)
    R = groups * beams
    parents = rng.integers(-1, R, R)
    assert Fork(parents, lengths, table, shared, free, head, pages, P).run().check()["status"] == 0
    keep = np.where(rng.random(R) < 0.5, np.arange(R), -1)  # some end, the others stay
    assert Fork(keep, lengths, table, shared, free, head, pages, P).run().check()["taken"] == 0
    # the list begins behind a few places: some pages that come back find none
    want = Fork(keep, lengths, table, shared, free[max(head - 5, 0):], min(head, 5), pages, P).run().check()
    assert want["status"] == (BU.LIST_FULL if want["head"] == 0 and (want["shared"] < 0).any() else 0)
    parents[R // 2] = R
    assert Fork(parents, lengths, table, shared, free, head, pages, P).run().check()["status"] == 8
    assert Fork(np.zeros(R, int), lengths, table, shared, free, len(free) + 1, pages, P).run().check()["status"] == 1


def test_fork_without_room_on_the_list():
    """Pages that the list has no place for keep their mark, and a later step gives them back."""
    rng = np.random.default_rng(4)
    lengths, table, shared, free, head, pages = state(rng, 2, 2, 8, 100, 6, lo=50, kept=False)
    short = free[head - 3:]  # three places before its position
    want = Fork(np.full(4, -1), lengths, table, shared, short, 3, pages, 8).run().check()
    assert want["status"] == BU.LIST_FULL and want["back"] == 3 and (want["shared"] == -1).sum() == head - 3
    more = np.concatenate([np.full(head, -1), want["free"]])
    again = Fork(np.full(4, -1), np.zeros(4, int), table, want["shared"], more, head, pages, 8).run().check()
    assert again["status"] == 0 and again["back"] == head - 3 and (again["shared"] == 0).all()


def test_fork_with_bad_pages():
    """Entries that are no page are handed on; no holder is counted for them."""
    rng = np.random.default_rng(6)
    lengths, table, shared, free, head, pages = state(rng, 3, 2, 8, 70, 9, lo=30)
    table[0, 0], table[1, 1], table[2, lengths[2] // 8], table[3, 0] = pages, -7, 2 ** 31 - 1, -2 ** 31
    free[head] = -3
    Fork([0, 0, 2, 2, 5, -1], lengths, table, shared, free, head, pages, 8).run().check()


def test_fork_replays_and_two_streams():
    rng = np.random.default_rng(7)
    forks = []
    for seed in range(2):
        st = state(rng, 20, 4, 16, 600, 400)
        parents = np.arange(20)[:, None] * 4 + rng.integers(0, 4, (20, 4))
        forks.append(Fork(parents.ravel(), *st[:3], st[3], st[4], st[5], 16))
    graphs = [PU.Graph(f.run) for f in forks]
    for _ in range(3):
        for f in forks:
            for b in f.outs.values():
                b.upload(np.full(b.n, 55))
        for g in graphs:
            g.do(g.hip.hipGraphLaunch(g.exe, g.stream))
        G.sync()
        for f in forks:
            f.check()
    for g in graphs:
        g.close()


class Compact:
    def __init__(self, lengths, table, shared, free, head, pages, P, after, capacity=None):
        capacity = pages - after if capacity is None else capacity
        self.args = (np.asarray(table), np.asarray(lengths), P, pages, after, np.asarray(shared), np.asarray(free), head,
                     capacity)
        self.R, self.width = table.shape
        self.inputs = [PU.ints(np.append(a, 9)) for a in (table, lengths, shared, free)] + [PU.ints([head])]
        self.outs = dict(table=PU.ints(np.full(table.size + 1, 55)), shared=PU.ints(np.full(pages + 1, 55)),
                         free=PU.ints(np.full(len(free) + 1, 55)), copies=PU.ints(np.full(3 * capacity + 1, 55)))
        self.summary = PU.ints([55] * 5)
        need = self.need = native()[1].sj_paged_compact_workspace_bytes(pages, len(free))
        self.ws = G.Dev(need, "u8").upload(np.full(need, 0xFF))

    def run(self, stream=None):
        t, n, s, f, h = (b.p for b in self.inputs)
        _, _, P, pages, after, _, free, _, capacity = self.args
        o = self.outs
        native()[0].api.sj_paged_compact(stream, t, self.width, n, self.R, P, pages, after, s, f, len(free), h, o["table"].p,
                                         o["shared"].p, o["free"].p, o["copies"].p, capacity, self.summary.p, self.ws.p,
                                         self.need)
        return self

    def check(self):
        want = BU.compact(*self.args)
        for key, b in self.outs.items():
            h = b.host()
            np.testing.assert_array_equal(h[:-1], np.asarray(want[key]).ravel(), key)
            assert h[-1] == 55
        np.testing.assert_array_equal(self.summary.host(), [want["moves"], want["head"], want["status"], want["left"], 55])
        return want


@pytest.mark.parametrize("groups,beams,P,hi,spare", [(1, 1, 16, 0, 4), (1, 1, 16, 40, 4), (3, 4, 8, 100, 40), (16, 4, 16, 900, 999),
                                                     (40, 5, 24, 3000, 9000), (100, 8, 16, 200, 40000), (5, 2, 1, 300, 77)])
@pytest.mark.parametrize("part", [0.0, 0.5, 1.0])
def test_compact(groups, beams, P, hi, spare, part):
    """To the least number of pages that hold what is used, half way, and all."""
    rng = np.random.default_rng(groups + P)
    lengths, table, shared, free, head, pages = state(rng, groups, beams, P, hi, spare)
    used = pages - (len(free) - head)
    c = Compact(lengths, table, shared, free, head, pages, P, int(used + part * (pages - used))).run()
    c.check()
    c.run()
    want = c.check()
    assert want["status"] == 0 and (part < 1 or want["moves"] == 0)


@pytest.mark.parametrize("status,change", [(1, "small"), (1, "head"), (1, "far"), (4, "capacity"), (5, "both")])
def test_void_compactions(status, change):
    rng = np.random.default_rng(5)
    lengths, table, shared, free, head, pages = state(rng, 6, 2, 8, 200, 100)
    used = pages - (len(free) - head)
    after = used - 1 if change in ("small", "both") else used + 20
    head = -1 if change == "head" else len(free) + 1 if change == "far" else head
    if change in ("head", "far"):
        free = np.concatenate([free[free >= 0], free[free < 0]]) if change == "head" else free
    c = Compact(lengths, table, shared, free, head, pages, 8, after, 2 if change in ("capacity", "both") else None).run()
    assert c.check()["status"] == status


@pytest.mark.parametrize("status,change", [(1, "small"), (1, "far"), (4, "capacity"), (5, "both")])
def test_void_compactions_of_many_workgroups(status, change):
    rng = np.random.default_rng(15)
    lengths, table, shared, free, head, pages = state(rng, 60, 2, 8, 2000, 30000)
    used = pages - (len(free) - head)
    after = used - 1 if change in ("small", "both") else used + 20
    head = len(free) + 1 if change == "far" else head
    c = Compact(lengths, table, shared, free, head, pages, 8, after, 2 if change in ("capacity", "both") else None).run()
    assert c.check()["status"] == status


@pytest.mark.parametrize("pages", [8192, 8193, 16384, 16385, 5_000_003])
def test_pools_of_one_workgroup_and_of_rounds(pages):
    """Pages of which one workgroup holds all, one more, and so many that a workgroup takes several rounds."""
    rng = np.random.default_rng(pages)
    R, P, cols = 40, 4, 60
    names = rng.permutation(pages)
    table, lengths = names[:R * cols].reshape(R, cols), np.full(R, P * cols)
    free = np.concatenate([np.full(R * cols, -1), names[R * cols:]])
    shared = np.zeros(pages, int)
    want = Fork(np.arange(0, R, 2), lengths, table, shared, free, R * cols, pages, P).run().check()
    assert want["status"] == 0 and want["back"] == R * cols // 2
    want = Compact(lengths, table, shared, free, R * cols, pages, P, pages // 3).run().check()
    assert want["status"] == 0 and want["moves"] > R * cols // 2
    want = Compact(lengths, table, shared, free, R * cols, pages, P, 100).run().check()
    assert want["status"] == 1


def test_compact_replays_of_many_workgroups():
    rng = np.random.default_rng(19)
    st = state(rng, 30, 4, 16, 900, 40000)
    c = Compact(st[0], st[1], st[2], st[3], st[4], st[5], 16, st[5] - 30000)
    g = PU.Graph(c.run)
    for _ in range(3):
        for b in c.outs.values():
            b.upload(np.full(b.n, 55))
        g.replay()
        c.check()
    g.close()


def test_compact_empty_and_bad_entries():
    rng = np.random.default_rng(8)
    lengths, table, shared, free, head, pages = state(rng, 4, 2, 8, 100, 60, lo=20)
    table[0, 0], table[1, 1], lengths[3], lengths[4] = -5, pages, -3, 8 * table.shape[1] + 50
    free[head + 1] = -9
    free[head + 2] = pages + 4
    used = pages - (len(free) - head)
    Compact(lengths, table, shared, free, head, pages, 8, used + 12).run().check()
    Compact(np.zeros(0, int), np.zeros((0, 3), int), shared, free, head, pages, 8, used + 12).run().check()


def test_compact_replays():
    rng = np.random.default_rng(9)
    st = state(rng, 30, 4, 16, 900, 5000)
    c = Compact(st[0], st[1], st[2], st[3], st[4], st[5], 16, st[5] - 3000)
    g = PU.Graph(c.run)
    for _ in range(3):
        for b in c.outs.values():
            b.upload(np.full(b.n, 55))
        g.replay()
        c.check()
    g.close()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("layers,P,width,ld,off,count", [(1, 16, 128, 128, 0, 7), (3, 8, 64, 72, 0, 9), (2, 16, 20, 21, 1, 5),
                                                         (4, 1, 7, 7, 3, 12), (2, 100, 256, 259, 5, 4), (1, 3, 1, 1, 0, 6),
                                                         (12, 16, 512, 512, 8, 40)])
def test_copy(dtype, layers, P, width, ld, off, count):
    rng = np.random.default_rng(P + width)
    pages = 2 * count + 3
    order = rng.permutation(pages)
    copies = np.stack([order[:count], order[count:2 * count], rng.integers(0, P + 3, count)], 1)
    copies[rng.random(count) < 0.2] = [-1, -1, 0]
    copies[-1, 1] = pages  # no page
    copies[0, 2] = P
    stride = pages * P * ld + 5
    both = []
    for seed in range(2):
        x = G.rnd((layers * stride + off + 1,), dtype, rng)
        both.append((x, G.dev(x, dtype)))
    C = PU.ints(copies)
    native()[0].api.sj_paged_copy(None, both[0][1].at(off), both[1][1].at(off), ld, CODE[dtype], layers, stride, pages, P,
                                  width, C.p, count)
    for x, d in both:
        want = x.copy()
        for l in range(layers):
            at = off + l * stride
            part = want[at:at + pages * P * ld].reshape(1, pages * P, ld)
            BU.copy(part, copies, P, width)
        np.testing.assert_array_equal(d.host(), want)  # nothing besides


def test_copy_of_pages_past_32_bits():
    """A cache of more than 2^32 bytes: pages at its far end."""
    P, width, pages = 4096, 512, 1100
    rng = np.random.default_rng(1)
    N, lib = native()
    K = G.Dev(pages * P * width, "bf16")
    row = G.rnd((3, width), "bf16", rng)
    src = (pages - 2) * P
    raw = (row.astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)
    N.api.sj_upload(K.at(src * width), ctypes.c_void_p(raw.ctypes.data), raw.nbytes)
    C = PU.ints([[pages - 2, pages - 1, 3]])
    N.api.sj_paged_copy(None, K.p, K.p, width, 4, 1, 0, pages, P, width, C.p, 1)
    back = np.empty_like(raw)
    N.api.sj_download(ctypes.c_void_p(back.ctypes.data), K.at((pages - 1) * P * width), raw.nbytes)
    np.testing.assert_array_equal(back, raw)
