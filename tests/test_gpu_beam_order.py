"""The order of candidates whose totals are the same 64 bits though their logits
are not: the lowest beam first, and of a beam's own tokens the larger logit."""
import numpy as np
import pytest

from tests import gpu_util as G
from tests import paged_util as PU
from tests.test_gpu_beam import Select

pytestmark = pytest.mark.gpu


def select(x, scores, beams, keep, ended, end):
    """Candidates in order by rank (length_power 0: the total), beam, logit, token: (parents, tokens, totals)."""
    out = []
    for g in range(len(x) // beams):
        parts = []
        for b in range(beams):
            r = g * beams + b
            if ended[r]:
                parts.append((np.array([float(scores[r])]), [b], [0.0], [end], [r]))
                continue
            m = x[r].max()
            total = float(scores[r]) + (x[r] - (m + np.log(np.exp(x[r] - m).sum())))
            v = np.arange(x.shape[1])
            parts.append((total, b + 0 * v, x[r], v, r + 0 * v))
        total, beam, logit, token, row = (np.concatenate([p[i] for p in parts]) for i in range(5))
        first = np.lexsort((token, -logit, beam, -total))[:keep]
        out.append((row[first], token[first], total[first]))
    return [np.concatenate([o[i] for o in out]) for i in range(3)]


def check(x, scores, beams, keep, dtype, ended=None, end=-1):
    x = G.O.round_to(x, dtype)
    if dtype == "f32":
        x = x.astype(np.float32).astype(np.float64)
    scores = np.asarray(scores, np.float32)
    s = Select(x, scores, beams, keep, dtype, lengths=np.full(len(x), 3), ended=ended, end=end)
    s.run()
    parents, tokens, totals = select(x, scores, beams, keep, np.zeros(len(x), int) if ended is None else ended, end)
    assert len(parents) == len(x) // beams * keep  # every place has a candidate
    np.testing.assert_array_equal(s.ints[0].host()[:-1], parents)
    np.testing.assert_array_equal(s.ints[1].host()[:-1], tokens)
    got = s.out.host()[:-1]
    # totals of 64 bits, the sum's powers to 7.8e-13, rounded once to fp32
    assert (np.abs(got - totals) <= np.abs(totals) * 2.0 ** -24 * 1.001 + 1e-12).all()
    return totals.reshape(-1, keep)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V,beams,keep", [(40, 4, 64), (257, 4, 4), (257, 2, 64), (900, 3, 8), (5000, 4, 16), (40000, 8, 64),
                                          (200000, 8, 40)])
def test_scores_that_leave_nothing_of_the_logits(dtype, V, beams, keep):
    """At -1e30 every total of a prompt is the score; more of the same rank than a workgroup's LDS holds among them."""
    rng = np.random.default_rng(V + keep)
    totals = check(rng.normal(0, 2, (3 * beams, V)), np.full(3 * beams, -1e30), beams, keep, dtype)
    assert (totals == totals[:, :1]).all()


@pytest.mark.parametrize("V,keep", [(40, 33), (257, 64), (900, 64), (5000, 64), (40000, 64), (200000, 32)])
def test_scores_that_round_the_logits(V, keep):
    """At -1e9 (a beam that a program has put aside) a total is good to 1.2e-7: logits of less difference share it."""
    rng = np.random.default_rng(V)
    x = rng.normal(0, 2, (6, V))
    top = 0.5 + rng.permutation(48) * 2.0 ** -24  # the row's largest, next to each other in fp32
    for r in range(6):
        x[r] = np.minimum(x[r], 0.4)
        at = rng.choice(V, min(48, V // 2), replace=False)
        x[r, at] = top[:len(at)]
    totals = check(x, np.full(6, -1e9), 1, keep, "f32")
    assert (np.diff(totals, axis=1) == 0).sum() > 50


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V,beams,keep", [(257, 4, 8), (900, 2, 40), (5000, 3, 64), (20000, 4, 7)])
def test_logits_next_to_nothing(dtype, V, beams, keep):
    """Logits of some 1e-20: their order is theirs, though no total sees them."""
    rng = np.random.default_rng(V)
    check(rng.normal(0, 1e-20, (4 * beams, V)), np.full(4 * beams, -3.0), beams, keep, dtype)


@pytest.mark.parametrize("V", [257, 5000])
def test_ended_beams_among_equal_totals(V):
    """An ended beam's one candidate takes the place of its beam."""
    rng = np.random.default_rng(V)
    ended = np.tile([0, 1, 0, 1], 3)
    check(rng.normal(0, 2, (12, V)), np.full(12, -1e30), 4, 64, "f32", ended=ended, end=V - 1)
    check(rng.normal(0, 2, (12, 5)), np.full(12, -1e30), 4, 12, "f32", ended=ended, end=2)


def test_replays_among_equal_totals():
    rng = np.random.default_rng(7)
    x = G.O.round_to(rng.normal(0, 2, (8, 9000)), "f32").astype(np.float32).astype(np.float64)
    scores = np.full(8, -1e30, np.float32)
    s = Select(x, scores, 4, 64, "f32")
    want = select(x, scores, 4, 64, np.zeros(8, int), -1)
    g = PU.Graph(s.run)
    for _ in range(3):
        s.clear()
        g.replay()
        for b, w in zip(s.ints, want[:2]):
            np.testing.assert_array_equal(b.host()[:-1], w)
    g.close()
