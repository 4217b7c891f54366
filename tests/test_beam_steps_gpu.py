"""kd_beam_select where a block goes through many steps of 4096 logits of a row (many rows, large vocabularies): the bound that rises from
step to step, equal logits of different steps, sums that are rescaled.

How far values may be off, from the operations on a row's sum, all of them on positive terms, so that relative errors add up.  u = 2^-24 is a
rounding.  An exponential 4 u; its argument's two roundings, u each of its size x, which the term's weight brings down to a mean of at most log V.  A
step of a thread: 8 additions, and a factor (4 u and its product's u; its arguments add up to no more than the terms' own: log V again).  Then a factor
and 6 additions for a warp, a factor and 5 for the block, for every 32 segments two factors and an addition, a factor and 5 additions, and the
logarithm (2 u of its size, up to log V).  A value is rounded to fp32 once."""
import math

import numpy as np
import pytest

from kandle_b200.core import Tensor
from kandle_b200.model_utils import beam_select
from tests.paged_cases import beam_answer

pytestmark = pytest.mark.gpu

STEP, BLOCKS = 4096, 4 * 148


def plan(B, K, V):
    """(segments of a row, steps of a segment)"""
    steps = math.ceil(V / STEP)
    segs = min(max(BLOCKS // (B * K), 1), steps)
    each = math.ceil(steps / segs)
    return math.ceil(V / (each * STEP)), each


def check(logits, scores, eos):
    B, K, V = logits.shape
    segs, steps = plan(B, K, V)
    assert steps > 1
    want = beam_answer(logits, scores, eos)
    s, p, t, e = (x.dataAsync() for x in beam_select(Tensor(logits), Tensor(scores), eos))
    assert np.array_equal(p, want[1]) and np.array_equal(t, want[2])
    off = (4 + 2 * math.log(V) + steps * (8 + 5) + 2 * math.log(V) + (5 + 6) + (5 + 5) + math.ceil(segs / 32) * (5 + 5 + 1) + (5 + 5) + 2 * math.log(V)) * 2.0 ** -24
    for a, b in ((s, want[0]), (e, want[3])):
        assert np.array_equal(np.isfinite(a), np.isfinite(b)) and not np.isnan(a).any()
        f = np.isfinite(b)
        assert (np.abs(a[f] - b[f]) <= off + np.abs(b[f]) * 2.0 ** -24).all()


def draw(B, K, V, seed, std=2.5):
    rng = np.random.default_rng(seed)
    return (rng.standard_normal((B, K, V), dtype=np.float32) * np.float32(std)), (-20 * rng.random((B, K))).astype(np.float32)


@pytest.mark.parametrize("B,K,V", [(32, 4, 151936), (20, 32, 20001), (128, 8, 9001), (150, 4, 20001), (60, 5, 40000), (600, 1, 12290)])
def test_the_best_candidates_of_long_segments(backend, B, K, V):
    logits, scores = draw(B, K, V, V)
    late = V - 5 if V % STEP > 5 else V // 2
    logits[:, ::2, late] += 12
    check(logits, scores, late)
    if V < 100000:
        check(logits, scores, -1)


@pytest.mark.parametrize("levels", [1, 2, 30, 4000])
@pytest.mark.parametrize("B,K", [(150, 4), (40, 16)])
def test_equal_logits_of_different_steps(backend, B, K, levels):
    """Few levels overflow the lists; many leave some equal ones at the bound, the lower token of which comes first."""
    V = 20001
    rng = np.random.default_rng(levels)
    logits = np.empty((B, K, V), np.float32)
    logits[:] = rng.integers(0, levels, (B, 1, V)) * np.float32(8 / levels)
    logits[:, :, ::7] = -0.0
    check(logits, np.zeros((B, K), np.float32), 17000)


@pytest.mark.parametrize("B,K,V", [(150, 4, 20001), (40, 16, 20001)])
def test_logits_that_rise_and_fall_along_a_row(backend, B, K, V):
    """The largest come in the last step, or in the first; sums are rescaled in every step."""
    logits, scores = draw(B, K, V, 3, 0.5)
    ramp = np.linspace(0, 60, V, dtype=np.float32)
    check(logits + ramp, scores, V - 2)
    check(logits - ramp, scores, 3)
    check(logits + np.abs(ramp - 30), scores, -1)


@pytest.mark.parametrize("low", [-np.inf, float(np.finfo(np.float32).min)])
@pytest.mark.parametrize("B,K,V", [(150, 4, 20001), (40, 16, 20001)])
def test_rows_of_which_most_is_masked(backend, B, K, V, low):
    """A few tokens may come: everywhere, in one step only, fewer than beams, and none."""
    logits, scores = draw(B, K, V, 4)
    rng = np.random.default_rng(5)
    keep = rng.random((B, K, V)) < 0.01
    keep[1::6, :, :17000] = False
    keep[2::6, :, 4096:] = False
    keep[3::6] = False
    keep[3::6, :, [9000, 9001, 19000]] = True
    keep[4::6, 1:] = False
    keep[5::6] = rng.random((len(keep[5::6]), K, V)) < 0.0002
    x = np.where(keep, logits, np.float32(low))
    check(x, scores, 19000)
    check(x, scores, -1)


def test_rows_without_a_finite_sum(backend):
    logits, scores = draw(150, 4, 20001, 6)
    logits[3, 1, 15000], logits[7, 2, 20000], logits[9, 0, 5000] = np.nan, np.inf, -np.inf
    logits[11, 3] = -np.inf
    scores[20, 1], scores[21, 0] = -np.inf, np.nan
    check(logits, scores, 15001)
