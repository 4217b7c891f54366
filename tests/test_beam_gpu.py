"""GPU checks of a step of beam search (kd_beam_select) against its definition in float64.

Which candidates are chosen has to agree exactly.  Their values: the sum of a row's exponentials is off by the rounding of each exponential
(2^-23), of its argument (2^-24 of its size, which e^-size weighs down to below log V), and of the sums (at most 32 in a thread and 12 beyond), all
relative, so lse by at most 60 * 2^-24; the value is rounded to fp32 once."""
import numpy as np
import pytest

from kandle_b200 import core, lib
from kandle_b200.core import Tensor
from kandle_b200.model_utils import beam_select
from tests.paged_cases import beam_answer

pytestmark = pytest.mark.gpu


def check(logits, scores, eos, got):
    want = beam_answer(logits, scores, eos)
    s, p, t, e = (x.dataAsync() for x in got)
    assert np.array_equal(p, want[1]) and np.array_equal(t, want[2])
    for a, b in ((s, want[0]), (e, want[3])):
        assert np.array_equal(np.isfinite(a), np.isfinite(b)) and not np.isnan(a).any()
        f = np.isfinite(b)
        assert (np.abs(a[f] - b[f]) <= 60 * 2.0 ** -24 + np.abs(b[f]) * 2.0 ** -24).all()


def draw(B, K, V, seed, std=2.5):
    rng = np.random.default_rng(seed)
    return (rng.standard_normal((B, K, V)) * std).astype(np.float32), (-20 * rng.random((B, K))).astype(np.float32)


@pytest.mark.parametrize("B,K,V", [(1, 1, 2), (1, 4, 3), (2, 3, 7), (1, 4, 151936), (3, 2, 51865), (2, 5, 4096), (1, 5, 4097), (4, 1, 1000), (1, 32, 9000), (2, 16, 20001), (7, 8, 333),
                                   (1, 32, 33), (1, 2, 8191)])
def test_the_best_candidates(backend, B, K, V):
    logits, scores = draw(B, K, V, B + K + V)
    for eos in (-1, 0, V - 1, V // 2):
        x = logits.copy()
        if eos >= 0:
            x[:, ::2, eos] += 12
        check(x, scores, eos, beam_select(Tensor(x), Tensor(scores), eos))


def test_the_first_step_has_one_live_beam(backend):
    logits, scores = draw(2, 4, 5000, 1)
    scores[:] = -np.inf
    scores[:, 0] = 0
    check(logits, scores, 3, beam_select(Tensor(logits), Tensor(scores), 3))
    scores[1] = -np.inf                                   # a request that is done
    check(logits, scores, 3, beam_select(Tensor(logits), Tensor(scores), 3))


@pytest.mark.parametrize("K", [1, 4, 32])
@pytest.mark.parametrize("levels", [1, 2, 40])
def test_equal_logits_go_by_beam_and_token(backend, K, levels):
    rng = np.random.default_rng(levels)
    logits = np.repeat(rng.integers(0, levels, (1, 1, 9001)).astype(np.float32), K, 1)
    logits[0, 0, 5] = -0.0 if levels > 1 else 0.0
    scores = np.zeros((1, K), np.float32)
    check(logits, scores, 2, beam_select(Tensor(logits), Tensor(scores), 2))


def test_masked_logits(backend):
    """Tokens that may not come are -inf, or the type's lowest value; a row may be left with fewer tokens than beams, or none."""
    logits, scores = draw(3, 4, 6000, 5)
    keep = np.random.default_rng(6).random(logits.shape) < 0.01
    for low in (-np.inf, np.finfo(np.float32).min):
        x = np.where(keep, logits, np.float32(low))
        x[1] = low
        x[1, :, 77] = logits[1, :, 77]
        if low == -np.inf:
            x[2, 0] = low
            x[2, 1:] = low
            x[2, 2, 4000:4002] = 1
        check(x, scores, 77, beam_select(Tensor(x), Tensor(scores), 77))
        check(x, scores, -1, beam_select(Tensor(x), Tensor(scores)))


def test_rows_without_a_finite_sum_are_worth_nothing(backend):
    logits, scores = draw(2, 4, 3000, 7)
    logits[0, 1, 50], logits[0, 2, 2999], logits[1, 0, 0], logits[1, 3, 7] = np.nan, np.inf, np.nan, np.nan
    logits[1, 1] = -np.inf
    check(logits, scores, 9, beam_select(Tensor(logits), Tensor(scores), 9))
    scores[0, 0], scores[1, 2] = np.nan, np.inf
    check(logits, scores, 0, beam_select(Tensor(logits), Tensor(scores), 0))


def test_scores_in_place_rows_as_a_view_and_without_ends(backend):
    B, K, V = 3, 4, 5003
    logits, scores = draw(B, K, V, 8)
    wide = np.zeros((B * K, V + 9), np.float32)
    wide[:, 5:5 + V] = logits.reshape(B * K, V)
    rows = Tensor(wide).slice([slice(None), slice(5, 5 + V)])
    s, p, t = Tensor(scores), core.zeros((B, K), "int32"), core.zeros((B, K), "int64")
    r = lambda x: x._handle.ref()  # noqa: E731
    lib.call("kd_beam_select", r(rows), r(s), 11, r(s), r(p), r(t), None)
    want = beam_answer(logits, scores, 11)
    assert np.array_equal(p.dataAsync(), want[1]) and np.array_equal(t.dataAsync(), want[2])
    assert np.abs(s.dataAsync() - want[0]).max() <= 60 * 2.0 ** -24 + 40 * 2.0 ** -24


def test_the_same_call_gives_the_same_bits(backend):
    logits, scores = draw(4, 8, 40000, 9)
    a, b = (beam_select(Tensor(logits), Tensor(scores), 1) for _ in range(2))
    assert all(np.array_equal(x.dataAsync(), y.dataAsync()) for x, y in zip(a, b))


def test_beam_select_refuses(backend):
    f = lambda *s: core.zeros(s)  # noqa: E731
    for logits, scores, eos in ((f(2, 3, 10), f(2, 4), -1), (f(5, 10), f(2, 3), -1), (core.zeros((2, 3, 10), "bfloat16"), f(2, 3), -1), (f(2, 3, 10), core.zeros((2, 3), "bfloat16"), -1),
                                (f(2, 3, 10), f(2, 3), 10), (f(1, 33, 50), f(1, 33), -1), (f(2, 3, 1), f(2, 3), -1), (f(6), f(2, 3), -1), (f(2, 3, 20).slice(":, :, ::2"), f(2, 3), -1),
                                (f(4, 3, 10).slice("::2"), f(2, 3), -1)):
        with pytest.raises((lib.KandleCudaError, ValueError)) as e:
            beam_select(logits, scores, eos)
        assert getattr(e.value, "status", 1) == 1
