"""Host logic of beam search: which hypotheses a prompt ends with, whoever is in the batch beside it."""
import numpy as np
import pytest

from kandle_b200.model_utils import BeamHypotheses
from tests.paged_cases import beam_answer, beam_search

V, K, EOS, STEPS = 6, 3, 0, 12


def model(seed):
    """Logits [V] behind a sequence of tokens: any, but always the same ones."""
    def logits(tokens):
        return (np.random.default_rng([seed, len(tokens), *tokens]).standard_normal(V) * 1.5).astype(np.float32)
    return logits


def search(models, power, steps=STEPS):
    """The loop of Qwen3Engine.generate_beams, with made-up models for the prompts and float64's choice.  Returns the answers and each prompt's
    step in which it was done."""
    prompts = [BeamHypotheses(K, EOS, power) for _ in models]
    scores = np.full((len(models), K), -np.inf, np.float32)
    scores[:, 0] = 0
    beams, when = [[[]] * K for _ in models], [None] * len(models)
    for step in range(1, steps + 1):
        logits = np.stack([[m(t) for t in b] for m, b in zip(models, beams)])
        new, parents, tokens, ends = beam_answer(logits, scores, EOS)
        scores = new.astype(np.float32)
        beams = [[b[q] + [int(t)] for q, t in zip(p, ts)] for b, p, ts in zip(beams, parents, tokens)]
        for i, prompt in enumerate(prompts):
            prompt.step(parents[i], tokens[i], scores[i], ends[i])
            if prompt.done and when[i] is None:
                when[i] = step
        if all(p.done for p in prompts):
            break
    return [p.best() for p in prompts], when


@pytest.mark.parametrize("power", [0.0, 1.0, 2.0])
def test_a_prompts_hypotheses_do_not_depend_on_the_others(power):
    early = 0
    for seed in range(0, 60, 3):
        models = [model(seed + i) for i in range(3)]
        got, when = search(models, power)
        early += len({w or STEPS for w in when}) > 1
        for m, g, w in zip(models, got, when):
            alone, own = search([m], power)
            assert own == [w] and alone == [g]
    assert early > 0, "prompts that are done in different steps"


@pytest.mark.parametrize("power", [0.0, 0.7, 1.0])
def test_the_hypotheses_are_those_of_the_rule(power):
    """Against the rule written down for one prompt alone (beam_search of the cases)."""
    ends = 0
    for seed in range(100, 140):
        got, when = search([model(seed)], power)
        want, done = beam_search(lambda beams, m=model(seed): np.stack([m(t) for t in beams]), K, EOS, STEPS, power)
        assert [h[0] for h in got[0]] == [h[0] for h in want] and np.allclose([h[1] for h in got[0]], [h[1] for h in want], rtol=1e-6)
        assert when == [done]
        ends += done is not None
    assert 0 < ends


def test_without_an_end_the_running_beams_are_the_answer():
    p = BeamHypotheses(2, -1, 1.0)
    none = np.full(2, -np.inf)
    p.step([0, 0], [4, 5], np.array([-1.0, -2.0]), none)
    p.step([1, 0], [3, 3], np.array([-2.5, -np.inf]), none)
    assert p.best() == [([5, 3], -1.25)] and not p.done


def test_a_prompt_that_is_done_stays_as_it_is():
    p = BeamHypotheses(1, 9, 1.0)
    p.step([0], [4], np.array([-3.0]), np.array([-1.0]))
    assert p.done and p.best() == [([9], -1.0)]
    p.step([0], [4], np.array([-0.1]), np.array([-0.2]))
    assert p.done and p.best() == [([9], -1.0)]
