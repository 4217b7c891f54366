"""Qwen3Engine: prompts in portions, further turns behind running sequences, and beam search over shared pages."""
import numpy as np
import pytest

from kandle_b200 import core, lib, synth
from kandle_b200.core import Tensor
from kandle_b200.engine import Qwen3Engine
from kandle_b200.model_utils.qwen3 import Qwen3Config
from tests.paged_cases import beam_answer

pytestmark = pytest.mark.gpu

DIMS = dict(vocab=1024, hidden=256, inter=512, layers=3, heads=4, kv_heads=2)


def engine(head_dim=128, batch=4, room=384, std=0.05, **more):
    w = {k: lib.round_to_bf16(v) for k, v in synth.qwen3_weights(std=std, head_dim=head_dim, **DIMS).items()}
    cfg = Qwen3Config(vocabSize=1024, hiddenSize=256, intermediateSize=512, numHiddenLayers=3, numAttentionHeads=4, numKeyValueHeads=2, headDim=head_dim, dtype="bfloat16")
    return Qwen3Engine(cfg, w, batch, room, **more)


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("paged", [True, False])
def test_a_prompt_in_portions_is_the_prompt(backend, head_dim, paged):
    """Logits of every place and the tokens that follow, against the prompt in one piece (bf16 activations: the bound of the engines' other tests)."""
    eng = engine(head_dim, paged=paged)
    ids = synth.token_ids("portions", (3, 301), 1024)
    tok, full = eng.prefill(ids, all_logits=True)
    want, full = tok.dataAsync(), full.dataAsync()
    rows = [t.dataAsync() for t in (eng.k_cache[2], eng.v_cache[2])]
    for cut in (300, 128, 97, 1000):
        tok, parts = eng.prefill(ids, all_logits=True, portion=cut)
        assert parts.shape == full.shape and eng.pos == 301
        assert np.abs(parts.dataAsync() - full).max() <= 2e-2 * max(1.0, np.abs(full).max())
        assert np.array_equal(tok.dataAsync(), parts.dataAsync()[:, -1].argmax(-1))
        for a, t in zip(rows, (eng.k_cache[2], eng.v_cache[2])):
            assert np.abs(a - t.dataAsync()).max() <= 2e-2 * np.abs(a).max() * 2
    first = full[:, -1]
    top = np.sort(first, -1)
    clear = top[:, -1] - top[:, -2] > 4e-2 * np.abs(first).max()
    assert np.array_equal(tok.dataAsync()[clear], want[clear])
    eng.dispose()


@pytest.mark.parametrize("paged", [True, False])
def test_a_further_turn_stands_behind_what_was_generated(backend, paged):
    """prefill, a few steps, the user's next tokens: the logits are those of the whole text as one prompt, and decoding goes on."""
    eng = engine(paged=paged)
    ids = synth.token_ids("turns", (4, 120), 1024)
    said = eng.generate(ids, 12)
    more = np.concatenate([said[:, -1:], synth.token_ids("next", (4, 20), 1024)], 1).astype(np.int32)   # the last token is not in the cache yet
    assert eng.pos == 131
    tok, parts = eng.extend(more, all_logits=True)
    got, after = parts.dataAsync(), tok.dataAsync()
    eng.start_decode(tok)
    steps = [eng.decode_step().dataAsync() for _ in range(3)]
    whole = np.concatenate([ids, said[:, :-1], more], 1).astype(np.int32)
    tok, full = eng.prefill(whole, all_logits=True)
    want = full.dataAsync()[:, 131:]
    assert np.abs(got - want).max() <= 2e-2 * max(1.0, np.abs(want).max())
    tail = np.concatenate([whole, after[:, None], *[s[:, None] for s in steps[:-1]]], 1).astype(np.int32)
    lg = eng.prefill(tail, all_logits=True)[1].dataAsync()[:, len(whole[0]):]
    chosen = np.take_along_axis(lg, np.stack(steps, 1)[..., None], -1)[..., 0]
    assert (lg.max(-1) - chosen <= 4e-2 * np.abs(lg).max()).all()
    eng.dispose()


def test_extend_refuses(backend):
    eng = engine(room=256, paged=True)
    ids = synth.token_ids("refuse", (2, 250), 1024)
    eng.prefill(ids)
    with pytest.raises(ValueError, match="overflow"):
        eng.extend(ids[:, :7])
    with pytest.raises(ValueError, match="running"):
        eng.extend(ids[:1, :3])
    with pytest.raises(ValueError):
        eng.prefill(ids, portion=0)
    with pytest.raises(ValueError):
        eng.prefill(synth.token_ids("long", (2, 257), 1024), portion=100)
    eng.extend(ids[:, :6])
    assert eng.pos == 256
    eng.dispose()


def _by_hand(eng, ids, K, steps, eos):
    """Beam search with the contiguous engine: every step's cache rows are moved on the host, the choice is float64's."""
    (B, S), R = ids.shape, ids.shape[0] * K
    eng.prefill(ids)

    def gather(rows):
        for caches in (eng.k_cache, eng.v_cache):
            for i, t in enumerate(caches):
                a = t.dataAsync()
                a[:R] = a[rows]
                core.copy_(t, Tensor(a, dtype="bfloat16"))

    logits = np.repeat(eng._prefill_bufs[(B, S)]["logits"].dataAsync().reshape(B, 1, -1), K, 1)
    scores = np.full((B, K), -np.inf, np.float32)
    scores[:, 0] = 0
    source = np.repeat(np.arange(B), K)
    running, ended = [[[]] * K for _ in range(B)], [[] for _ in range(B)]
    for step in range(1, steps + 1):
        s, parents, tokens, ends = beam_answer(logits, scores, eos)
        for i in range(B):
            ended[i] += [(running[i][j] + [eos], ends[i, j] / step) for j in range(K) if np.isfinite(ends[i, j])]
            running[i] = [running[i][p] + [int(t)] for p, t in zip(parents[i], tokens[i])]
        scores = s.astype(np.float32)
        if step == steps:
            break
        gather(source if step == 1 else (np.arange(B)[:, None] * K + parents).reshape(-1))
        eng.start_decode(Tensor(tokens.reshape(R)), use_graph=False)
        eng.decode_step()
        logits = eng._decode["logits"].dataAsync().reshape(B, K, -1)
    return running, scores, ended


@pytest.mark.parametrize("B,K,S,steps,use_graph", [(2, 4, 120, 14, True), (1, 3, 127, 6, False), (3, 2, 128, 5, True), (1, 4, 5, 12, True), (1, 8, 250, 12, True), (2, 1, 60, 4, True)])
def test_beams_are_those_of_a_search_by_hand(backend, B, K, S, steps, use_graph):
    ids = synth.token_ids(f"beams{S}", (B, S), 1024)
    eng = engine(batch=B * K, paged=True, spare_pages=B * K)
    first = eng.generate(ids, 6)
    got = eng.generate_beams(ids, K, steps, -1, use_graph=use_graph)
    flat = engine(batch=B * K)
    running, scores, _ = _by_hand(flat, ids, K, steps, -1)
    for i in range(B):
        assert [h[0] for h in got[i]] == running[i]
        assert np.allclose([h[1] for h in got[i]], scores[i] / steps, rtol=1e-5, atol=1e-5)
    if K == 1:
        assert np.array_equal([h[0][0] for h in got], eng.generate(ids, steps))
    # with end tokens, one of the greedy answer and one that a hypothesis comes to: all steps are gone through by hand, and the best of what
    # ended and what runs agree
    for eos in (int(first[0, 3]), got[0][0][0][steps // 2]):
        got = eng.generate_beams(ids, K, steps, eos, use_graph=use_graph)
        running, scores, ended = _by_hand(flat, ids, K, steps, eos)
        for i in range(B):
            pool = sorted(sorted(ended[i], key=lambda h: -h[1])[:K] + [(r, s / steps) for r, s in zip(running[i], scores[i])], key=lambda h: -h[1])[:K]
            if len(ended[i]) < K:              # not done before the last step
                assert [h[0] for h in got[i]] == [h[0] for h in pool]
            for tokens, score in got[i]:
                assert tokens.count(eos) <= 1 and (eos not in tokens or tokens[-1] == eos)
                assert any(tokens == h[0] and abs(score - h[1]) < 1e-4 for h in ended[i] + pool) or len(ended[i]) >= K
    assert any(ended)
    # the cache and the plain generation are as they were
    assert np.array_equal(eng.generate(ids, 6), first)
    again = eng.generate_beams(ids, K, steps, -1, use_graph=use_graph)
    assert [[h[0] for h in x] for x in again] == [[h[0] for h in x] for x in eng.generate_beams(ids, K, steps, -1, use_graph=not use_graph)]
    eng.dispose()
    flat.dispose()


def test_beams_refuse(backend):
    ids = synth.token_ids("beams.refuse", (2, 20), 1024)
    eng = engine(batch=4, room=128)
    with pytest.raises(ValueError, match="paged"):
        eng.generate_beams(ids, 2, 4)
    eng = engine(batch=4, room=128, paged=True)
    for K, steps in ((0, 4), (3, 4), (2, 0), (2, 109)):
        with pytest.raises(ValueError):
            eng.generate_beams(ids, K, steps)
    with pytest.raises(ValueError, match="overflow"):
        eng.generate_beams(ids, 2, 4)       # two pages a beam and one page a row: spare_pages is for that
    assert eng.generate(ids, 3).shape == (2, 3)
    eng.dispose()
