"""Qwen3Engine.generate_beams: prompts that are done before others of their batch."""
import numpy as np
import pytest

from kandle_b200 import core, lib, synth
from kandle_b200.core import Tensor
from kandle_b200.engine import Qwen3Engine
from kandle_b200.model_utils.qwen3 import Qwen3Config
from tests.paged_cases import beam_answer, beam_rule

pytestmark = pytest.mark.gpu

VOCAB, B, K, S, STEPS = 64, 3, 3, 20, 16     # few tokens, so that every one of them is an end now and then


def engine(**more):
    dims = dict(vocab=VOCAB, hidden=256, inter=512, layers=2, heads=4, kv_heads=2)
    w = {k: lib.round_to_bf16(v) for k, v in synth.qwen3_weights(std=0.05, head_dim=128, **dims).items()}
    cfg = Qwen3Config(vocabSize=VOCAB, hiddenSize=256, intermediateSize=512, numHiddenLayers=2, numAttentionHeads=4, numKeyValueHeads=2, headDim=128, dtype="bfloat16")
    return Qwen3Engine(cfg, w, B * K, 128, **more)


def steps_by_hand(eng, ids, eos):
    """The outputs of every step of a beam search with the contiguous engine: cache rows are moved on the host, the choice is float64's."""
    R = B * K
    eng.prefill(ids)
    logits = np.repeat(eng._prefill_bufs[(B, S)]["logits"].dataAsync().reshape(B, 1, -1), K, 1)
    scores = np.full((B, K), -np.inf, np.float32)
    scores[:, 0] = 0
    rows, outputs = np.repeat(np.arange(B), K), []
    for step in range(STEPS):
        if step:
            for caches in (eng.k_cache, eng.v_cache):
                for t in caches:
                    a = t.dataAsync()
                    a[:R] = a[rows]
                    core.copy_(t, Tensor(a, dtype="bfloat16"))
            eng.start_decode(Tensor(outputs[-1][2].reshape(R)), use_graph=False)
            eng.decode_step()
            logits = eng._decode["logits"].dataAsync().reshape(B, K, -1)
        outputs.append(beam_answer(logits, scores, eos))
        scores = outputs[-1][0].astype(np.float32)
        if step:                         # (the first step's beams all stand in their prompt's one row)
            rows = (np.arange(B)[:, None] * K + outputs[-1][1]).reshape(-1)
    return outputs


def test_every_prompt_of_a_batch_ends_with_its_own_hypotheses(backend):
    """Tokens and scores are those of the rule for each prompt, and do not change with the prompts beside it (the same rows of the same kernels)."""
    ids = synth.token_ids("beams.done", (B + 1, S), VOCAB)
    eng, flat = engine(paged=True, spare_pages=2 * B * K), engine()
    early = later = 0
    for eos in range(0, VOCAB, 7):
        outputs = steps_by_hand(flat, ids[:B], eos)
        for power in (0.0, 1.0):
            got = eng.generate_beams(ids[:B], K, STEPS, eos, power, use_graph=eos % 2 == 0)
            when = []
            for i in range(B):
                want, done = beam_rule([[x[i] for x in o] for o in outputs], K, eos, STEPS, power)
                when.append(done or STEPS)
                assert [h[0] for h in got[i]] == [h[0] for h in want]
                assert np.allclose([h[1] for h in got[i]], [h[1] for h in want], rtol=1e-5, atol=1e-5)
            early += len(set(when)) > 1
            others = ids[[0, B, 1]]
            assert eng.generate_beams(others, K, STEPS, eos, power, use_graph=eos % 2 == 0)[0] == got[0]
            later += any(w < max(when) for w in when)
    assert early and later
    eng.dispose()
    flat.dispose()
