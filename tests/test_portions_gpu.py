"""Qwen3Engine.prefill in portions: what a portion leaves out, and what sampled tokens see of it."""
import numpy as np
import pytest

from kandle_b200 import lib, synth
from kandle_b200.core import Tensor
from kandle_b200.engine import Qwen3Engine
from kandle_b200.model_utils.qwen3 import Qwen3Config

pytestmark = pytest.mark.gpu


def engine(**more):
    dims = dict(vocab=1024, hidden=256, inter=512, layers=2, heads=4, kv_heads=2)
    w = {k: lib.round_to_bf16(v) for k, v in synth.qwen3_weights(std=0.05, head_dim=128, **dims).items()}
    cfg = Qwen3Config(vocabSize=1024, hiddenSize=256, intermediateSize=512, numHiddenLayers=2, numAttentionHeads=4, numKeyValueHeads=2, headDim=128, dtype="bfloat16")
    return Qwen3Engine(cfg, w, 3, 256, **more)


@pytest.mark.parametrize("paged", [True, False])
def test_sampled_tokens_have_the_random_numbers_of_the_prompt_in_one_piece(backend, paged):
    eng = engine(paged=paged)
    ids = synth.token_ids("portions.sampled", (3, 90), 1024)
    drawn = []
    for portion in (None, 89, 40, 7):
        eng.set_sampler(0.8, 20, 0.9, seed=5)
        eng.prefill(ids, portion=portion)
        drawn.append((next(iter(eng._prefill_bufs.values()))["uniforms"].dataAsync(), eng.sampler["rng"].random(4)))
    for first, behind in drawn[1:]:
        assert np.array_equal(first, drawn[0][0]) and np.array_equal(behind, drawn[0][1])
    eng.dispose()


def test_only_the_last_portion_goes_through_the_vocabulary(backend):
    """Kernels launched: two portions take what their layers take, and one ending."""
    eng = engine(paged=True)
    ids = synth.token_ids("portions.count", (2, 96), 1024)

    def launches(run):
        run()
        backend.synchronize()
        before = backend.launch_count()
        run()
        return backend.launch_count() - before

    one = launches(lambda: eng.prefill(ids[:, :48]))
    eng.prefill(ids[:, :48])
    two = launches(lambda: eng.prefill(ids, portion=48))

    def behind():
        eng.pos, eng.cur_B = 48, 2
        eng.extend(ids[:, 48:])

    assert two < one + launches(behind)
    eng.dispose()


def test_tokens_come_as_lists_arrays_or_tensors(backend):
    """As prefill has always taken them; no token at all is refused, and nothing has changed then."""
    eng = engine(paged=True)
    ids = synth.token_ids("portions.lists", (2, 50), 1024)
    want = eng.prefill(ids[:, :30], all_logits=True)[1].dataAsync()
    behind = eng.extend(ids[:, 30:], all_logits=True)[1].dataAsync()
    for kind in (lambda a: a.tolist(), lambda a: a.astype(np.int64), lambda a: Tensor(np.ascontiguousarray(a, np.int32))):
        assert np.array_equal(eng.prefill(kind(ids[:, :30]), all_logits=True)[1].dataAsync(), want)
        for none in (ids[:, :0], [[], []], ids[0]):
            with pytest.raises(ValueError, match="at least one"):
                eng.extend(none)
        assert np.array_equal(eng.extend(kind(ids[:, 30:]), all_logits=True)[1].dataAsync(), behind) and eng.pos == 50
        assert np.array_equal(eng.prefill(kind(ids), all_logits=True, portion=30)[1].dataAsync(), np.concatenate([want, behind], 1))
    eng.dispose()
