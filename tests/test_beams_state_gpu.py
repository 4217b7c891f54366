"""Qwen3Engine.generate_beams: what an engine keeps from one search to the next."""
import numpy as np
import pytest

from kandle_b200 import core, lib, synth
from kandle_b200.core import Tensor
from kandle_b200.engine import Qwen3Engine
from kandle_b200.model_utils.qwen3 import Qwen3Config

pytestmark = pytest.mark.gpu

K, STEPS = 4, 12


def engine(batch=8, room=256, **more):
    dims = dict(vocab=512, hidden=256, inter=512, layers=2, heads=4, kv_heads=2)
    w = {k: lib.round_to_bf16(v) for k, v in synth.qwen3_weights(std=0.05, head_dim=128, **dims).items()}
    cfg = Qwen3Config(vocabSize=512, hiddenSize=256, intermediateSize=512, numHiddenLayers=2, numAttentionHeads=4, numKeyValueHeads=2, headDim=128, dtype="bfloat16")
    return Qwen3Engine(cfg, w, batch, room, paged=True, spare_pages=2 * batch, **more)


@pytest.mark.parametrize("use_graph", [False, True])
def test_beams_go_through_the_caches_and_the_table_that_the_engine_has_now(backend, use_graph):
    """Steps without a graph read the engine's tensors at every call; captured ones after dispose()."""
    eng = engine()
    ids = synth.token_ids("beams.swap", (2, 120), 512)
    want = eng.generate_beams(ids, K, STEPS, use_graph=use_graph)
    old = [*eng.k_cache, *eng.v_cache]
    before, table = [t.dataAsync() for t in old], eng.block_table
    eng.k_cache, eng.v_cache = ([core.zeros(t.shape, "bfloat16") for t in c] for c in (eng.k_cache, eng.v_cache))
    eng.block_table = Tensor(table.dataAsync())
    if use_graph:
        eng.dispose()
    assert eng.generate_beams(ids, K, STEPS, use_graph=use_graph) == want
    for a, t in zip(before, old):
        assert np.array_equal(a, t.dataAsync()), "nothing is written where the engine was before"
    assert any(t.dataAsync().any() for t in eng.k_cache)
    eng.dispose()


def test_searches_of_many_kinds_leave_nothing_behind(backend, collected):
    """Other end tokens and other numbers of beams: the captured steps and buffers of one kind are kept, not of all."""
    eng = engine()
    ids = synth.token_ids("beams.kinds", (2, 100), 512)
    want = {}
    kinds = [(2, 4, -1), (2, 4, 3), (2, 4, 500), (1, 8, -1), (2, 4, 77), (1, 8, 9)]
    for turn in range(2):
        for n, k, eos in kinds:
            got = eng.generate_beams(ids[:n], k, STEPS, eos)
            assert want.setdefault((n, k, eos), got) == got
            assert len(eng._decode["graph"]) <= 2
        used = backend.memory_stats()
        if turn == 0:
            first = used
    assert used == first
    want = eng.generate(np.repeat(ids, 4, 0), 5)
    eng.generate_beams(ids, 4, STEPS, 5)
    assert np.array_equal(eng.generate(np.repeat(ids, 4, 0), 5), want), "the captured step of the plain generation is another one"
    eng.dispose()


def test_the_prompts_pages_are_those_of_the_block_table_as_it_stands(backend):
    """A program may give the sequences other pages; the array that an engine was built with is the program's own."""
    pages = np.arange(16, dtype=np.int32).reshape(8, 2)
    given = pages.copy()
    eng = engine(page_table=given)
    ids = synth.token_ids("beams.table", (2, 130), 512)
    want = eng.generate_beams(ids, K, STEPS)
    given[:] = pages[::-1]
    assert eng.generate_beams(ids, K, STEPS) == want and np.array_equal(eng.block_table.dataAsync(), pages)
    other = np.random.default_rng(3).permutation(16).astype(np.int32).reshape(8, 2)
    backend.upload(eng.block_table._handle, other)
    for use_graph in (True, False):
        assert eng.generate_beams(ids, K, STEPS, use_graph=use_graph) == want
        assert np.array_equal(eng.block_table.dataAsync(), other), "the table is left as it was"
    eng.dispose()


@pytest.mark.parametrize("use_graph", [False, True])
def test_a_search_fills_the_cache_to_its_last_position(backend, use_graph):
    """As generate does: the last token's keys are not needed."""
    eng, roomy = engine(room=128), engine(room=384)
    ids = synth.token_ids("beams.full", (2, 117), 512)
    assert eng.generate(ids, 12).shape == (2, 12)
    assert eng.generate_beams(ids, K, 12, use_graph=use_graph) == roomy.generate_beams(ids, K, 12, use_graph=use_graph)
    with pytest.raises(ValueError, match="overflow"):
        eng.generate_beams(ids, K, 13)
    eng.dispose()
    roomy.dispose()
