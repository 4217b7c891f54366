"""Calls over a paged cache at the edges of what they take, and a step of beam search as a program makes it: the choice, the pages behind it and
the attention over them in one captured graph."""
import ctypes
import json
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from kandle_b200 import core, io, lib, paged, synth
from kandle_b200.core import Tensor
from kandle_b200.model_utils import beam_select
from tests.paged_cases import PAGE, attention_answer, attention_case, beam_answer, bf16, fork_answer
from tests.test_beams_engine_gpu import DIMS, engine
from tests.test_paged_gpu import check, put, run

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("count,most", [(300, 1), (700, 2), (260, 40)])
def test_more_sequences_than_a_block_keeps(backend, count, most):
    rng = np.random.default_rng(count)
    new = rng.integers(0, most + 1, count).tolist()
    new[-1] = most
    c = attention_case(new, [n + int(k) for n, k in zip(new, rng.integers(0, 200, count))], 4, 2, 64, seed=count)
    got = run(c, max_query=most)
    check(c, got)
    assert np.array_equal(run(c, max_query=most), got)


@pytest.mark.parametrize("new,keys,heads,kv_heads,dim", [([301], [700], 64, 1, 64), ([131, 2], [131, 900], 96, 2, 128), ([1, 260], [40, 290], 43, 1, 64)])
def test_tiles_of_few_tokens(backend, new, keys, heads, kv_heads, dim):
    """Groups of 64, 48 and 43 heads: two tokens to a tile, and rows of it that nobody has."""
    c = attention_case(new, keys, heads, kv_heads, dim, seed=heads)
    check(c, run(c))


def test_outputs_in_place_of_the_queries_are_refused(backend):
    c = attention_case([2], [5], 4, 2, 64)
    q = put(c["q"])
    with pytest.raises(lib.KandleCudaError) as e:
        paged.attention(q, put(c["k"]), put(c["v"]), put(c["table"]), put(c["keys"]), put(c["start"]), out=q)
    assert e.value.status == 1


@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 128), (64, 1, 64), (40, 1, 128)])
def test_a_context_that_repeats_itself(backend, heads, kv_heads, dim):
    """Five pages 1000 times over, 640000 positions: one token's answer is that of the five.  The sums are longer than attention_answer counts: chains of up to
    34 pages of 128 keys a block in fp32, 2^-24 for an addition, so 2^-11 of the mass for the sum and as much for its divisor: a quarter of its 2^-8."""
    c = attention_case([1], [5 * PAGE], heads, kv_heads, dim, seed=dim)
    want, tol = attention_answer(c)
    table = np.ascontiguousarray(np.tile(c["table"], (1, 1000)))
    got = run(dict(c, table=table, keys=c["keys"] * 1000), max_query=1)
    assert ((torch.tensor(got).double() - want).abs() <= 1.25 * tol).all()


def test_more_pages_than_are_counted_are_refused(backend):
    """8192 sequences that all name the same 2^18 pages: reported, and nothing is read or written."""
    B, pages = 8192, 1 << 18
    pool = core.zeros((2, 1, PAGE, 64), "bfloat16")
    table = core.zeros((1, pages), "int32").expand([B, pages])
    out = core.full((B, 2, 64), 7.0, "bfloat16")
    q = core.zeros((B, 2, 64), "bfloat16")
    paged.attention(q, pool, pool, table, core.full((1,), pages * PAGE, "int32"), out=out)
    with pytest.raises(lib.KandleCudaError, match="error code 107"):
        backend.synchronize()
    assert (out.dataAsync() == 7.0).all()
    ones = core.full((1,), 1, "int32")
    with pytest.raises(lib.KandleCudaError) as e:
        paged.attention(q, pool, pool, core.zeros((1, pages + 1), "int32").expand([B, pages + 1]), ones, out=out)
    assert e.value.status == 1
    assert (paged.attention(q, pool, pool, table, ones, out=out).dataAsync() == 0.0).all()


@pytest.mark.parametrize("n", [1000, 4096, 4097, 6000])
def test_long_lists_of_copies(backend, n):
    rng = np.random.default_rng(n)
    order = rng.permutation(2 * n + 5).astype(np.int32)
    values = [rng.integers(-128, 128, (2 * n + 5, 1, PAGE, 8)).astype(np.float32) for _ in range(2)]
    pools = [Tensor(v, dtype="bfloat16") for v in values]
    src, dst = order[:n].copy(), order[n:2 * n].copy()
    paged.copy_pages(pools, Tensor(src), Tensor(dst))
    backend.synchronize()
    for v, p in zip(values, pools):
        v[dst] = v[src]
        assert np.array_equal(p.dataAsync(), v)
    # the last pair goes where the first does, and one in the middle to where another comes from
    dst[-1], dst[n // 2] = dst[0], src[n // 3]
    left_out = [0, n - 1, n // 2]
    src[:] = rng.permutation(src)
    if src[n // 2] == dst[n // 2]:
        src[[n // 2, 1]] = src[[1, n // 2]]
    paged.copy_pages(pools, Tensor(src), Tensor(dst))
    with pytest.raises(lib.KandleCudaError, match="error code 105"):
        backend.synchronize()
    good = np.setdiff1d(np.arange(n), left_out)
    for v, p in zip(values, pools):
        v[dst[good]] = v[src[good]]
        assert np.array_equal(p.dataAsync(), v)


class Step:
    """beams of two requests over one layer's cache, on the host and on the device."""

    def __init__(self, length, seed, B=2, K=3, V=5000, heads=8, kv_heads=4, dim=64):
        rng = np.random.default_rng(seed)
        R, width = B * K, -(-max(length, 1) // PAGE) + 1
        pages = R * width + R
        order = rng.permutation(pages)
        self.table = order[:R * width].reshape(B, K, width).astype(np.int32)
        self.table[:, :, :length // PAGE] = self.table[:, :1, :length // PAGE]
        self.table = self.table.reshape(R, width)
        self.spare = order[R * width:].astype(np.int32)
        self.pools = [bf16(rng.standard_normal((pages, kv_heads, PAGE, dim))).float().numpy() for _ in range(2)]
        self.q = bf16(rng.standard_normal((R, heads, dim)) * 1.5)
        self.logits = (rng.standard_normal((B, K, V)) * 2.5).astype(np.float32)
        self.scores = (-3 * rng.random((B, K))).astype(np.float32)
        self.length, self.eos = length, 17

    def put(self):
        d = {n: Tensor(getattr(self, n)) for n in ("table", "spare", "logits", "scores")}
        d["q"], d["length"] = put(self.q), Tensor(np.array([self.length], np.int32))
        d["pools"] = [Tensor(p, dtype="bfloat16") for p in self.pools]
        d["out"] = core.empty(tuple(self.q.shape), "bfloat16")
        d["choice"] = beam_select(d["logits"], d["scores"], self.eos)
        return d

    def copy_to(self, d):
        fresh = self.put()
        for n in ("table", "spare", "logits", "scores", "q", "length"):
            core.copy_(d[n], fresh[n])
        for a, b in zip(d["pools"], fresh["pools"]):
            core.copy_(a, b)

    def call(self, d):
        beam_select(d["logits"], d["scores"], self.eos, out=(d["scores"], *d["choice"][1:]))
        paged.fork_pages(d["pools"], d["choice"][1], d["table"], d["spare"], d["length"])
        paged.attention(d["q"], *d["pools"], d["table"], d["length"], max_query=1, out=d["out"])

    def check(self, d):
        scores, parents, tokens, _ = beam_answer(self.logits, self.scores, self.eos)
        assert np.array_equal(d["choice"][1].dataAsync(), parents) and np.array_equal(d["choice"][2].dataAsync(), tokens)
        assert (np.abs(d["scores"].dataAsync() - scores) <= 60 * 2.0 ** -24 + np.abs(scores) * 2.0 ** -24).all()
        pools = [p.copy() for p in self.pools]
        table, spare = fork_answer(pools, parents, self.table, self.spare, self.length)
        assert np.array_equal(d["table"].dataAsync(), table) and np.array_equal(d["spare"].dataAsync(), spare)
        assert all(np.array_equal(a.dataAsync(), b) for a, b in zip(d["pools"], pools))
        R = len(table)
        check({"q": self.q, "k": bf16(pools[0]), "v": bf16(pools[1]), "table": table, "start": np.arange(R + 1), "keys": np.full(R, self.length), "scale": self.q.shape[-1] ** -0.5},
              d["out"].dataAsync())


@pytest.mark.parametrize("pdl", [0, 1])
def test_two_captured_steps_share_the_scratch(backend, pdl):
    """Replayed in turn, between calls that are not captured; each on a cache of another length."""
    first, second = Step(200, 1), Step(391, 2, B=1, K=8)
    states, graphs = [first.put(), second.put()], []
    for s, d in zip((first, second), states):
        s.call(d)
        s.check(d)
    for s, d in zip((first, second), states):
        lib.call("kd_graph_begin")
        lib.call("kd_set_pdl", pdl)
        try:
            s.call(d)
        finally:
            lib.call("kd_set_pdl", 0)
        g = ctypes.c_uint64(0)
        lib.call("kd_graph_end", ctypes.byref(g))
        graphs.append(g)
    loose = attention_case([3, 200], [300, 450], 8, 4, 64)
    for seed in (3, 4, 5):
        news = [Step(130 + 9 * seed, seed), Step(385 + seed, 10 * seed, B=1, K=8)]
        for s, d in zip(news, states):
            s.copy_to(d)
        lib.call("kd_graph_launch", graphs[0])
        lib.call("kd_graph_launch", graphs[1])
        check(loose, run(loose))
        for s, d in zip(news, states):
            s.check(d)
    for g in graphs:
        lib.call("kd_graph_destroy", g)


@pytest.mark.parametrize("low", [-3.4028235e38, -2.5e38])
def test_rows_of_the_lowest_numbers(backend, low):
    """A beam whose mask leaves nothing is uniform over its tokens, as in float64; one that it leaves something has those."""
    logits = np.full((1, 3, 9000), low, np.float32)
    logits[0, 1, [5, 4100, 8999]] = [1.0, 3.0, 2.0]
    logits[0, 2, ::2] = 0.25
    scores = np.array([[-0.5, -1.0, -0.75]], np.float32)
    s, p, t, e = (x.dataAsync() for x in beam_select(Tensor(logits), Tensor(scores), 4100))
    want = beam_answer(logits, scores, 4100)
    assert np.array_equal(p, want[1]) and np.array_equal(t, want[2])
    # 9000 equal terms in fp32: each addition is off by half a step of the sum so far at most, in chains of 32, and the exponential by 2^-22
    assert (np.abs(s - want[0]) <= 60 * 2.0 ** -24 + np.abs(want[0]) * 2.0 ** -24).all() and np.array_equal(np.isfinite(e), np.isfinite(want[3]))


def test_vocabularies_beyond_two_to_the_30_are_refused(backend):
    logits = core.empty((1, 1, (1 << 30) + 4), "float32")
    with pytest.raises(lib.KandleCudaError) as e:
        beam_select(logits, core.zeros((1, 1)), -1)
    assert e.value.status == 1
    logits.dispose()


@pytest.mark.parametrize("pdl", [0, 1])
def test_a_captured_call_of_two_kernels(backend, pdl):
    """A prompt that is cut into parts of two tiles beside a few tokens; replayed with other lengths and after a call that leaves other parts."""
    a = attention_case([300, 5], [1500, 130], 4, 2, 64, seed=1, table_width=14, spare_pages=9)
    b = attention_case([290, 15], [300, 1700], 4, 2, 64, seed=2, table_width=14, spare_pages=6)
    assert a["k"].shape == b["k"].shape and a["q"].shape == b["q"].shape
    d = {n: put(a[n]) for n in ("q", "k", "v", "table", "keys", "start")}
    out = core.empty(tuple(a["q"].shape), "bfloat16")
    call = lambda: paged.attention(d["q"], d["k"], d["v"], d["table"], d["keys"], q_start=d["start"], scale=a["scale"], out=out)  # noqa: E731
    call()
    check(a, out.dataAsync())
    lib.call("kd_graph_begin")
    lib.call("kd_set_pdl", pdl)
    try:
        call()
    finally:
        lib.call("kd_set_pdl", 0)
    g = ctypes.c_uint64(0)
    lib.call("kd_graph_end", ctypes.byref(g))
    other = attention_case([700, 1, 90], [900, 2000, 400], 8, 2, 128, seed=3)
    for c in (b, a, b):
        for n in d:
            core.copy_(d[n], put(c[n]))
        check(other, run(other))
        lib.call("kd_graph_launch", g)
        check(c, out.dataAsync())
    lib.call("kd_graph_destroy", g)


def test_command_line_searches_with_beams(backend, tmp_path):
    w = {k: lib.round_to_bf16(v) for k, v in synth.qwen3_weights(std=0.05, head_dim=64, **DIMS).items()}
    (tmp_path / "config.json").write_text(json.dumps({"architectures": ["Qwen3ForCausalLM"], "vocab_size": 1024, "hidden_size": 256, "intermediate_size": 512, "num_hidden_layers": 3,
                                                      "num_attention_heads": 4, "num_key_value_heads": 2, "head_dim": 64}))
    io.save_file({k: (lib.f32_to_bf16_bits(v).reshape(np.shape(v)), "BF16") for k, v in w.items()}, str(tmp_path / "model.safetensors"))
    ids = synth.token_ids("cli.beams", (2, 30), 1024)
    command = [sys.executable, "-m", "kandle_b200.generate", "--model", str(tmp_path), "--steps", "5", "--beams", "3", "--eos", "9"]
    for row in ids:
        command += ["--prompt", " ".join(map(str, row))]
    r = subprocess.run(command, capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert r.returncode == 0, r.stderr[-2000:]
    eng = engine(64, batch=6, room=35, paged=True, spare_pages=12)
    want = [h[0][0] for h in eng.generate_beams(ids, 3, 5, 9)]
    eng.dispose()
    assert [[int(x) for x in line.split()] for line in r.stdout.strip().split("\n")] == want
    for more in (["--temperature", "0.5"], ["--beams", "-1"]):
        r = subprocess.run(command + more, capture_output=True, text=True, timeout=300, cwd=ROOT)
        assert r.returncode == 2 and "--beams" in r.stderr
