"""Operators of a paged cache and of beam search refuse outputs that lie over what they read, before anything is launched."""
import numpy as np
import pytest
import torch

from kandle_b200 import core, lib, paged
from kandle_b200.core import Tensor
from tests.paged_cases import attention_answer, attention_case
from tests.test_paged_gpu import put

pytestmark = pytest.mark.gpu


def refused(call):
    with pytest.raises(lib.KandleCudaError) as e:
        call()
    assert e.value.status == 1 and "share" in str(e.value)


def test_attention_refuses_outputs_over_what_it_reads(backend):
    T, H, G, D = 40, 8, 2, 64
    row = core.zeros((T + 8, 3 * H, D), "bfloat16")
    view = lambda first, head, strides=(3 * H * D, D, 1): row._view((T, H, D), strides, first * 3 * H * D + head * D)  # noqa: E731
    k, v = (core.zeros((3, G, 128, D), "bfloat16") for _ in range(2))
    table, keys, start = Tensor(np.array([[0, 1]], np.int32)), Tensor(np.array([200], np.int32)), Tensor(np.array([0, T], np.int32))
    q = view(0, 0)
    before = backend.launch_count()
    for out in (q, view(1, 0), view(8, 0), view(0, H - 1), view(0, H, (3 * H * D, 2 * D, 1))):
        refused(lambda: paged.attention(q, k, v, table, keys, q_start=start, out=out))
    for pool in (k, v):
        refused(lambda: paged.attention(q, k, v, table, keys, out=pool._view((T, H, D), (H * D, D, 1), 64 * D)))
    assert backend.launch_count() == before
    wide = core.zeros((T * H * D + 64,), "bfloat16")
    ints = core.zeros((64,), "int32")
    paged.attention(q, k, v, table, keys, q_start=start, out=wide._view((T, H, D), (H * D, D, 1), 64))
    paged.attention(q, k, v, ints._view((1, 2), (2, 1), 0), ints._view((1,), (1,), 8), out=core.zeros((T, H, D), "bfloat16"))
    backend.synchronize()


def test_queries_and_outputs_may_be_heads_of_one_buffer(backend):
    """A projection's row holds queries and, behind them or in turn with them, room for the outputs."""
    H, G, D = 8, 2, 64
    c = attention_case([3, 150], [300, 400], H, G, D, seed=11)
    T = c["q"].shape[0]
    want, tol = attention_answer(c)
    for step, first in ((1, H), (2, 1)):
        rows = torch.zeros(T, 2 * H, D, dtype=torch.bfloat16)
        rows[:, :H * step:step] = c["q"]
        t = put(rows)
        q, out = (t._view((T, H, D), (2 * H * D, step * D, 1), at * D) for at in (0, first))
        paged.attention(q, put(c["k"]), put(c["v"]), put(c["table"]), put(c["keys"]), q_start=put(c["start"]), scale=c["scale"], out=out)
        assert ((torch.tensor(out.dataAsync()).double() - want).abs() <= tol).all()
        assert np.array_equal(q.dataAsync(), c["q"].float().numpy())


def test_beam_select_refuses_outputs_over_what_it_reads(backend):
    """The outputs of a request are written while others' logits are still read; only the scores may be updated in place."""
    B, K, V = 3, 4, 300
    logits, scores = core.zeros((B, K, V)), core.zeros((B, K))
    outs = [core.zeros((B, K), t) for t in ("float32", "int32", "int64", "float32")]
    r = lambda x: x._handle.ref() if x is not None else None  # noqa: E731
    call = lambda s, *o: lib.call("kd_beam_select", r(logits), r(s), -1, *map(r, o))  # noqa: E731
    wide = core.zeros((B * K + 8,))
    part = lambda at: wide._view((B, K), (K, 1), at)  # noqa: E731
    inside = logits._view((B, K), (K, 1), 40)
    refused(lambda: call(scores, inside, *outs[1:]))
    refused(lambda: call(scores, *outs[:3], inside))
    refused(lambda: call(part(0), part(4), *outs[1:]))
    refused(lambda: call(part(4), part(0), *outs[1:]))
    refused(lambda: call(scores, *outs[:3], outs[0]))
    refused(lambda: call(scores, *outs[:3], scores))
    call(part(0), part(0), *outs[1:])
    call(scores, scores, *outs[1:3], None)
    call(part(0), *outs)
    backend.synchronize()


def test_forks_and_copies_refuse_lists_and_tables_in_one_another(backend):
    B, K = 2, 3
    pools = [core.zeros((8, 2, 128, 64), "bfloat16") for _ in range(3)]
    ints = core.zeros((200,), "int32")
    part = lambda at, *shape: ints._view(shape, (shape[1], 1) if len(shape) == 2 else (1,), at)  # noqa: E731
    parents, table, spare, length = (lambda: part(0, B, K)), (lambda: part(10, B * K, 4)), (lambda: part(40, B * K)), (lambda: part(50, 1))
    call = lambda a, b, c, d, p=pools: paged.fork_pages(p, a, b, c, d)  # noqa: E731
    refused(lambda: call(part(12, B, K), table(), spare(), length()))
    refused(lambda: call(parents(), table(), part(33, B * K), length()))
    refused(lambda: call(parents(), table(), spare(), part(33, 1)))
    refused(lambda: call(part(41, B, K), table(), spare(), length()))
    refused(lambda: call(parents(), table(), spare(), part(45, 1)))
    both = core.zeros((8 * 2 * 128 * 32 + 8,), "int32")
    pool = both._view((8, 2, 128, 32), (8192, 4096, 32, 1), 0)
    over = lambda *shape: both._view(shape, (shape[1], 1) if len(shape) == 2 else (1,), 100)  # noqa: E731
    for args in ((over(B, K), table(), spare(), length()), (parents(), over(B * K, 4), spare(), length()), (parents(), table(), over(B * K), length()), (parents(), table(), spare(), over(1))):
        refused(lambda: call(*args, p=[pool]))
    refused(lambda: paged.copy_pages([pool], over(2), part(60, 2)))
    refused(lambda: paged.copy_pages([pool], part(60, 2), over(2)))
    call(parents(), table(), spare(), length())
    paged.copy_pages([pool], both._view((2,), (1,), 8 * 8192), part(60, 2))
    paged.copy_pages(pools, part(70, 0), part(60, 0))
    with pytest.raises(lib.KandleCudaError, match="error code 105"):      # (two pairs 0 -> 0)
        backend.synchronize()
