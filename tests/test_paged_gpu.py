"""GPU checks of attention over a paged cache (kd_attention_paged), copies of pages (kd_kv_pages_copy) and beams that share pages
(kd_kv_pages_fork) against their definitions in float64 and plain loops."""
import ctypes

import numpy as np
import pytest
import torch

from kandle_b200 import core, lib, paged
from kandle_b200.core import Tensor
from tests.paged_cases import PAGE, attention_answer, attention_case, fork_answer

pytestmark = pytest.mark.gpu

FILL = 7.0     # what outputs hold before a call


def put(t):
    """A torch bf16 or numpy array on the device, bit for bit."""
    if isinstance(t, torch.Tensor):
        return Tensor(t.contiguous().view(torch.int16).numpy().view(np.uint16), dtype="bfloat16", shape=tuple(t.shape))
    return Tensor(t)


def run(c, out=None, **more):
    out = core.full(c["q"].shape, FILL, "bfloat16") if out is None else out
    d = {n: put(c[n]) for n in ("q", "k", "v", "table", "keys", "start")}
    paged.attention(d["q"], d["k"], d["v"], d["table"], d["keys"], q_start=d["start"], scale=c["scale"], out=out, **more)
    return out.dataAsync()


def check(c, got):
    want, tol = attention_answer(c)
    off = (torch.tensor(got).double() - want).abs()
    worst = (off - tol).max()
    assert torch.isfinite(off).all() and worst <= 0, f"over the bound by {worst:.3g}; largest difference {off.max():.3g}"


SHAPES = [
    # one token, short and long, a page's edges
    ([1], [1], 16, 8, 128), ([1], [127], 4, 4, 64), ([1], [128], 8, 2, 128), ([1], [129], 2, 1, 64), ([1], [5000], 16, 8, 128),
    ([1, 1, 1, 1, 1], [640, 3, 1100, 1, 256], 8, 4, 128),
    # a few tokens, groups that do and do not divide a tile, one head
    ([5], [5], 6, 2, 128), ([9, 2, 17], [300, 2, 140], 32, 8, 128), ([3], [700], 5, 1, 64), ([7, 8], [1000, 129], 14, 2, 128), ([16], [2000], 64, 1, 64),
    ([2, 33], [900, 50], 24, 8, 64), ([1], [300], 64, 1, 128), ([4], [513], 12, 12, 64),
    # portions of prompts
    ([128], [128], 2, 1, 128), ([129], [129], 2, 2, 128), ([200], [1000], 4, 2, 64), ([257], [400], 3, 1, 128), ([300, 1, 77], [300, 513, 1500], 8, 2, 128),
    ([513], [2300], 4, 4, 64), ([64], [4000], 16, 8, 128), ([100, 300], [228, 4500], 16, 8, 128), ([90], [333], 40, 8, 128),
]


@pytest.mark.parametrize("new,keys,heads,kv_heads,dim", SHAPES)
def test_attention_of_packed_sequences(backend, new, keys, heads, kv_heads, dim):
    """Rows behind a sequence's keys and pages that nobody owns hold NaN; unused entries of the table are -1."""
    c = attention_case(new, keys, heads, kv_heads, dim, seed=len(keys) + keys[0])
    got = run(c)
    check(c, got)
    assert np.array_equal(run(c, max_query=max(new)), got), "the bound on new tokens changes no bit"
    assert np.array_equal(run(c, max_query=max(new)), got), "the same call gives the same bits"


@pytest.mark.parametrize("most,longest,heads,kv_heads,dim", [(1, 700, 32, 16, 128), (1, 260, 64, 32, 64), (3, 900, 32, 8, 128), (6, 500, 48, 24, 128), (9, 1300, 40, 20, 64), (40, 400, 64, 16, 128),
                                                             (300, 700, 16, 8, 128), (300, 600, 24, 12, 64), (150, 200, 64, 8, 64)])
def test_attention_of_many_sequences(backend, most, longest, heads, kv_heads, dim):
    """Blocks go through many pieces of sequences of all lengths, some without keys or new tokens."""
    rng = np.random.default_rng(most * longest)
    count = 60 if most < 100 else 30
    new = np.minimum(rng.integers(0, most + 1, count) + (rng.random(count) < 0.8), most).tolist()
    keys = [0 if rng.random() < 0.05 else n + int(k) for n, k in zip(new, rng.integers(0, longest, count) * (rng.random(count) < 0.8))]
    new[7], keys[7] = most, longest
    c = attention_case(new, keys, heads, kv_heads, dim, seed=most)
    got = run(c, max_query=most)
    check(c, got)
    assert np.array_equal(run(c, max_query=most), got)


@pytest.mark.parametrize("junk", [float("inf"), -3e38])
def test_attention_ignores_what_stale_rows_hold(backend, junk):
    c = attention_case([1, 40, 150], [70, 300, 1000], 8, 4, 128, junk=junk)
    check(c, run(c))


def test_tokens_that_see_nothing_get_zero_rows(backend):
    """Fewer keys than new tokens: the first tokens stand before position 0.  No key at all is a zero row too."""
    for new, keys in (([5, 3], [2, 0]), ([300], [170]), ([1], [0]), ([200, 1], [0, 5])):
        c = attention_case(new, keys, 4, 2, 128)
        got = run(c)
        check(c, got)
        for a, n, k in zip(c["start"], new, keys):
            assert not got[a:a + max(0, n - k)].any()


def test_rows_outside_the_sequences_stay_as_they_are(backend):
    c = attention_case([3, 130, 2], [40, 200, 129], 4, 2, 128)
    want, tol = attention_answer(c)
    c["q"] = torch.cat([c["q"][:2] * 0, c["q"], c["q"][:9] * 0])
    c["start"] = c["start"] + 2
    got = run(c)
    assert (got[:2] == FILL).all() and (got[-9:] == FILL).all()
    assert ((torch.tensor(got[2:-9]).double() - want).abs() <= tol).all()


def test_no_new_tokens_in_some_sequences(backend):
    c = attention_case([0, 4, 0, 1], [300, 200, 0, 129], 4, 2, 64)
    check(c, run(c))


@pytest.mark.parametrize("tokens,keys", [(1, 300), (6, 129), (170, 500)])
def test_attention_of_equal_chunks_with_one_length(backend, tokens, keys):
    """q_start left out, one length for all, and queries and outputs as views into wider rows."""
    B, H, G, D = 3, 8, 4, 128
    c = attention_case([tokens] * B, [keys] * B, H, G, D)
    wide = torch.zeros(B * tokens, (H + 2 * G) * D, dtype=torch.bfloat16)
    wide[:, :H * D] = c["q"].reshape(B * tokens, H * D)
    row = put(wide)
    q = row._view((B * tokens, H, D), ((H + 2 * G) * D, D, 1), 0)
    out = core.full((H, B * tokens, D), FILL, "bfloat16")
    paged.attention(q, put(c["k"]), put(c["v"]), put(c["table"]), Tensor(np.array([keys], np.int32)), out=out.permute([1, 0, 2]))
    check(c, out.dataAsync().transpose(1, 0, 2))


def test_pools_and_tables_that_are_views(backend):
    """Keys and values side by side in one page, and a block table with longer rows than are used."""
    c = attention_case([1, 140], [200, 600], 4, 2, 128, table_width=7)
    both = put(torch.stack([c["k"], c["v"]], 1))
    k, v = both.select(1, 0), both.select(1, 1)
    table = put(c["table"]).slice([slice(None), slice(0, 5)])
    got = paged.attention(put(c["q"]), k, v, table, put(c["keys"]), q_start=put(c["start"])).dataAsync()
    check(c, got)


def test_pages_behind_two_to_the_31_numbers(backend):
    H, G, D, pages = 4, 8, 128, 17000
    c = attention_case([1, 70], [300, 200], 2 * G, G, D)
    far = np.arange(pages - 5, pages, dtype=np.int32)
    used = c["k"].shape[0] - 2
    pools = []
    for name in ("k", "v"):
        pool = core.empty((pages, G, PAGE, D), "bfloat16")
        for b in range(2):
            for i, p in enumerate(c["table"][b]):
                if p >= 0:
                    core.copy_(pool.select(0, int(far[b * 3 + i])), put(c[name][int(p)]))
        pools.append(pool)
    assert used == 5
    table = np.array([[far[0], far[1], far[2]], [far[3], far[4], -1]], np.int32)
    got = paged.attention(put(c["q"]), *pools, Tensor(table), put(c["keys"]), q_start=put(c["start"])).dataAsync()
    check(c, got)


def test_a_captured_call_follows_lengths_tables_and_queries(backend):
    a, b = attention_case([1, 3], [200, 700], 8, 4, 128, seed=1, table_width=6, spare_pages=4), attention_case([2, 2], [400, 30], 8, 4, 128, seed=2, table_width=6, spare_pages=7)
    assert a["k"].shape == b["k"].shape
    d = {n: put(a[n]) for n in ("q", "k", "v", "table", "keys", "start")}
    out = core.empty(a["q"].shape, "bfloat16")
    call = lambda: paged.attention(d["q"], d["k"], d["v"], d["table"], d["keys"], q_start=d["start"], max_query=8, scale=a["scale"], out=out)  # noqa: E731
    call()
    check(a, out.dataAsync())
    lib.call("kd_graph_begin")
    call()
    g = ctypes.c_uint64(0)
    lib.call("kd_graph_end", ctypes.byref(g))
    for c in (b, a, b):
        for n in d:
            core.copy_(d[n], put(c[n]))
        lib.call("kd_graph_launch", g)
        check(c, out.dataAsync())
    lib.call("kd_graph_destroy", g)


def test_bad_device_values_are_reported_and_stay_inside(backend):
    good = attention_case([2, 150], [300, 400], 4, 2, 128, table_width=4)

    def expect(code, c, **more):
        run_error = None
        try:
            run(c, **more)
        except lib.KandleCudaError as e:
            run_error = e
        assert run_error is not None and run_error.status == 6 and f"error code {code}" in str(run_error)
        check(good, run(good))

    for page in (-1, good["k"].shape[0], 2 ** 30):
        for b in range(2):
            table = good["table"].copy()
            table[b, 1] = page
            expect(103, dict(good, table=table))
    expect(102, dict(good, keys=np.array([300, 513], np.int32)))
    expect(102, dict(good, keys=np.array([-4, 400], np.int32)))
    expect(104, good, max_query=100)
    expect(104, dict(good, start=np.array([0, 2, 153], np.int32)))
    expect(104, dict(good, start=np.array([-1, 2, 152], np.int32)))
    expect(104, dict(good, start=np.array([0, 60, 2], np.int32)))


def test_attention_refuses(backend):
    c = attention_case([1, 2], [5, 6], 4, 2, 128, junk=0.0)
    q, k, v, table, keys, start = (put(c[n]) for n in ("q", "k", "v", "table", "keys", "start"))
    f32 = core.zeros((3, 4, 128))

    def refused(status, *args, **kw):
        with pytest.raises(lib.KandleCudaError) as e:
            paged.attention(*args, **kw)
        assert e.value.status == status

    refused(1, f32, k, v, table, keys, start)
    refused(1, q, k, v, table, keys, start, out=f32)
    refused(1, q, k, v, table, keys, None)                                    # 3 tokens over 2 sequences
    refused(1, q, k, v, table, keys, keys)                                    # two starts for two sequences
    refused(1, q, k, v, keys.view(1, 2), start, start)
    refused(1, q, k, v, table, keys, start, scale=0.0)
    refused(1, q, k, v, table, keys, start, scale=float("nan"))
    refused(1, q, k, v, table, keys, start, max_query=-1)
    refused(1, core.zeros((3, 3, 128), "bfloat16"), k, v, table, keys, start)  # 3 heads on 2
    refused(1, core.zeros((3, 4, 96), "bfloat16"), k, v, table, keys, start)
    refused(1, q, core.zeros((5, 2, 64, 128), "bfloat16"), v, table, keys, start)
    refused(1, q, k, core.zeros((9, 2, 128, 128), "bfloat16"), table, keys, start)
    wide = core.zeros((3, 4, 132), "bfloat16").slice(":, :, :128")
    refused(1, wide, k, v, table, keys, start, out=core.zeros((3, 4, 128), "bfloat16"))
    refused(1, core.zeros((3, 4, 129), "bfloat16").slice(":, :, 1:"), k, v, table, keys, start)


# ----------------------------------------------------------------------------- pages
def _pools(rng, n, pages, heads, dim, dtype="bfloat16"):
    values = [rng.integers(-128, 128, (pages, heads, PAGE, dim)).astype(np.float32) for _ in range(n)]
    return values, [Tensor(v, dtype=dtype) for v in values]


@pytest.mark.parametrize("n,pages,heads,dim,dtype,moves", [
    (2, 5, 2, 64, "bfloat16", [(1, 3)]), (7, 40, 3, 128, "bfloat16", [(i, 20 + i) for i in range(17)]), (3, 9, 1, 32, "float32", [(8, 0), (7, 7), (0, 1)]),
    (2, 4, 2, 16, "uint8", [(0, 2)]), (130, 3, 1, 8, "bfloat16", [(2, 0)])])
def test_pages_copy(backend, n, pages, heads, dim, dtype, moves):
    if moves[0] == (8, 0):
        moves = [(8, 2), (7, 7), (0, 1)]
    values, pools = _pools(np.random.default_rng(1), n, pages, heads, dim, dtype if dtype != "uint8" else "float32")
    if dtype == "uint8":
        values = [v.clip(0) for v in values]
        pools = [Tensor(v.astype(np.uint8)) for v in values]
    src, dst = (np.array(x, np.int32) for x in zip(*moves))
    paged.copy_pages(pools, Tensor(src), Tensor(dst))
    for v, p in zip(values, pools):
        v[dst] = v[src]
        assert np.array_equal(p.dataAsync().astype(np.float32), v)


def test_pages_copy_between_interleaved_pools(backend):
    rng = np.random.default_rng(2)
    x = rng.integers(-100, 100, (6, 2, 3, PAGE, 64)).astype(np.float32)
    t = Tensor(x, dtype="bfloat16")
    paged.copy_pages([t.select(1, 0), t.select(1, 1)], Tensor(np.array([5, 0], np.int32)), Tensor(np.array([1, 3], np.int32)))
    x[[1, 3]] = x[[5, 0]]
    assert np.array_equal(t.dataAsync(), x)


def test_pages_copy_of_nothing(backend):
    values, pools = _pools(np.random.default_rng(3), 2, 3, 1, 64)
    none = core.empty((0,), "int32")
    paged.copy_pages(pools, none, none)
    paged.copy_pages([], Tensor(np.array([0], np.int32)), Tensor(np.array([1], np.int32)))
    assert all(np.array_equal(p.dataAsync(), v) for p, v in zip(pools, values))


@pytest.mark.parametrize("code,moves,good", [(105, [(0, 4), (1, 4), (2, 5)], [(2, 5)]), (105, [(0, 1), (1, 2), (3, 5)], [(1, 2), (3, 5)]), (103, [(0, 6), (1, 4)], [(1, 4)]),
                                             (103, [(-1, 2), (1, 4)], [(1, 4)]), (103, [(2 ** 30, 2)], []), (105, [(3, 4), (3, 4)], [])])
def test_pages_copy_reports_lists_that_contradict_themselves(backend, code, moves, good):
    values, pools = _pools(np.random.default_rng(4), 2, 6, 2, 64)
    src, dst = (np.array(x, np.int32) for x in zip(*moves))
    paged.copy_pages(pools, Tensor(src), Tensor(dst))
    with pytest.raises(lib.KandleCudaError, match=f"error code {code}"):
        backend.synchronize()
    for v, p in zip(values, pools):
        for a, b in good:
            v[b] = v[a].copy()
        assert np.array_equal(p.dataAsync(), v)


def test_pages_copy_refuses(backend):
    one, two = Tensor(np.array([0], np.int32)), Tensor(np.array([1, 2], np.int32))
    pool = core.zeros((4, 2, PAGE, 64), "bfloat16")
    for pools, a, b in (([pool], one, two), ([pool], Tensor(np.array([0])), one), ([core.zeros((4, 2, 64, 64), "bfloat16")], one, one),
                        ([pool, core.zeros((5, 2, PAGE, 64), "bfloat16")], one, one), ([pool, core.zeros((4, 2, PAGE, 64))], one, one),
                        ([core.zeros((4, 2, PAGE, 4), "bfloat16")], one, one), ([core.zeros((4, 2, PAGE, 128), "bfloat16").slice(":, :, :, :64")], one, one)):
        with pytest.raises(lib.KandleCudaError) as e:
            paged.copy_pages(pools, a, b)
        assert e.value.status == 1


def _fork_state(rng, B, K, length, max_pages, n_pools, heads, dim):
    pages = B * K * max_pages + B * K + 3
    order = rng.permutation(pages)
    table = order[:B * K * max_pages].reshape(B * K, max_pages).astype(np.int32)
    table = table.reshape(B, K, max_pages)
    table[:, :, :length // PAGE] = table[:, :1, :length // PAGE]
    values, pools = _pools(rng, n_pools, pages, heads, dim)
    return values, pools, table.reshape(B * K, max_pages).copy(), order[B * K * max_pages:B * K * max_pages + B * K].astype(np.int32)


@pytest.mark.parametrize("B,K,length,max_pages", [(1, 4, 200, 3), (3, 2, 1, 1), (2, 5, 127, 2), (2, 4, 128, 2), (1, 4, 0, 1), (4, 8, 700, 7), (2, 32, 300, 3), (5, 1, 77, 1),
                                                  (1, 3, 384, 3), (1, 4, 38500, 302)])
def test_beams_go_on_behind_their_parents(backend, B, K, length, max_pages):
    rng = np.random.default_rng(B * K + length)
    values, pools, table, spare = _fork_state(rng, B, K, length, max_pages, 3, 2, 64 if max_pages < 100 else 16)
    T, S, L = Tensor(table), Tensor(spare), Tensor(np.array([length], np.int32))
    for parents in (rng.integers(0, K, (B, K)), np.zeros((B, K), int), np.arange(K)[::-1][None].repeat(B, 0), rng.integers(0, K, (B, K)) // 2):
        parents = np.ascontiguousarray(parents, np.int32)
        paged.fork_pages(pools, Tensor(parents), T, S, L)
        table, spare = fork_answer(values, parents, table, spare, length)
        assert np.array_equal(T.dataAsync(), table) and np.array_equal(S.dataAsync(), spare)
        assert all(np.array_equal(p.dataAsync(), v) for p, v in zip(pools, values))
        tails = np.concatenate([table[:, length // PAGE], spare]) if length % PAGE else spare
        assert len(set(tails.tolist())) == tails.size, "every last page and spare page has one owner"


def test_fork_of_more_pools_than_a_launch_takes(backend):
    rng = np.random.default_rng(9)
    values, pools, table, spare = _fork_state(rng, 1, 3, 50, 1, 131, 1, 8)
    T, S = Tensor(table), Tensor(spare)
    parents = np.array([[2, 2, 2]], np.int32)
    paged.fork_pages(paged.Pools(pools), Tensor(parents), T, S, Tensor(np.array([50], np.int32)))
    table, spare = fork_answer(values, parents, table, spare, 50)
    assert np.array_equal(T.dataAsync(), table) and np.array_equal(S.dataAsync(), spare)
    assert all(np.array_equal(p.dataAsync(), v) for p, v in zip(pools, values))


def test_fork_reports_and_refuses(backend):
    rng = np.random.default_rng(10)
    values, pools, table, spare = _fork_state(rng, 1, 2, 50, 1, 2, 1, 8)

    def call(parents, length, t=table, s=spare):
        paged.fork_pages(pools, Tensor(np.array(parents, np.int32)), Tensor(t), Tensor(s), Tensor(np.array([length], np.int32)))

    for code, args in ((106, ([[0, 2]], 50)), (106, ([[-1, 1]], 50)), (102, ([[0, 1]], 129)), (102, ([[1, 0]], -1)), (103, ([[0, 0]], 50, np.array([[99], [1]], np.int32))),
                       (103, ([[0, 0]], 50, table, np.array([-7, -7], np.int32)))):
        call(*args)
        with pytest.raises(lib.KandleCudaError, match=f"error code {code}"):
            backend.synchronize()
    assert all(np.array_equal(p.dataAsync(), v) for p, v in zip(pools, values))
    i32 = lambda *shape: core.zeros(shape, "int32")  # noqa: E731
    one = i32(1)
    for parents, t, s, n in ((i32(1, 33), i32(33, 1), i32(33), one), (i32(2), i32(2, 1), i32(2), one), (i32(1, 2), i32(3, 1), i32(2), one), (i32(1, 2), i32(2, 1), i32(3), one),
                             (i32(1, 2), i32(2, 1), i32(2), i32(2)), (core.zeros((1, 2)), i32(2, 1), i32(2), one)):
        with pytest.raises(lib.KandleCudaError) as e:
            paged.fork_pages(pools, parents, t, s, n)
        assert e.value.status == 1
