"""The operators of a paged cache and of beam search, as cases that can be timed.

  attend   attention of new tokens over a paged cache, sequences of unequal lengths side by side
  beams    the best continuations of every request's beams
  fork     beams take over their parents' pages: block table rows, and copies of partly filled pages
  copy     pages to other places in all pools of a model

Pages hold 128 positions.  A state's inputs are drawn on the GPU from the seed; lengths follow from the case alone.
"""
import math

import torch

own = False

PAGE = 128
EOS = 2


# ----------------------------------------------------------------------------- cases
def listed():
    return [
        # one user's next token, the sequence in pages: launch and latency
        {"name": "attend_1x1_at_700", "kind": "attend", "batch": 1, "tokens": 1, "past": 700, "heads": 16, "kv_heads": 8, "dim": 128, "ragged": False},
        # next tokens of a serving batch whose requests are of all ages
        {"name": "attend_32x1_ragged", "kind": "attend", "batch": 32, "tokens": 1, "past": 6000, "heads": 16, "kv_heads": 8, "dim": 128, "ragged": True},
        # drafts being verified, a few tokens each
        {"name": "attend_8x9_ragged", "kind": "attend", "batch": 8, "tokens": 9, "past": 9001, "heads": 32, "kv_heads": 8, "dim": 128, "ragged": True},
        # a batch in which short questions, portions of prompts and answers meet, small heads without groups
        {"name": "attend_12x700_mixed", "kind": "attend", "batch": 12, "tokens": 700, "past": 1500, "heads": 12, "kv_heads": 12, "dim": 64, "ragged": True},
        # a portion of one long document
        {"name": "attend_1x512_at_16384", "kind": "attend", "batch": 1, "tokens": 512, "past": 16384, "heads": 16, "kv_heads": 8, "dim": 128, "ragged": False},
        # portions of several long prompts, the 2560-wide heads
        {"name": "attend_4x2048_at_6144", "kind": "attend", "batch": 4, "tokens": 2048, "past": 6144, "heads": 32, "kv_heads": 8, "dim": 128, "ragged": False},
        # one request with four beams over the large vocabulary, and a batch of them
        {"name": "beams_1x4_151936", "kind": "beams", "batch": 1, "beams": 4, "vocab": 151936},
        {"name": "beams_32x4_151936", "kind": "beams", "batch": 32, "beams": 4, "vocab": 151936},
        # a step of one request in the middle of a page, all layers of the 0.6B model; and a batch with eight beams
        {"name": "fork_1x4_at_333", "kind": "fork", "batch": 1, "beams": 4, "length": 333, "layers": 28, "kv_heads": 8, "dim": 128},
        {"name": "fork_16x8_at_1000", "kind": "fork", "batch": 16, "beams": 8, "length": 1000, "layers": 9, "kv_heads": 8, "dim": 128},
        # a prompt's two pages for a second reader, and a pool whose holes are closed
        {"name": "copy_2_pages", "kind": "copy", "pages": 2, "layers": 28, "kv_heads": 8, "dim": 128},
        {"name": "copy_300_pages", "kind": "copy", "pages": 300, "layers": 9, "kv_heads": 8, "dim": 128},
    ]


def _between(rng, lo, hi):
    """A whole number from lo to hi, even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "beams", "beams", "fork", "copy"])
    if kind == "attend":
        most = work(listed()[5])["flops"]
        while True:
            kv = rng.choice([1, 2, 4, 8, 12])
            c = {"kind": kind, "batch": _between(rng, 1, 48), "tokens": _between(rng, 1, 2048), "past": _between(rng, 1, 20000), "heads": kv * rng.choice([1, 2, 3, 4, 8]),
                 "kv_heads": kv, "dim": rng.choice([64, 128]), "ragged": rng.random() < 0.6}
            # (the plain form's scores are a dense block of every sequence's longest lengths)
            if work(c)["flops"] <= most and c["heads"] * c["batch"] * c["tokens"] * (c["past"] + c["tokens"]) <= 2e9:
                return c
    if kind == "beams":
        beams = _between(rng, 1, 16)
        return {"kind": kind, "batch": _between(rng, 1, max(1, 128 // beams)), "beams": beams, "vocab": _between(rng, 1000, 151936)}
    heads = {"layers": rng.choice([2, 4, 6, 9]), "kv_heads": rng.choice([1, 2, 4, 8]), "dim": rng.choice([64, 128])}
    if kind == "fork":
        return {"kind": kind, "batch": _between(rng, 1, 16), "beams": _between(rng, 2, 8), "length": _between(rng, 1, 2000), **heads}
    return {"kind": kind, "pages": _between(rng, 1, 300), **heads}


def _lengths(c):
    """New tokens and keys of every sequence: the first is the longest, the others are spread evenly below it."""
    new, keys = [], []
    for i in range(c["batch"]):
        f, g = ((i * 0.6180339887498949) % 1.0, (i * 0.7548776662466927) % 1.0) if c["ragged"] and i else (1.0, 1.0)
        n = max(1, math.ceil(c["tokens"] * f))
        new.append(n)
        keys.append(n + int(c["past"] * g))
    return new, keys


def work(case):
    c = case
    if c["kind"] == "attend":
        new, keys = _lengths(c)
        pairs = sum(n * (k - n) + n * (n + 1) // 2 for n, k in zip(new, keys))
        return {"bytes": 2.0 * c["dim"] * (2 * sum(new) * c["heads"] + 2 * sum(keys) * c["kv_heads"]), "flops": 4.0 * c["dim"] * c["heads"] * pairs}
    if c["kind"] == "beams":
        n = float(c["batch"] * c["beams"] * c["vocab"])
        return {"bytes": 4.0 * n, "flops": 4.0 * n}
    rows = 2.0 * c["layers"] * c["kv_heads"] * c["dim"] * 2          # bytes of one position in all pools
    if c["kind"] == "fork":
        moved = c["batch"] * (c["beams"] // 2) * (c["length"] % PAGE)
        table = 4.0 * c["batch"] * c["beams"] * (c["length"] // PAGE + 1)
        return {"bytes": 2.0 * rows * moved + 2.0 * table, "flops": 0.0}
    return {"bytes": 2.0 * rows * c["pages"] * PAGE, "flops": 0.0}


# ----------------------------------------------------------------------------- inputs
def _normal(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _attend_inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    new, keys = _lengths(c)
    pages = [-(-k // PAGE) for k in keys]
    total = sum(pages) + 3
    order = torch.randperm(total, generator=g, device="cuda").int()
    table = torch.zeros(c["batch"], max(pages), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    starts = torch.tensor([0] + new, dtype=torch.int64).cumsum(0)
    pools = [_normal(g, total, c["kv_heads"], PAGE, c["dim"], dtype=torch.bfloat16) for _ in range(2)]
    # rows that are normed as a model's queries and keys are, some pairs far more alike than others
    return {"q": _normal(g, sum(new), c["heads"], c["dim"], std=1.5, dtype=torch.bfloat16), "k": pools[0], "v": pools[1], "table": table,
            "start": starts.int().cuda(), "keys": torch.tensor(keys, dtype=torch.int32, device="cuda"), "scale": c["dim"] ** -0.5}


def _beams_inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, K, V = c["batch"], c["beams"], c["vocab"]
    logits = _normal(g, B, K, V, std=2.5)
    # some beams are about to end
    logits[:, :, EOS] += 9.0 * (torch.rand(B, K, generator=g, device="cuda") < 0.3)
    scores = -20.0 * torch.rand(B, 1, generator=g, device="cuda") - 3.0 * torch.rand(B, K, generator=g, device="cuda")
    return {"logits": logits, "scores": scores}


def _pools(c, pages, g):
    return _normal(g, 2 * c["layers"], pages, c["kv_heads"], PAGE, c["dim"], dtype=torch.bfloat16)


def _fork_inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, K, n = c["batch"], c["beams"], c["length"]
    whole = n // PAGE
    # whole pages are a request's common ones; every beam has a last page and a spare one of its own
    pages = B * whole + 2 * B * K
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.zeros(B * K, whole + 2, dtype=torch.int32, device="cuda")
    table[:, :whole] = order[:B * whole].view(B, 1, whole).expand(B, K, whole).reshape(B * K, whole)
    table[:, whole] = order[B * whole:B * whole + B * K]
    # half of the beams go on, each with as many children as chance gives it beyond the first
    live = torch.rand(B, K, generator=g, device="cuda").argsort(1)[:, :K - K // 2]
    more = live.gather(1, torch.randint(0, K - K // 2, (B, K // 2), generator=g, device="cuda"))
    parents = torch.cat([live, more], 1).gather(1, torch.rand(B, K, generator=g, device="cuda").argsort(1))
    return {"pools": _pools(c, pages, g), "table": table, "spare": order[B * whole + B * K:].clone(), "parents": parents.int().contiguous(),
            "length": torch.tensor([n], dtype=torch.int32, device="cuda")}


def _copy_inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = 2 * c["pages"] + 3
    order = torch.randperm(pages, generator=g, device="cuda").int()
    return {"pools": _pools(c, pages, g), "src": order[:c["pages"]].clone(), "dst": order[c["pages"]:2 * c["pages"]].clone()}


_INPUTS = {"attend": _attend_inputs, "beams": _beams_inputs, "fork": _fork_inputs, "copy": _copy_inputs}


def prepare(case, seed):
    s = _INPUTS[case["kind"]](case, int(seed))
    s["case"] = dict(case)
    if own:
        _place(s)
    return s


# ----------------------------------------------------------------------------- the framework's own tensors
class _Seen:
    """A tensor of the framework as torch sees it."""

    def __init__(self, t):
        kind, size = {"float32": ("<f4", 4), "bfloat16": ("<i2", 2), "int64": ("<i8", 8), "int32": ("<i4", 4)}[t.dtype]
        self.kept = t
        self.__cuda_array_interface__ = {"shape": tuple(t.shape), "typestr": kind, "data": (t._handle.storage.device_ptr() + t.offset * size, False),
                                         "strides": None, "version": 2}


def _seen(t):
    x = torch.as_tensor(_Seen(t), device="cuda")
    return x.view(torch.bfloat16) if t.dtype == "bfloat16" else x


def _place(s):
    """Puts a state's inputs into tensors of the framework, with the outputs that a program keeps from call to call."""
    import kandle_b200
    from kandle_b200 import core, paged

    backend = kandle_b200.init(0)
    c, d = s["case"], {}
    for name in [n for n, x in s.items() if isinstance(x, torch.Tensor)]:
        x = s.pop(name)
        d[name] = core.empty(tuple(x.shape), str(x.dtype).split(".")[1])
        backend.synchronize()
        _seen(d[name]).copy_(x)
    if c["kind"] == "attend":
        d["out"] = core.empty(d["q"].shape, "bfloat16")
        s["most"] = max(_lengths(c)[0])
    elif c["kind"] == "beams":
        B, K = c["batch"], c["beams"]
        d.update(next=core.empty((B, K)), parents=core.empty((B, K), "int32"), tokens=core.empty((B, K), "int64"), ended=core.empty((B, K)))
    else:
        d["list"] = paged.Pools([d["pools"].select(0, i) for i in range(2 * c["layers"])])
    torch.cuda.synchronize()
    s["d"] = d
    s["out"] = {"attend": lambda: _seen(d["out"]), "beams": lambda: {n: _seen(d[n]) for n in ("next", "parents", "tokens", "ended")},
                "fork": lambda: {n: _seen(d[n]) for n in ("pools", "table", "spare")}, "copy": lambda: _seen(d["pools"])}[c["kind"]]()


def _run_own(s):
    from kandle_b200 import paged
    from kandle_b200.model_utils import sampling

    d, kind = s["d"], s["case"]["kind"]
    if kind == "attend":
        paged.attention(d["q"], d["k"], d["v"], d["table"], d["keys"], q_start=d["start"], max_query=s["most"], scale=s["scale"], out=d["out"])
    elif kind == "beams":
        sampling.beam_select(d["logits"], d["scores"], EOS, out=(d["next"], d["parents"], d["tokens"], d["ended"]))
    elif kind == "fork":
        paged.fork_pages(d["list"], d["parents"], d["table"], d["spare"], d["length"])
    else:
        paged.copy_pages(d["list"], d["src"], d["dst"])
    return s["out"]


# ----------------------------------------------------------------------------- plain forms
def _attend(s):
    q, start, keys = s["q"], s["start"].long(), s["keys"].long()
    H, (_, G, _, D) = q.shape[1], s["k"].shape
    B, P = s["table"].shape
    new = start[1:] - start[:-1]
    N = s["case"]["tokens"]
    i, j = torch.arange(N, device=q.device), torch.arange(P * PAGE, device=q.device)
    rows = (start[:-1, None] + i).clamp(max=q.shape[0] - 1)
    qp = q[rows].float().view(B, N, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, -1, D)
    held = (j < keys[:, None]).view(B, 1, -1, 1)
    k, v = (torch.where(held, x[s["table"].long()].permute(0, 2, 1, 3, 4).reshape(B, G, P * PAGE, D).float(), 0.0) for x in (s["k"], s["v"]))
    seen = (j <= ((keys - new)[:, None] + i)[:, :, None]) & (i < new[:, None])[:, :, None]
    seen = seen[:, None, None].expand(B, 1, H // G, N, P * PAGE).reshape(B, 1, -1, P * PAGE)
    p = torch.where(seen, torch.matmul(qp, k.transpose(-1, -2)) * s["scale"], -math.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True).clamp(min=-1e30))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    o = o.view(B, G, H // G, N, D).permute(0, 3, 1, 2, 4).reshape(B, N, H, D)
    token = torch.arange(q.shape[0], device=q.device)
    b = torch.searchsorted(start[1:], token, right=True)
    return o[b, token - start[b]].to(q.dtype)


def _beams(s):
    x = s["logits"].double()
    B, K, V = x.shape
    top = x.amax(-1, keepdim=True)
    v = x - (top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))) + s["scores"].double()[:, :, None]
    v, at = torch.sort(torch.nan_to_num(v, nan=-math.inf).view(B, -1), dim=1, descending=True, stable=True)
    v, at = v[:, :2 * K], at[:, :2 * K]
    end = at % V == EOS
    first = torch.sort(end, dim=1, stable=True)[1][:, :K]
    keep, kept = at.gather(1, first), v.gather(1, first)
    place = torch.where(end[:, :K], torch.div(at[:, :K], V, rounding_mode="floor"), K)
    ended = torch.full((B, K + 1), -math.inf, dtype=v.dtype, device=v.device).scatter_(1, place, v[:, :K])[:, :K]
    return {"next": kept.float(), "parents": torch.div(keep, V, rounding_mode="floor").int(), "tokens": keep % V, "ended": ended.float()}


def _fork(s):
    pools, table, spare, parents = s["pools"], s["table"], s["spare"].long(), s["parents"].long()
    B, K = parents.shape
    whole, rest = s["case"]["length"] // PAGE, s["case"]["length"] % PAGE
    row = torch.arange(B, device=table.device)[:, None] * K + parents
    held = whole + (rest > 0)                     # columns behind the last held page are every row's own
    old = table[row.view(-1), :held]
    if rest:
        tail = table[:, whole].long()
        same = parents[:, :, None] == parents[:, None, :]
        again = torch.tril(same, -1).any(-1)                                       # not the first child of its parent
        dead = ~(parents[:, :, None] == torch.arange(K, device=table.device)).any(1)
        take, give = again.view(-1).nonzero()[:, 0], dead.view(-1).nonzero()[:, 0]   # as many of each in every request, in order
        pools[:, spare[take], :, :rest] = pools[:, tail[row.view(-1)[take]], :, :rest]
        old[take, whole] = spare[take].int()
        spare = spare.clone()
        spare[take] = tail[give]
    table[:, :held] = old
    s["spare"].copy_(spare)
    return {"pools": pools, "table": table, "spare": s["spare"]}


def _copy(s):
    s["pools"][:, s["dst"].long()] = s["pools"][:, s["src"].long()]
    return s["pools"]


def run(state):
    if own:
        return _run_own(state)
    return {"attend": _attend, "beams": _beams, "fork": _fork, "copy": _copy}[state["case"]["kind"]](state)


# ----------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    c = case
    s = _INPUTS[c["kind"]](c, int(seed))
    if c["kind"] == "attend":
        new, keys = _lengths(c)
        group, done = c["heads"] // c["kv_heads"], []
        for b, (n, m) in enumerate(zip(new, keys)):
            at = int(s["start"][b])
            pages = s["table"][b, :-(-m // PAGE)].tolist()
            k, v = (torch.cat([x[p] for p in pages], 1)[:, :m].double() for x in (s["k"], s["v"]))
            parts = []
            for a in range(0, n, 256):
                e = min(n, a + 256)
                x = torch.einsum("ngrd,gmd->grnm", s["q"][at + a:at + e].double().view(e - a, c["kv_heads"], group, -1), k) * s["scale"]
                late = torch.arange(m, device="cuda")[None] > torch.arange(m - n + a, m - n + e, device="cuda")[:, None]
                parts.append(torch.einsum("grnm,gmd->ngrd", torch.softmax(x.masked_fill_(late, -math.inf), -1), v).reshape(e - a, c["heads"], -1))
            done += parts
        return torch.cat(done)
    if c["kind"] == "beams":
        B, K, V = c["batch"], c["beams"], c["vocab"]
        scored, out = torch.log_softmax(s["logits"].double(), -1) + s["scores"].double()[..., None], {"next": [], "ended": []}
        for b in range(B):
            best = torch.topk(scored[b].reshape(-1), 2 * K)
            pairs = list(zip(best.values.tolist(), best.indices.tolist()))
            out["next"].append([v for v, i in pairs if i % V != EOS][:K])
            ends = {i // V: v for v, i in pairs[:K] if i % V == EOS}
            out["ended"].append([ends.get(j, -math.inf) for j in range(K)])
        return {"next": torch.tensor(out["next"], dtype=torch.float64), "ended": torch.tensor(out["ended"], dtype=torch.float64), "parents": None, "tokens": None}
    if c["kind"] == "copy":
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            s["pools"][:, b] = s["pools"][:, a]
        return s["pools"].double()
    K, at, rest = c["beams"], c["length"] // PAGE, c["length"] % PAGE
    for b in range(c["batch"]):
        for r, parent in enumerate(s["parents"][b].tolist()):
            if rest and parent in s["parents"][b, :r].tolist():
                s["pools"][:, int(s["spare"][b * K + r]), :, :rest] = s["pools"][:, int(s["table"][b * K + parent, at]), :, :rest]
    return {"pools": s["pools"].double(), "table": None, "spare": None}
