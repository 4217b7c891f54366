"""Inputs and float64 answers for the operators of a paged cache and of beam search."""
import numpy as np
import torch

PAGE = 128


def bf16(a):
    return torch.tensor(np.asarray(a, np.float32)).bfloat16()


def attention_case(new, keys, heads, kv_heads, dim, seed=0, std=1.5, junk=float("nan"), spare_pages=2, table_width=None):
    """Packed queries, pools whose rows behind a sequence's keys (and whole pages that nobody owns) hold `junk`, and a table with -1 in
    entries that nobody may read."""
    rng = np.random.default_rng(seed)
    pages = [-(-k // PAGE) for k in keys]
    total = sum(pages) + spare_pages
    order = rng.permutation(total)
    width = table_width or max(max(pages), 1)
    table = np.full((len(keys), width), -1, np.int32)
    pools = [np.full((total, kv_heads, PAGE, dim), junk, np.float32) for _ in range(2)]
    at = 0
    for b, (n, k) in enumerate(zip(pages, keys)):
        table[b, :n] = order[at:at + n]
        at += n
        for i in range(n):
            rows = min(PAGE, k - i * PAGE)
            for p in pools:
                p[table[b, i], :, :rows] = rng.standard_normal((kv_heads, rows, dim))
    q = rng.standard_normal((sum(new), heads, dim)) * std
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    return {"q": bf16(q), "k": bf16(pools[0]), "v": bf16(pools[1]), "table": table, "start": start, "keys": np.asarray(keys, np.int32), "scale": dim ** -0.5}


def attention_answer(c):
    """The definition in float64, and how far a bf16 kernel may be from it.

    A probability is rounded to bf16 before it meets its value: half a step, 2^-8 of it.  A score is a sum of D products in fp32, off by D
    2^-24 of the sum of their absolute values at most, times the scale, and so is the exponent's argument, for the key and for the sum of
    all; the exponential and the sums over keys in fp32 add 2^-20 (a chain of up to 16384 keys, in 64 or more parts, is below that).  The result
    is rounded to bf16 once more."""
    q, k, v = c["q"].double(), c["k"].double(), c["v"].double()
    group = q.shape[1] // k.shape[1]
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    for b in range(len(c["keys"])):
        a, e, ctx = int(c["start"][b]), int(c["start"][b + 1]), int(c["keys"][b])
        if ctx == 0 or a == e:
            continue
        pages = [int(p) for p in c["table"][b, :-(-ctx // PAGE)]]
        kk, vv = (torch.cat([x[p] for p in pages], 1)[:, :ctx].repeat_interleave(group, 0) for x in (k, v))
        qq = q[a:e].transpose(0, 1)
        s = qq @ kk.transpose(1, 2) * c["scale"]
        size = (qq.abs() @ kk.abs().transpose(1, 2) * c["scale"]).amax(-1, keepdim=True)
        hidden = torch.arange(ctx)[None] > (ctx - (e - a) + torch.arange(e - a))[:, None]
        p = torch.exp(s.masked_fill(hidden, -np.inf) - s.masked_fill(hidden, -np.inf).amax(-1, keepdim=True).clamp(min=-1e300))
        p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
        o, mass = p @ vv, p @ vv.abs()
        off = mass * (2.0 ** -8 + 2 * q.shape[-1] * 2.0 ** -24 * size + 2.0 ** -20)
        out[a:e], tol[a:e] = o.transpose(0, 1), (off + (o.abs() + off) * 2.0 ** -8).transpose(0, 1)
    return out, tol


def beam_answer(logits, scores, eos):
    """float64: (scores, parents, tokens, ended) of every request.  Ties go to the lower beam, then the lower token; within a beam the
    logits decide."""
    B, K, V = logits.shape
    x = logits.astype(np.float64)
    with np.errstate(all="ignore"):
        m = x.max(-1)
        lse = m + np.log(np.exp(x - m[..., None]).sum(-1))
        live = np.isfinite(lse) & np.isfinite(scores)
        v = np.where(live[..., None], x - lse[..., None] + scores[..., None].astype(np.float64), -np.inf)
    out = [np.zeros((B, K), t) for t in (np.float64, np.int32, np.int64, np.float64)]
    for b in range(B):
        order = np.argsort(-v[b].reshape(-1), kind="stable")
        best = [i for i in order[:2 * K + V] if i % V != eos][:K]
        for r, i in enumerate(best):
            out[0][b, r], out[1][b, r], out[2][b, r] = v[b].reshape(-1)[i], i // V, i % V
        out[3][b] = -np.inf
        for i in order[:K]:
            if i % V == eos:
                out[3][b, i // V] = v[b].reshape(-1)[i]
    return out


def fork_answer(pools, parents, table, spare, length):
    """pools: arrays [pages, H, 128, D] (changed in place), and the new (table, spare)."""
    B, K = parents.shape
    table, spare, old = table.copy(), spare.copy(), table.copy()
    whole, rest = length // PAGE, length % PAGE
    for b in range(B):
        rows = range(b * K, (b + 1) * K)
        dead = [old[b * K + q, whole] for q in range(K) if q not in parents[b]] if rest else []
        seen = set()
        for r, p in zip(rows, parents[b]):
            table[r, :whole] = old[b * K + p, :whole]
            if not rest:
                continue
            page = old[b * K + p, whole]
            if p in seen:
                for pool in pools:
                    pool[spare[r], :, :rest] = pool[page, :, :rest]
                page, spare[r] = spare[r], dead.pop(0)
            seen.add(p)
            table[r, whole] = page
    return table, spare


def beam_rule(outputs, beams, eos, steps, power):
    """The rule of Qwen3Engine.generate_beams for one prompt, over the outputs of its steps (scores, parents, tokens, ended), each [beams].
    Returns the hypotheses (tokens, worth), best first, and the step in which the prompt was done (None: it was not)."""
    tokens, ended = [[]] * beams, []
    for step, (s, parents, new, ends) in enumerate(outputs, 1):
        ended += [(tokens[j] + [eos], ends[j] / step ** power) for j in range(beams) if np.isfinite(ends[j])]
        ended = sorted(ended, key=lambda h: -h[1])[:beams]
        tokens = [tokens[p] + [int(t)] for p, t in zip(parents, new)]
        if len(ended) == beams and s[0] / step ** power <= ended[-1][1]:
            return ended, step
        if step == steps:
            break
    return sorted(ended + [(t, x / steps ** power) for t, x in zip(tokens, s) if np.isfinite(x)], key=lambda h: -h[1])[:beams], None


def beam_search(logits_of, beams, eos, steps, power):
    """beam_rule with float64's choice.  logits_of: the beams' tokens -> logits [beams, V]."""
    def outputs():
        tokens, scores = [[]] * beams, np.full((1, beams), -np.inf)
        scores[0, 0] = 0
        while True:
            s, parents, new, ends = beam_answer(logits_of(tokens)[None], scores, eos)
            yield s[0], parents[0], new[0], ends[0]
            tokens, scores = [tokens[p] + [int(t)] for p, t in zip(parents[0], new[0])], s
    return beam_rule(outputs(), beams, eos, steps, power)
