"""Helpers of the answer step's tests: ragged steps over a paged cache, and the three operators'
definitions in 64 bits (written apart from the kernels)."""

from __future__ import annotations

import math

import torch

UNIT = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}  # largest relative rounding error
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134}  # largest rounding error below the normal range


def make_step(zc, news, lengths, *, kv_heads, dim, page, dtype, seed=0, spare=3, heads_first=False, fill=None, max_new=None, extra_tokens=0):
    """A cache of random pages and a step with news[s] new of lengths[s] cached tokens per sequence. Slots that hold
    no cached token are NaN unless `fill` says otherwise."""
    g = torch.Generator().manual_seed(seed)
    per = [max(0, -(-n // page)) for n in lengths]
    pages = sum(per) + spare
    shape = (pages, kv_heads, page, dim) if heads_first else (pages, page, kv_heads, dim)
    value = math.nan if fill is None else fill
    keys, values = (torch.full(shape, value, dtype=dtype, device="cuda") for _ in range(2))
    if heads_first:
        keys, values = keys.transpose(1, 2), values.transpose(1, 2)
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(lengths), max([*per, 1])), 2**31 - 1, dtype=torch.int32)  # columns past a sequence's pages are no pages
    at = 0
    for s, n in enumerate(per):
        table[s, :n] = order[at:at + n].to(torch.int32)
        at += n
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    batch = zc.StepBatch(torch.tensor(starts, dtype=torch.int32).cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(),
                         table.cuda(), tokens=starts[-1] + extra_tokens, max_new=max_new if max_new is not None else max(news),
                         max_length=max(lengths))
    return zc.PagedKvCache(keys, values), batch, table


def slots_of(table, s, page, positions):
    """(pages, slots) of positions of sequence s."""
    return table[s, positions // page].long(), positions % page


def fill_cached(cache, table, lengths, seed=1, scale=1.0):
    """Random keys and values in every cached position; returns them per sequence in fp64 [length, heads, dim]."""
    g = torch.Generator().manual_seed(seed)
    kept = []
    for s, n in enumerate(lengths):
        at = torch.arange(max(n, 0))
        p, o = (t.cuda() for t in slots_of(table, s, cache.page_size, at))
        pair = []
        for store in (cache.keys, cache.values):
            x = (torch.randn((max(n, 0), cache.kv_heads, cache.head_dim), generator=g) * scale).to(store.dtype).cuda()
            store[p, o] = x
            pair.append(x.double())
        kept.append(pair)
    return kept


def attention_reference(q, kept, news, lengths, scale, causal, window):
    """(out, lse, bound of the rounding of weights) in fp64: bound = sum_j p_j |v_j| per element, and the part of
    weights below the normal range."""
    heads = q.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    spread = torch.zeros_like(out)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    mass = torch.zeros(q.shape[:2], dtype=torch.float64, device="cuda")  # sum_j |v_j| / sum_j exp(s_j - max)
    at = 0
    for (k, v), new, length in zip(kept, news, lengths):
        groups = heads // k.shape[1]
        for i in range(new):
            pos = length - new + i
            j = torch.arange(k.shape[0], device="cuda")
            see = torch.ones_like(j, dtype=torch.bool) if pos >= 0 else torch.zeros_like(j, dtype=torch.bool)
            if causal:
                see &= j <= pos
            if window:
                see &= j > pos - window
            if not bool(see.any()):
                continue
            ks, vs = k[see].repeat_interleave(groups, 1), v[see].repeat_interleave(groups, 1)
            s = torch.einsum("hd,jhd->hj", q[at + i].double(), ks) * scale
            p = torch.softmax(s, -1)
            out[at + i] = torch.einsum("hj,jhd->hd", p, vs)
            spread[at + i] = torch.einsum("hj,jhd->hd", p, vs.abs())
            lse[at + i] = torch.logsumexp(s, -1)
            mass[at + i] = vs.abs().amax((0, 2)) * len(ks) / torch.exp(lse[at + i] - s.amax(-1))
        at += new
    return out, lse, spread, mass


def check_attention(out, lse, reference, dtype):
    """Derived bound: a weight is rounded once (UNIT relative, TINY absolute below the normal range), the output once;
    fp32 scores of magnitude <= 50 (fp32 dot products and exp2) change a weight by less than 2^-13 relatively."""
    want, want_lse, spread, mass = reference
    u = UNIT[dtype]
    limit = spread * (u + 2.0**-13) + want.abs() * u * (1 + u) + TINY[dtype] * (1 + mass[..., None])
    off = (out.double() - want).abs()
    assert bool(torch.isfinite(out).all()), "output is not finite"
    assert bool((off <= limit).all()), f"off by {float((off - limit).max()):.3g} more than allowed"
    empty = want_lse == -math.inf
    assert bool((lse[empty] == -math.inf).all()) and bool((out[empty] == 0).all())
    assert bool(((lse.double() - want_lse)[~empty].abs() <= 2.0**-15 * (1 + want_lse[~empty].abs())).all()), "lse is off"


def rotate_reference(x, weight, eps, angles, rotary, interleaved):
    """fp64 norm and rotation of [tokens, heads, dim]; angles [tokens, rotary] (cosines, sines) or None."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    if angles is None:
        return x
    x = x.clone()
    half = rotary // 2
    turn = torch.complex(angles[:, :half].double(), angles[:, half:].double())[:, None]
    a, b = (slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else (slice(0, half), slice(half, rotary))
    z = torch.complex(x[..., a], x[..., b]) * turn
    x[..., a], x[..., b] = z.real, z.imag
    return x


def sample_reference(x, t, k, p, low, u):
    """(token, logprob) of one row of logits (fp32 values on the CPU), straight from the definition: a ranked list and
    whole-number weights as Python integers."""
    x = [float(v) for v in x]
    alive = [i for i in range(len(x)) if not math.isnan(x[i]) and x[i] != -math.inf]
    if not alive:
        return -1, -3.4028234663852886e38
    ranked = sorted(alive, key=lambda i: (-x[i], i))
    if not t > 0:
        return ranked[0], 0.0
    m = x[ranked[0]]
    xs = torch.tensor([x[i] for i in ranked], dtype=torch.float32)
    if m == math.inf:
        e = (xs == math.inf).float()
    else:
        e = torch.exp(((xs - xs[0]) / torch.tensor(t, dtype=torch.float32)).cuda()).cpu()
    w = [int(v) for v in (e.double() * 2.0**40).round().to(torch.int64)]
    n = k if 0 < k < len(ranked) else len(ranked)
    total = sum(w[:n])
    kept, before = [], 0
    for r in range(n):
        if r and p < 1 and not (float(before) < float(torch.tensor(p, dtype=torch.float32)) * float(total)):
            break
        if r == 0 or float(e[r]) >= float(torch.tensor(low, dtype=torch.float32)) or not low > 0:
            kept.append((ranked[r], w[r]))
        before += w[r]
    kept.sort()
    z = sum(v for _, v in kept)
    u = float(torch.tensor(u, dtype=torch.float32))
    u = min(u, 1 - 2.0**-24) if u >= 0 else 0.0
    target = min(math.floor(u * float(z)), z - 1)
    upto = 0
    for i, v in kept:
        upto += v
        if target < upto:
            return i, math.log(v / z)
    raise AssertionError("no token")
