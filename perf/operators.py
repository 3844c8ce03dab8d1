"""The operators of the answer step over retrieved passages, as cases with their plain forms.

A language model that answers from retrieved passages keeps its keys and values in a paged cache. One step
of it runs, in each layer, `kv_append` (norm and rotate the step's queries and keys, store keys and values in
their pages) and `paged_attention` (the step's tokens over the cache), and at its end `sample` (the next
token of every sequence). Each case below is one call of one of the three. Where `own` is false the call is
computed by elementary torch operations in 32 bits, else by this repository's kernels.
"""

import itertools
import math
import random
import sys
from pathlib import Path

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_UNITS = float(1 << 40)  # a sampling weight counts units of 2^-40 of the largest, so sums are exact


def _zc():
    package = str(Path(__file__).resolve().parents[1] / "zero-copy-gpu-vector-search-re-ranking-engine_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import zcgvs_sm100

    return zcgvs_sm100


# ------------------------------------------------------------------------------------------------
# Cases
# ------------------------------------------------------------------------------------------------
def _append(name, **kw):
    case = {"op": "append", "type": "bf16", "sequences": 1, "new": 1, "kv": 512, "ragged": 0, "page": 16, "q_heads": 32,
            "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": False, "norm": True, "heads_first": False}
    return {**({"name": name} if name else {}), **case, **kw}


def _attend(name, **kw):
    case = {"op": "attend", "type": "bf16", "sequences": 1, "new": 1, "kv": 512, "ragged": 0, "page": 16, "q_heads": 32,
            "kv_heads": 8, "dim": 128, "causal": True, "window": 0, "heads_first": False}
    return {**({"name": name} if name else {}), **case, **kw}


def _sampling(name, **kw):
    case = {"op": "sample", "type": "f32", "rows": 1, "vocab": 32000, "temperature": 0.8, "top_k": 0, "top_p": 1.0, "min_p": 0.0,
            "spread": 2.5}
    return {**({"name": name} if name else {}), **case, **kw}


def listed():
    return [
        # One answer being decoded: a single token through one layer, where the call's latency is all.
        _append("append, one token", kv=1500),
        # A full decode batch of a server, ragged lengths, fp16, heads-first pages, partial interleaved rotation.
        _append("append, 200 decoding", sequences=200, kv=3000, ragged=3, type="f16", heads_first=True, rotary=64, interleaved=True,
                norm=False, page=32),
        # The passages of several requests being read: long ragged chunks.
        _append("append, passages", sequences=7, new=4096, kv=6000, ragged=5, page=64),
        # One answer being decoded over a few short passages.
        _attend("decode, one short", kv=777),
        # A server's decode batch: ragged lengths over a few thousand tokens each.
        _attend("decode, 96 ragged", sequences=96, kv=6000, ragged=7),
        # One answer over a whole collection held in the cache.
        _attend("decode, one long", kv=131000, page=64),
        # The next chunk of a long prompt over what is already in the cache.
        _attend("chunk of 512 over 16K", new=512, kv=16384, page=64),
        # Whole prompts read at once.
        _attend("prompts, 2 of 4096", sequences=2, new=4096, kv=4096, page=128),
        # Chunks and decoding tokens in one batch, fp16, smaller heads, a window, heads-first pages.
        _attend("mixed, window", sequences=24, new=300, kv=5000, ragged=11, type="f16", q_heads=24, kv_heads=4, dim=64, window=1024,
                heads_first=True),
        # One answer's next token from a small vocabulary.
        _sampling("sample, one row", top_k=50, top_p=0.95),
        # A decode batch with the common filters.
        _sampling("sample, 96 rows", rows=96, vocab=128256, top_k=64, top_p=0.9, min_p=0.02),
        # A large batch of half-precision logits, odd vocabulary, nucleus over the whole of it.
        _sampling("sample, 320 rows", rows=320, vocab=151669, type="bf16", temperature=1.1, top_p=0.92, spread=3.0),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "sample"])
    if op == "sample":
        rows = _log(rng, 1, 320)
        vocab = _log(rng, 1000, 160000)
        return _sampling(None, rows=rows, vocab=vocab, type=rng.choice(["f32", "f16", "bf16"]),
                         temperature=round(rng.uniform(0.3, 1.5), 2), top_k=rng.choice([0, 1, rng.randint(2, 100), rng.randint(100, 900)]),
                         top_p=rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]), min_p=rng.choice([0.0, round(rng.uniform(0.005, 0.2), 3)]),
                         spread=round(rng.uniform(1.0, 4.0), 2))
    dim = rng.choice([64, 80, 96, 128, 128])
    kv_heads, group = rng.choice([(1, 8), (2, 7), (4, 6), (8, 4), (8, 1), (5, 3), (8, 8)])
    common = {"type": rng.choice(["f16", "bf16"]), "page": rng.choice([8, 16, 32, 64, 128]), "kv_heads": kv_heads, "q_heads": kv_heads * group,
              "dim": dim, "ragged": rng.randint(1, 999), "heads_first": rng.random() < 0.3}
    if op == "append":
        sequences = _log(rng, 1, 200)
        new = 1 if rng.random() < 0.4 else _log(rng, 1, max(1, 20000 // sequences))
        return _append(None, sequences=sequences, new=new, kv=new + _log(rng, 1, 2000), rotary=rng.choice([dim, dim // 2]),
                       interleaved=rng.random() < 0.5, norm=rng.random() < 0.5, **common)
    if rng.random() < 0.5:
        sequences, new = _log(rng, 1, 96), rng.choice([1, 1, 1, 2, 5])
        kv = _log(rng, 16, min(100000, 500000 // sequences))
    else:
        sequences, new = _log(rng, 1, 12), _log(rng, 6, 2048)
        scores = sequences * new * kv_heads * group  # for every cached token
        kv = new + _log(rng, 8, max(16, min(20000, (1 << 29) // scores)))
    return _attend(None, sequences=sequences, new=new, kv=kv, causal=rng.random() < 0.85, window=rng.choice([0, 0, 0, _log(rng, 8, 4000)]), **common)


def _lengths(case):
    """(new tokens, cached tokens with them) of every sequence: the largest first, then spread below it; with
    three ragged sequences or more the second is an idle one, without a new token."""
    n, new, kv = case["sequences"], case["new"], case["kv"]
    if not case["ragged"]:
        return [new] * n, [kv] * n
    rng = random.Random(case["ragged"])
    news = [new] + [rng.randint(max(1, new // 8), new) for _ in range(n - 1)]
    kvs = [kv] + [max(a, rng.randint(max(1, kv // 4), kv)) for a in news[1:]]
    if n >= 3:
        news[1] = 0
    return news, kvs


# ------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------
def _paged(case, generator):
    """The cache and the step's description, as a serving program holds them."""
    kind, page = _TYPES[case["type"]], case["page"]
    news, kvs = _lengths(case)
    per = [-(-k // page) for k in kvs]
    pages = sum(per) + 3
    shape = (pages, case["kv_heads"], page, case["dim"]) if case["heads_first"] else (pages, page, case["kv_heads"], case["dim"])
    fresh = case["op"] == "append"
    k, v = (torch.zeros(shape, dtype=kind, device="cuda") if fresh else torch.randn(shape, dtype=kind, device="cuda", generator=generator)
            for _ in range(2))
    if case["heads_first"]:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    table = torch.zeros((len(kvs), max(per)), dtype=torch.int32)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(generator.initial_seed())).to(torch.int32)
    table[torch.arange(max(per)) < torch.tensor(per)[:, None]] = order[:sum(per)]
    starts = [0, *itertools.accumulate(news)]
    state = {"case": case, "k_cache": k, "v_cache": v, "table": table.cuda(), "starts": torch.tensor(starts, dtype=torch.int32).cuda(),
             "lengths": torch.tensor(kvs, dtype=torch.int32).cuda(), "tokens": starts[-1], "max_new": max(news), "max_kv": max(kvs)}
    if own:
        zc = _zc()
        state["cache"] = zc.PagedKvCache(k, v)
        state["batch"] = zc.StepBatch(state["starts"], state["lengths"], state["table"], tokens=state["tokens"],
                                      max_new=state["max_new"], max_length=state["max_kv"])
        state["workspace"] = zc.Workspace()
    return state


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = _TYPES[case["type"]]
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        logits = torch.randn((rows, vocab), device="cuda", generator=g) * case["spread"]
        # A few tokens stand out, as where the text leaves little choice.
        likely = torch.randint(vocab, (rows, 24), device="cuda", generator=g)
        logits.scatter_(1, likely, case["spread"] * (3 + torch.randn((rows, 24), device="cuda", generator=g)))
        logits += torch.randn((rows, 1), device="cuda", generator=g) * 3
        uniforms = torch.rand(rows, device="cuda", generator=g)
        # The requests of a batch have their own settings: around the case's, and every eighth one is greedy.
        row = torch.arange(rows, device="cuda")
        temperature = case["temperature"] * (1 + 0.1 * (row % 3))
        temperature = torch.where(row % 8 == 7, torch.zeros_like(temperature), temperature)
        top_k = (case["top_k"] + (row % 4) * (1 if case["top_k"] else 0)).to(torch.int32)
        return {"case": case, "logits": logits.to(kind), "uniforms": uniforms, "temperature": temperature, "top_k": top_k,
                "top_p": torch.full((rows,), case["top_p"], device="cuda"), "min_p": torch.full((rows,), case["min_p"], device="cuda")}
    state = _paged(case, g)
    heads, d = case["q_heads"], case["dim"]
    if case["op"] == "attend":
        state["q"] = torch.randn((state["tokens"], heads, d), dtype=kind, device="cuda", generator=g) * 2
        state["scale"] = 1 / math.sqrt(d)
        return state
    # The three parts of one projection's rows, as views of it.
    width = heads + 2 * case["kv_heads"]
    rows = torch.randn((state["tokens"], width, d), dtype=kind, device="cuda", generator=g)
    state["q"], state["k"], state["v"] = rows[:, :heads], rows[:, heads:heads + case["kv_heads"]], rows[:, heads + case["kv_heads"]:]
    if case["norm"]:
        state["q_norm"], state["k_norm"] = ((1 + 0.2 * torch.randn(d, device="cuda", generator=g)).to(kind) for _ in range(2))
    else:
        state["q_norm"] = state["k_norm"] = None
    half = case["rotary"] // 2
    angle = torch.arange(case["kv"], dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    state["rotary"] = torch.cat([angle.cos(), angle.sin()], 1).float().cuda()
    return state


# ------------------------------------------------------------------------------------------------
# One call
# ------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        zc = _zc()
        if op == "append":
            q = zc.kv_append(state["cache"], state["batch"], state["q"], state["k"], state["v"], rotary=state["rotary"],
                             interleaved=state["case"]["interleaved"], q_norm=state["q_norm"], k_norm=state["k_norm"], eps=1e-6)
            return {"q": q, "k_cache": state["k_cache"], "v_cache": state["v_cache"]}
        if op == "attend":
            out, lse = zc.paged_attention(state["cache"], state["batch"], state["q"], scale=state["scale"], causal=state["case"]["causal"],
                                          window=state["case"]["window"], return_lse=True, workspace=state["workspace"])
            return {"out": out, "lse": lse}
        token, logprob = zc.sample(state["logits"], state["uniforms"], temperature=state["temperature"], top_k=state["top_k"],
                                   top_p=state["top_p"], min_p=state["min_p"])
        return {"token": token, "logprob": logprob}
    return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[op](state)


def _tokens_of(state):
    """Of every token: its sequence, its place among the sequence's new ones, and its position in the cache."""
    starts, lengths = state["starts"].long(), state["lengths"].long()
    news = starts[1:] - starts[:-1]
    seq = torch.repeat_interleave(torch.arange(len(news), device="cuda"), news, output_size=state["tokens"])
    place = torch.arange(state["tokens"], device="cuda") - starts[seq]
    return seq, place, lengths[seq] - news[seq] + place


def _rotated(x, weight, angles, rotary, interleaved):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.float()
    half = rotary // 2
    cos, sin = angles[:, None, :half], angles[:, None, half:]
    a, b = (x[..., 0:rotary:2], x[..., 1:rotary:2]) if interleaved else (x[..., :half], x[..., half:rotary])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., rotary:]], -1)


def _plain_append(state):
    case = state["case"]
    seq, _, position = _tokens_of(state)
    angles = state["rotary"][position]
    page, slot = state["table"][seq, position // case["page"]].long(), position % case["page"]
    kind = state["q"].dtype
    q = _rotated(state["q"], state["q_norm"], angles, case["rotary"], case["interleaved"]).to(kind)
    state["k_cache"][page, slot] = _rotated(state["k"], state["k_norm"], angles, case["rotary"], case["interleaved"]).to(kind)
    state["v_cache"][page, slot] = state["v"]
    return {"q": q, "k_cache": state["k_cache"], "v_cache": state["v_cache"]}


def _plain_attend(state):
    case = state["case"]
    n, heads, groups, d, most = case["sequences"], case["kv_heads"], case["q_heads"] // case["kv_heads"], case["dim"], state["max_new"]
    seq, place, position = _tokens_of(state)
    at = torch.arange(state["max_kv"], device="cuda")
    page, slot = state["table"].long()[:, at // case["page"]], at % case["page"]
    k = state["k_cache"][page, slot].float().permute(0, 2, 3, 1)                     # [sequence, head, d, kv]
    v = state["v_cache"][page, slot].float().permute(0, 2, 1, 3)                     # [sequence, head, kv, d]
    q = torch.zeros((n, most, heads, groups, d), device="cuda")
    q[seq, place] = state["q"].float().view(-1, heads, groups, d)
    where = torch.full((n, most), -1, device="cuda")
    where[seq, place] = position
    seen = at < state["lengths"].long()[:, None, None]
    seen = seen & (where >= 0)[:, :, None]
    if case["causal"]:
        seen = seen & (at <= where[:, :, None])
    if case["window"]:
        seen = seen & (at > where[:, :, None] - case["window"])
    s = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(n, heads, groups * most, d), k).view(n, heads, groups, most, -1)
    s.mul_(state["scale"]).masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(n, heads, groups * most, -1), v).view(n, heads, groups, most, d) / torch.where(total == 0, 1.0, total)
    lse = (total.log() + top)[..., 0]
    out, lse = out.permute(0, 3, 1, 2, 4)[seq, place], lse.permute(0, 3, 1, 2)[seq, place]
    return {"out": out.reshape(-1, case["q_heads"], d).to(state["q"].dtype), "lse": lse.reshape(-1, case["q_heads"])}


def _plain_sample(state):
    x = state["logits"].float()
    rows, vocab = x.shape
    value, order = torch.sort(x, dim=1, descending=True, stable=True)
    greedy = (state["temperature"] <= 0)[:, None]
    e = torch.exp((value - value[:, :1]) / torch.where(greedy, 1.0, state["temperature"][:, None]))
    units = (e * _UNITS).round().to(torch.int64)
    place = torch.arange(vocab, device="cuda")
    top_k = state["top_k"].long()[:, None]
    keep = (place < torch.where(top_k <= 0, vocab, top_k)) & (e >= state["min_p"][:, None]) & (~greedy | (place == 0))
    among = torch.where(place < torch.where(top_k <= 0, vocab, top_k), units, 0)
    before = among.cumsum(1) - among
    top_p = state["top_p"].double()[:, None]
    keep &= (top_p >= 1) | (before.double() < top_p * among.sum(1, keepdim=True).double()) | (place == 0)
    units = torch.where(keep, units, 0)
    total = units.sum(1)
    by_index = torch.zeros_like(units).scatter_(1, order, units).cumsum(1)
    target = torch.minimum((state["uniforms"].double() * total.double()).floor().long(), total - 1)
    token = torch.searchsorted(by_index, target[:, None], right=True)
    chosen = by_index.gather(1, token) - torch.where(token > 0, by_index.gather(1, (token - 1).clamp(min=0)), 0)
    return {"token": token[:, 0].to(torch.int32), "logprob": torch.log(chosen[:, 0].double() / total.double()).float()}


# ------------------------------------------------------------------------------------------------
# What a call cannot do without, and its outputs in 64 bits
# ------------------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * 28, "flops": 4 * n}
    news, kvs = _lengths(case)
    tokens, d = sum(news), case["dim"]
    if case["op"] == "append":
        values = tokens * (case["q_heads"] + 2 * case["kv_heads"]) * d
        return {"bytes": 2 * values * size + 4 * tokens * case["rotary"], "flops": 8 * values}
    pairs = keys = 0  # pairs of a row and a key it sees, and keys that any row of their sequence sees, of one head
    for new, kv in zip(news, kvs):
        low = [max(0, p - case["window"] + 1) if case["window"] else 0 for p in range(kv - new, kv)]
        pairs += sum((p + 1 if case["causal"] else kv) - a for p, a in zip(range(kv - new, kv), low))
        keys += kv - low[0] if new else 0
    return {"bytes": (2 * keys * case["kv_heads"] * d + 2 * tokens * case["q_heads"] * d) * size + 4 * tokens * case["q_heads"],
            "flops": 4 * pairs * case["q_heads"] * d}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "sample":  # the chosen token's logarithm, row by row
        logprob = torch.zeros(case["rows"], dtype=torch.float64)
        for r, (t, n, p, low, u) in enumerate(zip(*(state[name].tolist() for name in ("temperature", "top_k", "top_p", "min_p", "uniforms")))):
            if t <= 0:
                continue
            x = state["logits"][r].double()
            e = torch.exp((x - x.max()) / t)
            ranked = torch.argsort(x, descending=True, stable=True)
            ranked = ranked[:n] if n > 0 else ranked
            mass = e[ranked]
            before = mass.cumsum(0) - mass
            kept = ranked[((before < p * mass.sum()) | (p >= 1)) & (mass >= low)].sort().values
            up_to = e[kept].cumsum(0)
            at = int((up_to <= u * up_to[-1]).sum().clamp(max=len(kept) - 1))
            logprob[r] = torch.log(e[kept[at]] / up_to[-1])
        return {"token": None, "logprob": logprob.cuda()}
    news, kvs = _lengths(case)
    page, table = case["page"], state["table"].long().cpu()
    groups = case["q_heads"] // case["kv_heads"]
    if case["op"] == "append":
        half = case["rotary"] // 2
        k_cache, v_cache = state["k_cache"].double(), state["v_cache"].double()
        q_out = torch.empty(state["q"].shape, dtype=torch.float64, device="cuda")
        at = 0
        for s, (new, kv) in enumerate(zip(news, kvs)):
            position = torch.arange(kv - new, kv)
            where = table[s, position // page].cuda(), (position % page).cuda()
            turn = torch.complex(state["rotary"][position.cuda(), :half].double(), state["rotary"][position.cuda(), half:].double())[:, None]

            def made(x, w):
                x = x[at:at + new].double()
                if w is not None:
                    x = w.double() * x / torch.sqrt(x.square().sum(-1, keepdim=True) / case["dim"] + 1e-6)
                x = x.clone()
                first, second = (slice(0, case["rotary"], 2), slice(1, case["rotary"], 2)) if case["interleaved"] else (
                    slice(0, half), slice(half, case["rotary"]))
                z = torch.complex(x[..., first], x[..., second]) * turn
                x[..., first], x[..., second] = z.real, z.imag
                return x

            q_out[at:at + new] = made(state["q"], state["q_norm"])
            k_cache[where] = made(state["k"], state["k_norm"])
            v_cache[where] = state["v"][at:at + new].double()
            at += new
        return {"q": q_out, "k_cache": k_cache, "v_cache": v_cache}
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(state["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    at = 0
    for s, (new, kv) in enumerate(zip(news, kvs)):
        position = torch.arange(kv)
        where = table[s, position // page].cuda(), (position % page).cuda()
        j = position.cuda()
        k, v = state["k_cache"][where].double(), state["v_cache"][where].double()
        step = max(1, (1 << 27) // max(1, kv * groups))  # rows of scores at a time
        for a in range(0, new, step):
            b = min(new, a + step)
            i = (kv - new + torch.arange(a, b, device="cuda"))[:, None]
            hidden = torch.zeros((b - a, kv), dtype=torch.bool, device="cuda")
            if case["causal"]:
                hidden |= j > i
            if case["window"]:
                hidden |= j <= i - case["window"]
            for h in range(case["kv_heads"]):
                of = slice(h * groups, (h + 1) * groups)
                score = torch.einsum("tgd,jd->tgj", state["q"][at + a:at + b, of].double(), k[:, h]) * state["scale"]
                score = score.masked_fill(hidden[:, None], -math.inf)
                lse[at + a:at + b, of] = torch.logsumexp(score, -1)
                share = torch.nan_to_num(torch.softmax(score, -1))
                out[at + a:at + b, of] = torch.einsum("tgj,jd->tgd", share, v[:, h])
        at += new
    return {"out": out, "lse": lse}
