"""GPU: the operators together: the example's search, chunked reading and decoding, and a decoding step replayed from
a CUDA graph with lengths that move on the device."""

from __future__ import annotations

import math
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import answer_step as ref  # noqa: E402


@pytest.fixture(scope="module")
def example(zc):
    sys.path.insert(0, str(ROOT / "examples"))
    import answer_from_passages

    return answer_from_passages


def _plain_logits(decoder, prompt):
    """The last token's logits in fp64, the whole prompt at once."""
    x = decoder.embedding[torch.tensor(prompt, device="cuda")].double()
    rows = (x @ decoder.qkv.double()).view(len(prompt), -1, decoder.dim)
    q, k, v = rows.split([decoder.q_heads, decoder.kv_heads, decoder.kv_heads], 1)
    angles = decoder.rotary[:len(prompt)]
    q = ref.rotate_reference(q, decoder.q_norm, 1e-6, angles, decoder.dim, False)
    k = ref.rotate_reference(k, decoder.k_norm, 1e-6, angles, decoder.dim, False)
    groups = decoder.q_heads // decoder.kv_heads
    k, v = k.repeat_interleave(groups, 1), v.repeat_interleave(groups, 1)
    p = torch.softmax(torch.einsum("hd,jhd->hj", q[-1], k) * decoder.dim**-0.5, -1)
    o = torch.einsum("hj,jhd->hd", p, v).reshape(-1)
    return (x[-1] + o @ decoder.out.double()) @ decoder.head.double()


def test_reading_in_chunks_equals_reading_at_once(example):
    """Logits after chunks of 64, of 7 and of the whole prompt against fp64: each value passes through at most 8
    roundings to bf16 (2^-9 relative each), so a logit is off by at most 2^-6 of the largest."""
    decoder = example.Decoder()
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(decoder.vocab, (n,), generator=g).tolist() for n in (250, 1, 33, 129)]
    for chunk in (64, 7, 1000):
        _, logits = example.answer(decoder, prompts, chunk=chunk, tokens=1)
        for s, prompt in enumerate(prompts):
            want = _plain_logits(decoder, prompt)
            assert float((logits[s].double() - want).abs().max()) <= 2.0**-6 * float(want.abs().max())


def test_answers_repeat_and_stay_in_the_vocabulary(example):
    decoder = example.Decoder()
    prompts = [list(range(5, 105)), list(range(400, 417))]
    first, _ = example.answer(decoder, prompts, tokens=12)
    again, _ = example.answer(decoder, prompts, tokens=12)
    assert torch.equal(first, again) and first.shape == (2, 12)
    assert bool(((first >= 0) & (first < decoder.vocab)).all())
    greedy, logits = example.answer(decoder, prompts, tokens=1, temperature=0.0)
    assert torch.equal(greedy[:, 0].long(), logits.argmax(1))


def test_retrieval_finds_the_passages(example):
    vectors = torch.randn((5000, 128), device="cuda")
    ids = example.retrieve(vectors[[3, 77]] * 2, vectors, 2)
    assert ids[:, 0].tolist() == [3, 77]


def test_a_decoding_step_replays_from_a_graph(zc):
    """Append, attention and sampling captured once; the replays follow the device's lengths and uniform numbers."""
    n, heads, kv_heads, dim, page, longest = 3, 4, 2, 64, 16, 80
    lengths = [5, 33, 70]
    cache, batch, table = ref.make_step(zc, [1] * n, [longest] * n, kv_heads=kv_heads, dim=dim, page=page, dtype=torch.float16)
    kept = ref.fill_cached(cache, table, [longest] * n)
    g = torch.Generator().manual_seed(2)
    rows = torch.randn((n, heads + 2 * kv_heads, dim), generator=g).half().cuda()
    q, k, v = rows[:, :heads], rows[:, heads:heads + kv_heads], rows[:, heads + kv_heads:]
    turn = zc.rotary_table(longest, dim)
    uniforms = torch.rand(n, device="cuda")
    ws = zc.Workspace()
    ws.get(zc.paged_attention_workspace_bytes(dim))
    out = torch.empty((n, heads, dim), dtype=torch.float16, device="cuda")
    turned = torch.empty_like(out)
    drawn = (torch.empty(n, dtype=torch.int32, device="cuda"), torch.empty(n, device="cuda"))

    def step():
        zc.kv_append(cache, batch, q, k, v, rotary=turn, out=turned)
        zc.paged_attention(cache, batch, turned, scale=0.125, out=out, workspace=ws)
        zc.sample(out.view(n, heads * dim), uniforms, out=drawn)

    batch.kv_lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for move in range(4):
        now = [x + move for x in lengths]
        batch.kv_lengths.copy_(torch.tensor(now, dtype=torch.int32))
        uniforms.uniform_()
        graph.replay()
        torch.cuda.synchronize()
        for s in range(n):
            pos = now[s] - 1
            kept[s][0][pos] = cache.keys[int(table[s, pos // page]), pos % page].double()
            kept[s][1][pos] = v[s].double()
        have = [[x[:m] for x in pair] for pair, m in zip(kept, now)]
        want, _, spread, mass = ref.attention_reference(turned, have, [1] * n, now, 0.125, True, 0)
        limit = spread * (2.0**-11 + 2.0**-13) + want.abs() * 2.0**-11 + 2.0**-25 * (1 + mass[..., None])
        assert bool(((out.double() - want).abs() <= limit * (1 + 2.0**-10)).all())
        for s in range(n):
            token, logprob = ref.sample_reference(out.view(n, -1)[s].float().cpu(), 1.0, 0, 1.0, 0.0, float(uniforms[s]))
            assert int(drawn[0][s]) == token and math.isclose(float(drawn[1][s]), logprob, rel_tol=1e-6)
    assert ws.status() == 0
