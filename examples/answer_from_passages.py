"""Search, then answer: retrieves passages for some questions and lets a small decoder read and answer them.

The decoder is one layer with random weights, so the answers mean nothing; the steps are those of a real one:

    scan_topk          the passages of every question
    kv_append          the passages' and the question's tokens, chunk by chunk, into the paged cache
    paged_attention    over the cache: chunks of all questions in one batch, then one token each
    sample             the next token of every answer

Run it with `python examples/answer_from_passages.py` on a machine with a B200 and the built library.
"""

from __future__ import annotations

import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "zero-copy-gpu-vector-search-re-ranking-engine_b200"))

import torch  # noqa: E402
import zcgvs_sm100 as zc  # noqa: E402

PAGE = 16


class Decoder:
    """One attention layer with random bf16 weights between a token embedding and a head."""

    def __init__(self, vocab=2000, width=512, q_heads=8, kv_heads=2, dim=64, rows=4096, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weights(*shape):
            return (torch.randn(shape, device="cuda", generator=g) * shape[0] ** -0.5).to(torch.bfloat16)

        self.vocab, self.q_heads, self.kv_heads, self.dim = vocab, q_heads, kv_heads, dim
        self.embedding = weights(vocab, width) * 10
        self.qkv = weights(width, (q_heads + 2 * kv_heads) * dim)
        self.out = weights(q_heads * dim, width)
        self.head = weights(width, vocab)
        self.q_norm = torch.ones(dim, dtype=torch.bfloat16, device="cuda")
        self.k_norm = torch.ones(dim, dtype=torch.bfloat16, device="cuda")
        self.rotary = zc.rotary_table(rows, dim)

    def step(self, tokens, cache, batch, workspace):
        """Logits [tokens, vocab] of one step's tokens; their keys and values go to the cache."""
        x = self.embedding[tokens.long()]
        rows = (x @ self.qkv).view(len(tokens), -1, self.dim)
        q, k, v = rows.split([self.q_heads, self.kv_heads, self.kv_heads], 1)
        q = zc.kv_append(cache, batch, q, k, v, rotary=self.rotary, q_norm=self.q_norm, k_norm=self.k_norm, out=q)
        o = zc.paged_attention(cache, batch, q, scale=self.dim**-0.5, workspace=workspace)
        x = x + o.reshape(len(tokens), -1) @ self.out
        return (x @ self.head).float()


def new_cache(decoder, pages):
    shape = (pages, PAGE, decoder.kv_heads, decoder.dim)
    return zc.PagedKvCache(*(torch.zeros(shape, dtype=torch.bfloat16, device="cuda") for _ in range(2)))


def step_batch(news, lengths, table):
    """The step in which sequence s gets news[s] tokens and then holds lengths[s]."""
    starts = torch.zeros(len(news) + 1, dtype=torch.int32)
    starts[1:] = torch.tensor(news, dtype=torch.int32).cumsum(0)
    return zc.StepBatch(starts.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), table, tokens=sum(news), max_new=max(news),
                        max_length=max(lengths))


def answer(decoder, prompts, *, chunk=64, tokens=16, temperature=0.8, top_k=40, top_p=0.95, seed=0):
    """Token ids [prompts, tokens]: reads the prompts (lists of token ids) chunk by chunk, all in one batch, then
    decodes. Returns (answers, last prompt logits)."""
    n = len(prompts)
    per = [-(-(len(p) + tokens) // PAGE) for p in prompts]
    table = torch.zeros((n, max(per)), dtype=torch.int32)
    order = torch.randperm(sum(per), generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    for s, pages in enumerate(order.split(per)):
        table[s, :len(pages)] = pages
    table = table.cuda()
    cache, workspace = new_cache(decoder, sum(per)), zc.Workspace()
    done = [0] * n
    last = torch.zeros((n, decoder.vocab), device="cuda")
    while any(d < len(p) for d, p in zip(done, prompts)):
        news = [min(chunk, len(p) - d) for d, p in zip(done, prompts)]
        ids = torch.tensor([t for d, m, p in zip(done, news, prompts) for t in p[d:d + m]], dtype=torch.int32).cuda()
        done = [d + m for d, m in zip(done, news)]
        logits = decoder.step(ids, cache, step_batch(news, done, table), workspace)
        at = 0
        for s, m in enumerate(news):
            at += m
            if m:
                last[s] = logits[at - 1]
    settings = {"temperature": torch.full((n,), temperature, device="cuda"), "top_p": torch.full((n,), top_p, device="cuda"),
                "top_k": torch.full((n,), top_k, dtype=torch.int32, device="cuda")}
    g = torch.Generator(device="cuda").manual_seed(seed)
    answers, logits = [], last
    for _ in range(tokens):
        ids, _ = zc.sample(logits, torch.rand(n, device="cuda", generator=g), **settings)
        answers.append(ids)
        done = [d + 1 for d in done]
        logits = decoder.step(ids, cache, step_batch([1] * n, done, table), workspace)
    workspace.raise_on_status()
    return torch.stack(answers, 1), last


def retrieve(questions, passages, k):
    """Ids [questions, k] of the passages nearest to the questions' vectors (fp16 rows, cosine)."""
    rows = torch.nn.functional.normalize(passages, dim=1)
    store = zc.convert_f16(rows)
    ids, _ = zc.scan_topk(store, zc.DTYPE_F16, rows.shape[1], torch.nn.functional.normalize(questions, dim=1), k)
    return ids


def main():
    torch.manual_seed(0)
    decoder = Decoder()
    vectors = torch.randn((20000, 384), device="cuda")
    texts = torch.randint(decoder.vocab, (20000, 80))
    questions = vectors[[7, 123, 4567]] + 0.5 * torch.randn((3, 384), device="cuda")
    found = retrieve(questions, vectors, 3).cpu()
    prompts = []
    for s in range(3):
        question = torch.randint(decoder.vocab, (11 + s,))
        prompts.append(torch.cat([texts[i] for i in found[s].tolist()] + [question]).tolist())
    answers, _ = answer(decoder, prompts)
    for s in range(3):
        print(f"question {s}: passages {found[s].tolist()}, {len(prompts[s])} prompt tokens -> {answers[s].tolist()}")


if __name__ == "__main__":
    main()
