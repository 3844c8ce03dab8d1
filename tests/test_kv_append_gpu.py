"""GPU: zcgvs_kv_append against its definition in 64 bits: every head is normed, rotated and rounded
once, so a value may be off by half a unit of its type plus a few fp32 roundings of its pair's size."""

from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import answer_step as ref  # noqa: E402


def _inputs(tokens, q_heads, kv_heads, dim, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    rows = (torch.randn((tokens, q_heads + 2 * kv_heads, dim), generator=g) * 3).to(dtype).cuda()
    return rows, rows[:, :q_heads], rows[:, q_heads:q_heads + kv_heads], rows[:, q_heads + kv_heads:]


def _close(got, want, size, dtype):
    """size: the magnitude of what was added up (the pair's norm)."""
    limit = want.abs() * ref.UNIT[dtype] + size * 2.0**-20 + ref.TINY[dtype]
    assert bool(((got.double() - want).abs() <= limit).all()), float(((got.double() - want).abs() - limit).max())


def _run(zc, news, lengths, *, q_heads=6, kv_heads=2, dim=64, page=16, dtype=torch.bfloat16, rotary=None, interleaved=False, norm=True,
         heads_first=False, positions=None, in_place=False, extra=0, rows=4096, with_rotary=True):
    cache, batch, table = ref.make_step(zc, news, lengths, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, fill=7.0,
                                        heads_first=heads_first, extra_tokens=extra)
    before = cache.keys.clone(), cache.values.clone()
    rows_t, q, k, v = _inputs(batch.tokens, q_heads, kv_heads, dim, dtype, 5)
    kept = rows_t.clone()
    rotary = dim // 16 * 16 if rotary is None else rotary
    turn = zc.rotary_table(rows, rotary, 500.0) if with_rotary and rotary else None
    g = torch.Generator().manual_seed(9)
    wq, wk = ((1 + 0.3 * torch.randn(dim, generator=g)).to(dtype).cuda() if norm else None for _ in range(2))
    out = zc.kv_append(cache, batch, q, k, v, rotary=turn, interleaved=interleaved, q_norm=wq, k_norm=wk, eps=1e-5,
                       positions=None if positions is None else torch.tensor(positions, dtype=torch.int32).cuda(),
                       out=q if in_place else None)
    torch.cuda.synchronize()
    q, k, v = kept[:, :q_heads], kept[:, q_heads:q_heads + kv_heads], kept[:, q_heads + kv_heads:]
    want_k, want_v = before[0].double(), before[1]
    touched = torch.zeros(cache.keys.shape[:2], dtype=torch.bool, device="cuda")
    at = 0
    for s, (new, length) in enumerate(zip(news, lengths)):
        for j in range(new):
            pos = length - new + j
            turned = pos if positions is None else positions[at]
            row = slice(at, at + 1)
            if turn is not None and not 0 <= turned < rows:
                assert bool((out[at] == 0).all())
                at += 1
                continue
            angles = turn[turned:turned + 1] if turn is not None else None
            want_q = ref.rotate_reference(q[row], wq, 1e-5, angles, rotary, interleaved)
            _close(out[row], want_q, want_q.norm(dim=-1, keepdim=True), dtype)
            if pos >= 0:
                p, o = int(table[s, pos // page]), pos % page
                y = ref.rotate_reference(k[row], wk, 1e-5, angles, rotary, interleaved)
                _close(cache.keys[p, o][None], y, y.norm(dim=-1, keepdim=True), dtype)
                want_v[p, o] = v[at]
                touched[p, o] = True
            at += 1
    assert torch.equal(cache.values, want_v), "values"
    assert torch.equal(cache.keys[~touched], before[0][~touched]), "a slot that is not the step's was written"
    return out, cache


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,rotary,interleaved", [(128, 128, False), (128, 64, True), (64, 64, True), (96, 96, False), (80, 48, False),
                                                    (72, 64, True), (16, 16, False), (8, 0, False), (120, 112, False)])
def test_head_sizes_and_rotations(zc, dim, rotary, interleaved, dtype):
    _run(zc, [1, 5, 0, 9], [1, 40, 12, 9], dim=dim, rotary=rotary, interleaved=interleaved, dtype=dtype, page=8)


@pytest.mark.parametrize("q_heads,kv_heads", [(1, 1), (7, 1), (40, 8), (64, 64), (5, 5)])
@pytest.mark.parametrize("dim", [64, 128])
def test_head_counts(zc, q_heads, kv_heads, dim):
    _run(zc, [3, 2], [17, 2], q_heads=q_heads, kv_heads=kv_heads, dim=dim)


@pytest.mark.parametrize("page", [1, 3, 16, 100])
@pytest.mark.parametrize("heads_first", [False, True])
def test_pages_and_layouts(zc, page, heads_first):
    _run(zc, [4, 30, 1], [104, 31, 77], page=page, heads_first=heads_first)


def test_plain_store_without_norm_and_rotation(zc):
    _run(zc, [2, 3], [9, 3], norm=False, with_rotary=False)


def test_more_sequences_than_a_warp_searches_in_one_round(zc):
    n = 1100
    _run(zc, [(s * 7) % 3 for s in range(n)], [3 + s % 5 for s in range(n)], q_heads=2, kv_heads=1, dim=16, page=4)


def test_positions_of_the_callers(zc):
    _run(zc, [4, 2], [10, 2], positions=[100, 0, 7, 4095, 3, 2])


def test_tokens_without_a_rotation_row_or_a_slot(zc):
    # The second sequence has fewer cached tokens than new ones: its first two are at negative positions.
    _run(zc, [3, 4], [64, 2], rows=63)
    _run(zc, [2], [5], positions=[-1, 5000])


def test_queries_in_place_and_padding_tokens(zc):
    out, _ = _run(zc, [3, 1], [20, 6], in_place=True)
    cache, batch, _ = ref.make_step(zc, [2], [2], kv_heads=1, dim=64, page=8, dtype=torch.float16, fill=7.0, extra_tokens=5)
    rows, q, k, v = _inputs(7, 2, 1, 64, torch.float16, 1)
    out = torch.full_like(q, 3.0)
    zc.kv_append(cache, batch, q, k, v, rotary=zc.rotary_table(8, 64), out=out)
    assert bool((out[2:] == 3).all()), "padding tokens are left alone"
    assert int((cache.keys != 7).any(-1).sum()) == 2


def test_keys_alone_and_queries_alone(zc):
    cache, batch, table = ref.make_step(zc, [3], [9], kv_heads=2, dim=64, page=4, dtype=torch.bfloat16, fill=7.0)
    _, q, k, v = _inputs(3, 4, 2, 64, torch.bfloat16, 2)
    turn = zc.rotary_table(16, 64)
    assert zc.kv_append(cache, batch, None, k, v, rotary=turn) is None
    keys = cache.keys.clone()
    both = zc.kv_append(cache, batch, q, k, v, rotary=turn)
    assert torch.equal(keys, cache.keys)
    cache.keys.fill_(7.0)
    alone = zc.kv_append(cache, batch, q, None, None, rotary=turn)
    assert torch.equal(alone, both) and bool((cache.keys == 7).all())


def test_pages_out_of_range_are_not_written(zc):
    cache, batch, table = ref.make_step(zc, [1, 1], [1, 1], kv_heads=1, dim=64, page=4, dtype=torch.float16, fill=7.0)
    batch.page_table[0, 0] = -1
    batch.page_table[1, 0] = cache.pages
    _, q, k, v = _inputs(2, 1, 1, 64, torch.float16, 3)
    zc.kv_append(cache, batch, q, k, v)
    torch.cuda.synchronize()
    assert bool((cache.keys == 7).all()) and bool((cache.values == 7).all())


def test_value_bits_and_infinities_pass_unchanged(zc):
    cache, batch, table = ref.make_step(zc, [1], [1], kv_heads=1, dim=64, page=4, dtype=torch.bfloat16, fill=7.0)
    _, q, k, v = _inputs(1, 1, 1, 64, torch.bfloat16, 4)
    v[0, 0, :3] = torch.tensor([float("inf"), float("-inf"), float("nan")], dtype=torch.bfloat16)
    zc.kv_append(cache, batch, q, k, v)
    got = cache.values[int(table[0, 0]), 0, 0]
    assert torch.equal(got.view(torch.int16), v[0, 0].view(torch.int16))
