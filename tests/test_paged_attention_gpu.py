"""GPU: zcgvs_paged_attention against its definition in 64 bits, at the lengths, heads, masks and layouts
where it can go wrong (tolerance: answer_step.check_attention)."""

from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import answer_step as ref  # noqa: E402


def _queries(tokens, heads, dim, dtype, seed=3, scale=1.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((tokens, heads, dim), generator=g) * scale).to(dtype).cuda()


def _run(zc, news, lengths, *, group=4, kv_heads=2, dim=128, page=16, dtype=torch.bfloat16, causal=True, window=0, heads_first=False,
         scale=None, workspace=None, max_new=None, seed=0):
    cache, batch, table = ref.make_step(zc, news, lengths, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, heads_first=heads_first,
                                        max_new=max_new, seed=seed)
    kept = ref.fill_cached(cache, table, lengths, seed=seed + 1)
    q = _queries(batch.tokens, kv_heads * group, dim, dtype)
    scale = 1 / math.sqrt(dim) if scale is None else scale
    out, lse = zc.paged_attention(cache, batch, q, scale=scale, causal=causal, window=window, return_lse=True, workspace=workspace)
    ref.check_attention(out, lse, ref.attention_reference(q, kept, news, lengths, scale, causal, window), dtype)
    return out, lse, cache, batch, q


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [8, 40, 64, 72, 96, 128])
def test_decode_head_sizes(zc, dim, dtype):
    _run(zc, [1, 1, 1], [1, 63, 300], dim=dim, dtype=dtype)


@pytest.mark.parametrize("length", [1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 1000])
def test_decode_lengths_around_tiles(zc, length):
    _run(zc, [1], [length])


@pytest.mark.parametrize("group,kv_heads", [(1, 1), (1, 6), (3, 5), (7, 2), (8, 8), (16, 1), (17, 1), (33, 1), (64, 1), (65, 1), (130, 1)])
def test_groups(zc, group, kv_heads):
    _run(zc, [1, 2], [200, 77], group=group, kv_heads=kv_heads, dim=64)


@pytest.mark.parametrize("new", [2, 5, 16, 31, 32, 33, 64, 100, 257])
@pytest.mark.parametrize("dim", [64, 128])
def test_chunks(zc, new, dim):
    _run(zc, [new], [new + 150], dim=dim)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 80, 128])
def test_prompts_from_nothing(zc, dim, dtype):
    _run(zc, [200, 1, 77], [200, 1, 77], dim=dim, dtype=dtype, group=2, kv_heads=3)


@pytest.mark.parametrize("page", [1, 3, 8, 24, 64, 128, 200, 256, 384])
@pytest.mark.parametrize("news", [[1, 1], [150, 40]])
def test_page_sizes(zc, page, news):
    _run(zc, news, [411, 190], page=page)


@pytest.mark.parametrize("news", [[1, 1], [140, 3]])
def test_heads_first_pages(zc, news):
    _run(zc, news, [300, 170], heads_first=True, kv_heads=3, dim=96)


@pytest.mark.parametrize("window", [1, 2, 17, 64, 100, 1000])
@pytest.mark.parametrize("news", [[1, 1], [130, 20]])
def test_windows(zc, window, news):
    _run(zc, news, [420, 333], window=window)


@pytest.mark.parametrize("news", [[1, 4], [150, 33]])
@pytest.mark.parametrize("window", [0, 50])
def test_without_a_causal_mask(zc, news, window):
    _run(zc, news, [300, 90], causal=False, window=window)


@pytest.mark.parametrize("many", [False, True])
def test_rows_that_see_nothing(zc, many):
    """Sequences without cached tokens, with fewer cached than new ones (negative positions), and without new ones."""
    news = [2, 5, 0, 3, 1] if not many else [140, 200, 0, 3, 130]
    lengths = [0, 3, 50, 3, 0] if not many else [0, 70, 50, 3, 129]
    _run(zc, news, lengths)
    _run(zc, news, lengths, causal=False)


def test_ragged_batch_of_many_sequences(zc):
    n = 700
    news = [1 if s % 5 else (s // 5) % 3 for s in range(n)]
    lengths = [1 + (s * 37) % 150 for s in range(n)]
    _run(zc, news, lengths, kv_heads=1, group=2, dim=64)


def test_chunks_and_decoding_in_one_batch(zc):
    news = [1, 120, 1, 0, 40, 1, 1, 3]
    lengths = [500, 121, 3, 10, 400, 129, 1, 64]
    _run(zc, news, lengths)


def test_many_chunks_among_many_decoding(zc):
    n = 560
    _run(zc, [130 if s % 80 == 3 else 1 for s in range(n)], [131 + s % 40 for s in range(n)], kv_heads=1, group=2, dim=64)


@pytest.mark.parametrize("scale", [0.0, -0.1, 1.0])
def test_scales(zc, scale):
    _run(zc, [1, 20], [100, 60], scale=scale, dim=64)


def test_max_new_is_only_a_hint(zc):
    """A host bound that is too small or far too large changes no result."""
    for hint in (0, 1, 100000):
        _run(zc, [70, 1], [200, 90], max_new=hint)


@pytest.mark.parametrize("news", [[1], [300]])
def test_a_large_maximum_after_small_ones(zc, news):
    """Keys that grow along the sequence: the running maximum rises tile after tile by much more than a weight's range."""
    length, dim = 900, 64
    cache, batch, table = ref.make_step(zc, news, [length], kv_heads=1, dim=dim, page=16, dtype=torch.bfloat16)
    kept = ref.fill_cached(cache, table, [length])
    ramp = torch.linspace(0, 3, length, device="cuda")[:, None, None]
    k = (ramp * torch.ones((1, 1, dim), device="cuda")).to(torch.bfloat16)
    p, o = (t.cuda() for t in ref.slots_of(table, 0, 16, torch.arange(length)))
    cache.keys[p, o] = k
    q = torch.full((news[0], 2, dim), 0.25, dtype=torch.bfloat16, device="cuda")
    q[:, 1] = -0.25  # and one whose maximum comes first
    out, lse = zc.paged_attention(cache, batch, q, scale=1.0, return_lse=True)
    want = ref.attention_reference(q, [[k.double(), kept[0][1]]], news, [length], 1.0, True, 0)
    ref.check_attention(out, lse, want, torch.bfloat16)


@pytest.mark.parametrize("news", [[1, 1], [200, 90]])
def test_result_is_the_same_every_time_and_in_any_workspace(zc, news):
    ws = zc.Workspace()
    buf = ws.get(zc.paged_attention_workspace_bytes(128))
    first, lse, cache, batch, q = _run(zc, news, [5000, 700], kv_heads=1, workspace=ws)
    for fill in (255, 1):
        buf[4:] = fill  # what another call left there; the status word is zero
        again = zc.paged_attention(cache, batch, q, scale=1 / math.sqrt(128), return_lse=True, workspace=ws)
        assert torch.equal(first, again[0]) and torch.equal(lse, again[1])
    assert ws.status() == 0


@pytest.mark.parametrize("news", [[1, 2], [140, 33]])
def test_strided_queries_and_outputs(zc, news):
    lengths = [200, 90]
    cache, batch, table = ref.make_step(zc, news, lengths, kv_heads=2, dim=64, page=8, dtype=torch.float16)
    kept = ref.fill_cached(cache, table, lengths)
    wide = _queries(batch.tokens, 11, 64, torch.float16)
    q = wide[:, 1:9:2]
    room = torch.full((4, batch.tokens, 72), 5.0, dtype=torch.float16, device="cuda")
    out = room[:, :, :64].transpose(0, 1)
    _, lse = zc.paged_attention(cache, batch, q, scale=0.125, out=out, return_lse=True)
    ref.check_attention(out, lse, ref.attention_reference(q, kept, news, lengths, 0.125, True, 0), torch.float16)
    assert bool((room[:, :, 64:] == 5).all())


@pytest.mark.parametrize("news", [[1], [130]])
def test_missing_pages_read_as_zeros(zc, news):
    length, page = 200, 16
    cache, batch, table = ref.make_step(zc, news, [length], kv_heads=1, dim=64, page=page, dtype=torch.bfloat16)
    kept = ref.fill_cached(cache, table, [length])
    batch.page_table[0, 2] = -1
    batch.page_table[0, 5] = cache.pages
    for x in kept[0]:
        x[32:48] = 0
        x[80:96] = 0
    q = _queries(batch.tokens, 3, 64, torch.bfloat16)
    out, lse = zc.paged_attention(cache, batch, q, scale=0.125, return_lse=True)
    ref.check_attention(out, lse, ref.attention_reference(q, kept, news, [length], 0.125, True, 0), torch.bfloat16)


@pytest.mark.parametrize("news", [[1, 1], [100, 130]])
def test_positions_past_the_page_table_do_not_exist(zc, news):
    """A length beyond the table's columns: queries keep their positions, keys end at the table."""
    lengths = [160, 160]
    cache, batch, table = ref.make_step(zc, news, lengths, kv_heads=1, dim=64, page=16, dtype=torch.float16)
    kept = ref.fill_cached(cache, table, lengths)
    short = zc.StepBatch(batch.query_starts, batch.kv_lengths, batch.page_table[:, :7], tokens=batch.tokens, max_new=max(news))
    q = _queries(batch.tokens, 2, 64, torch.float16)
    out, lse = zc.paged_attention(cache, short, q, scale=0.125, return_lse=True)
    want = ref.attention_reference(q, [[x[:112] for x in pair] for pair in kept], news, lengths, 0.125, True, 0)
    ref.check_attention(out, lse, want, torch.float16)


@pytest.mark.parametrize("news", [[1], [140]])
def test_recycled_pages_before_the_window_are_not_read(zc, news):
    length, window, page = 700, 100, 16
    cache, batch, table = ref.make_step(zc, news, [length], kv_heads=1, dim=128, page=page, dtype=torch.bfloat16)
    kept = ref.fill_cached(cache, table, [length])
    first = length - news[0] - window + 1  # the first position any token sees
    for column in range(first // page):
        cache.keys[int(table[0, column])] = math.nan
        cache.values[int(table[0, column])] = math.nan
    inside = torch.arange(first // page * page, first)  # the same page, before the window
    p, o = (t.cuda() for t in ref.slots_of(table, 0, page, inside))
    cache.keys[p, o] = math.nan
    cache.values[p, o] = math.nan
    q = _queries(batch.tokens, 4, 128, torch.bfloat16)
    out, lse = zc.paged_attention(cache, batch, q, scale=0.1, window=window, return_lse=True)
    for x in kept[0]:
        x[:first] = 0
    ref.check_attention(out, lse, ref.attention_reference(q, kept, news, [length], 0.1, True, window), torch.bfloat16)


@pytest.mark.parametrize("new", [1, 140])
def test_offsets_past_32_bits(zc, new):
    """A cache of more than 2^31 elements, used at its far end."""
    page, heads, dim, length = 64, 8, 128, 300
    pages = (1 << 31) // (page * heads * dim) + 40
    keys = torch.zeros((pages, page, heads, dim), dtype=torch.bfloat16, device="cuda")
    values = torch.zeros_like(keys)
    table = torch.arange(pages - 5, pages, dtype=torch.int32)[None].contiguous()
    cache = zc.PagedKvCache(keys, values)
    batch = zc.StepBatch(torch.tensor([0, new], dtype=torch.int32).cuda(), torch.tensor([length], dtype=torch.int32).cuda(), table.cuda(),
                         tokens=new, max_new=new)
    kept = ref.fill_cached(cache, table, [length])
    q = _queries(new, 16, dim, torch.bfloat16)
    out, lse = zc.paged_attention(cache, batch, q, scale=0.09, return_lse=True)
    ref.check_attention(out, lse, ref.attention_reference(q, kept, [new], [length], 0.09, True, 0), torch.bfloat16)


@pytest.mark.parametrize("news", [[1, 1], [150, 20]])
def test_on_another_stream(zc, news):
    lengths = [300, 64]
    cache, batch, table = ref.make_step(zc, news, lengths, kv_heads=2, dim=64, page=16, dtype=torch.float16)
    kept = ref.fill_cached(cache, table, lengths)
    q = _queries(batch.tokens, 4, 64, torch.float16)
    out = torch.empty_like(q)
    ws = zc.Workspace()
    ws.get(zc.paged_attention_workspace_bytes(64))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    _, lse = zc.paged_attention(cache, batch, q, scale=0.125, out=out, return_lse=True, workspace=ws, stream=side)
    side.synchronize()
    ref.check_attention(out, lse, ref.attention_reference(q, kept, news, lengths, 0.125, True, 0), torch.float16)


def test_padding_tokens_are_left_alone(zc):
    cache, batch, table = ref.make_step(zc, [1, 1], [20, 30], kv_heads=1, dim=64, page=8, dtype=torch.float16, extra_tokens=3)
    ref.fill_cached(cache, table, [20, 30])
    q = _queries(5, 2, 64, torch.float16)
    out = torch.full_like(q, 9.0)
    zc.paged_attention(cache, batch, q, scale=0.125, out=out)
    assert bool((out[2:] == 9).all()) and bool((out[:2] != 9).all())


@pytest.mark.parametrize("page", [3, 8])
@pytest.mark.parametrize("group,new", [(4, 5), (4, 12), (9, 3), (20, 3), (5, 6)])
def test_row_tiles_of_32_and_64(zc, group, new, page):
    """Rows that fill two and four warps, with pages that TMA boxes fit and that they do not."""
    _run(zc, [new, 1, new - 1], [new + 200, 70, 90], group=group, page=page)
    _run(zc, [new, 1], [new + 100, 64], group=group, page=page, dim=64, window=40, dtype=torch.float16)


@pytest.mark.parametrize("group", [3, 5, 7, 24])
@pytest.mark.parametrize("dim", [64, 128])
def test_chunks_of_groups_that_are_no_power_of_two(zc, group, dim):
    _run(zc, [300, 130], [700, 130], group=group, kv_heads=1, dim=dim)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_chunks_cut_between_many_ctas(zc, dtype):
    """One unit over far more key tiles than a CTA takes: its parts are joined by a kernel of their own."""
    _run(zc, [65], [30000], group=1, kv_heads=1, dtype=dtype, page=64)
    _run(zc, [70, 2], [9000, 5000], group=4, kv_heads=2, dtype=dtype, page=128, window=6000)


def test_a_decoding_unit_cut_between_all_ctas(zc):
    _run(zc, [1], [70001], group=8, kv_heads=1, page=64)
