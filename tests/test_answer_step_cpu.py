"""CPU: what the answer step's entry points refuse, before they touch a device."""

from __future__ import annotations

import ctypes

import pytest

F16, BF16 = 1, 5
A, B = 4096, 8192  # addresses that are never read


def _cache(zc, **kw):
    f = dict(keys=A, values=B, pages=10, page_stride=16 * 2 * 64, slot_stride=2 * 64, head_stride=64, page_size=16, kv_heads=2, head_dim=64,
             dtype=F16)
    return zc._PagedCacheStruct(**{**f, **kw})


def _batch(zc, **kw):
    f = dict(query_starts=A, kv_lengths=A, page_table=A, page_table_stride=4, pages_per_sequence=4, sequences=2, tokens=5, max_new=3,
             max_length=64)
    return zc._StepBatchStruct(**{**f, **kw})


def _append(zc, cache=None, batch=None, **kw):
    a = dict(q=A, q_token=256, q_head=64, q_heads=4, k=A, k_token=128, k_head=64, v=A, v_token=128, v_head=64, q_norm=None, k_norm=None,
             eps=1e-6, rotary=A, rows=100, rotary_dim=64, interleaved=0, positions=None, out=A, out_token=256, out_head=64)
    a.update(kw)
    cache = _cache(zc) if cache is None else cache
    batch = _batch(zc) if batch is None else batch
    return zc.lib().zcgvs_kv_append(ctypes.byref(cache), ctypes.byref(batch), *a.values(), None)


def _attend(zc, cache=None, batch=None, **kw):
    a = dict(q=A, q_token=256, q_head=64, q_heads=4, scale=0.1, causal=1, window=0, out=A, out_token=256, out_head=64, lse=None,
             workspace=A, bytes=1 << 40)
    a.update(kw)
    cache = _cache(zc) if cache is None else cache
    batch = _batch(zc) if batch is None else batch
    return zc.lib().zcgvs_paged_attention(ctypes.byref(cache), ctypes.byref(batch), *a.values(), None)


def _sample(zc, **kw):
    a = dict(logits=A, dtype=0, stride=100, rows=2, vocab=100, temperature=None, top_k=None, top_p=None, min_p=None, uniforms=A, tokens=A,
             logprobs=None)
    a.update(kw)
    return zc.lib().zcgvs_sample(*a.values(), None)


def _says(zc, status, expect, text):
    assert status == expect, zc.lib().zcgvs_last_error_message()
    assert text in zc.lib().zcgvs_last_error_message().decode()


CACHE_FAULTS = [
    (dict(dtype=0), 1, "F16 or BF16"), (dict(dtype=4), 1, "F16 or BF16"), (dict(page_size=0), 1, "page_size"), (dict(kv_heads=0), 1, "kv_heads"),
    (dict(head_dim=0), 1, "multiple of 8"), (dict(head_dim=60), 1, "multiple of 8"), (dict(head_dim=136), 3, "exceeds 128"),
    (dict(pages=-1), 1, "pages"), (dict(keys=None), 1, "null cache"), (dict(values=None), 1, "null cache"), (dict(keys=A + 2), 1, "16-byte"),
    (dict(slot_stride=130), 1, "multiples of 8"), (dict(page_stride=-8), 1, "negative"),
]
BATCH_FAULTS = [
    (dict(query_starts=None), 1, "query_starts"), (dict(kv_lengths=None), 1, "kv_lengths"), (dict(page_table=None), 1, "page_table"),
    (dict(pages_per_sequence=0), 1, "pages_per_sequence"), (dict(page_table_stride=3), 1, "page_table_stride"),
    (dict(pages_per_sequence=1 << 28, page_table_stride=1 << 28), 1, "2^31"),
]


@pytest.mark.parametrize("fault,status,text", CACHE_FAULTS)
def test_a_bad_cache_is_refused(zc, fault, status, text):
    _says(zc, _append(zc, cache=_cache(zc, **fault)), status, text)
    _says(zc, _attend(zc, cache=_cache(zc, **fault)), status, text)


@pytest.mark.parametrize("fault,status,text", BATCH_FAULTS)
def test_a_bad_step_is_refused(zc, fault, status, text):
    _says(zc, _append(zc, batch=_batch(zc, **fault)), status, text)
    _says(zc, _attend(zc, batch=_batch(zc, **fault)), status, text)


@pytest.mark.parametrize("fault,text", [
    (dict(k=None), "together"), (dict(v=None), "together"), (dict(out=None), "q_out"), (dict(q_heads=0), "q_heads"), (dict(q_heads=-1), "q_heads"),
    (dict(q=A + 8), "q must be 16-byte"), (dict(k_token=129), "k's strides"), (dict(v_head=-64), "v's strides"), (dict(out=A + 4), "q_out"),
    (dict(rotary_dim=8), "rotary_dim"), (dict(rotary_dim=80), "rotary_dim"), (dict(rows=0), "rotary_rows"), (dict(rows=1 << 40), "rotary_rows"),
    (dict(rotary=A + 4), "16-byte"), (dict(q_norm=A + 2), "16-byte"),
])
def test_append_refuses(zc, fault, text):
    _says(zc, _append(zc, **fault), zc.ERR_INVALID_ARG, text)


@pytest.mark.parametrize("fault,text", [
    (dict(q=None), "null q"), (dict(out=None), "null q or out"), (dict(q_heads=3), "multiple of kv_heads"), (dict(q=A + 8), "q must be 16-byte"),
    (dict(out_token=7), "out's strides"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(window=-1), "window"),
    (dict(workspace=None), "workspace"), (dict(bytes=100), "workspace"), (dict(workspace=A + 16), "256-byte"),
])
def test_attention_refuses(zc, fault, text):
    _says(zc, _attend(zc, **fault), zc.ERR_INVALID_ARG, text)


@pytest.mark.parametrize("fault,status,text", [
    (dict(dtype=2), 1, "F32, F16 or BF16"), (dict(vocab=327681, stride=400000), 3, "ZCGVS_MAX_VOCAB"), (dict(logits=None), 1, "null"),
    (dict(uniforms=None), 1, "null"), (dict(tokens=None), 1, "null"), (dict(stride=99), 1, "row_stride"), (dict(logits=A + 2), 1, "aligned"),
])
def test_sample_refuses(zc, fault, status, text):
    _says(zc, _sample(zc, **fault), status, text)


def test_null_structs_and_empty_steps(zc):
    lib = zc.lib()
    cache, batch = ctypes.byref(_cache(zc)), ctypes.byref(_batch(zc))
    for c, b in ((None, batch), (cache, None)):
        assert lib.zcgvs_paged_attention(c, b, A, 256, 64, 4, 0.1, 1, 0, A, 256, 64, None, A, 1 << 40, None) == zc.ERR_INVALID_ARG
        assert lib.zcgvs_kv_append(c, b, A, 256, 64, 4, A, 128, 64, A, 128, 64, None, None, 1e-6, None, 0, 0, 0, None, A, 256, 64,
                                   None) == zc.ERR_INVALID_ARG
    for fault in (dict(tokens=0), dict(sequences=0), dict(tokens=-3)):
        assert _append(zc, batch=_batch(zc, **fault)) == zc.OK
        assert _attend(zc, batch=_batch(zc, **fault)) == zc.OK
    assert _sample(zc, rows=0) == zc.OK and _sample(zc, vocab=0) == zc.OK
    assert _append(zc, q=None, q_heads=0, k=None, v=None) == zc.OK
    assert lib.zcgvs_paged_attention_workspace_bytes(0) == 0 and lib.zcgvs_paged_attention_workspace_bytes(129) == 0


def test_a_corpus_is_not_stored_in_bf16(zc):
    fake = ctypes.c_void_p(4096)
    assert zc.lib().zcgvs_scan_topk(fake, BF16, 1.0, None, 100, 8, fake, 1, None, zc.METRIC_DOT, 10, 0, fake, fake, fake, 1 << 20,
                                    None) != zc.OK


def test_the_binding_refuses_tensors_it_cannot_pass_on(zc):
    torch = pytest.importorskip("torch")
    keys = torch.zeros((4, 8, 2, 64), dtype=torch.float16)
    cache = zc.PagedKvCache(keys, torch.zeros_like(keys))
    with pytest.raises(zc.InvalidArgument, match="same shape"):
        zc.PagedKvCache(keys, torch.zeros((4, 8, 2, 32), dtype=torch.float16))
    with pytest.raises(zc.InvalidArgument, match="contiguous"):
        zc.PagedKvCache(keys.transpose(2, 3), keys.transpose(2, 3))
    with pytest.raises(zc.InvalidArgument, match="unsupported type"):
        zc.PagedKvCache(keys.float(), keys.float())
    starts, lengths = torch.tensor([0, 2, 3], dtype=torch.int32), torch.tensor([5, 9], dtype=torch.int32)
    table = torch.zeros((2, 3), dtype=torch.int32)
    batch = zc.StepBatch(starts, lengths, table, tokens=3)
    for args in ((starts.long(), lengths, table), (starts[:2], lengths, table), (starts, lengths, table.T.contiguous()),
                 (starts, lengths, table.long())):
        with pytest.raises(zc.InvalidArgument):
            zc.StepBatch(*args, tokens=3)
    q = torch.zeros((3, 4, 64), dtype=torch.float16)
    kv = torch.zeros((3, 2, 64), dtype=torch.float16)
    for bad in (q.bfloat16(), q[:2], q[..., :32], torch.zeros((3, 64, 4), dtype=torch.float16).transpose(1, 2)):
        with pytest.raises(zc.InvalidArgument):
            zc.paged_attention(cache, batch, bad, scale=0.1)
        with pytest.raises(zc.InvalidArgument):
            zc.kv_append(cache, batch, bad, kv, kv)
    with pytest.raises(zc.InvalidArgument):
        zc.kv_append(cache, batch, q, q, kv)
    with pytest.raises(zc.InvalidArgument, match="rotary"):
        zc.kv_append(cache, batch, q, kv, kv, rotary=torch.zeros((9, 64), dtype=torch.float64))
    logits = torch.zeros((2, 10))
    with pytest.raises(zc.InvalidArgument, match="uniforms"):
        zc.sample(logits, torch.zeros(3))
    with pytest.raises(zc.InvalidArgument, match="top_k"):
        zc.sample(logits, torch.zeros(2), top_k=torch.zeros(2))
    with pytest.raises(zc.InvalidArgument, match="contiguous rows"):
        zc.sample(torch.zeros((10, 2)).T, torch.zeros(2))
