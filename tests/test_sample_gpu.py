"""GPU: zcgvs_sample against its definition (answer_step.sample_reference). Tokens must be equal: weights are whole
numbers, so no sum depends on its order."""

from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import answer_step as ref  # noqa: E402


def _check(zc, logits, settings, uniforms):
    """settings: (temperature, top_k, top_p, min_p) per row."""
    rows = len(settings)
    t, k, p, low = (torch.tensor(c, dtype=d).cuda() for c, d in zip(zip(*settings), (torch.float32, torch.int32, torch.float32, torch.float32)))
    u = torch.tensor(uniforms, dtype=torch.float32)
    tokens, logprobs = zc.sample(logits, u.cuda(), temperature=t, top_k=k, top_p=p, min_p=low)
    host = logits.float().cpu()
    for r in range(rows):
        token, logprob = ref.sample_reference(host[r], *settings[r], float(u[r]))
        assert int(tokens[r]) == token, (r, settings[r])
        assert math.isclose(float(logprobs[r]), logprob, rel_tol=1e-6, abs_tol=1e-7)


def _logits(rows, vocab, seed, spread=3.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((rows, vocab), generator=g) * spread).to(dtype).cuda()


def _settings():
    out = []
    for t in (1.0, 0.3, 2.5):
        for k, p, low in ((0, 1.0, 0.0), (1, 1.0, 0.0), (5, 1.0, 0.0), (300, 1.0, 0.0), (0, 0.9, 0.0), (0, 0.01, 0.0), (0, 1.0, 0.1),
                          (40, 0.8, 0.02), (0, 0.999, 0.0), (10**9, 0.5, 0.0), (0, 0.0, 0.0), (3, 0.7, 2.0)):
            out.append((t, k, p, low))
    return out + [(0.0, 0, 1.0, 0.0), (-1.0, 7, 0.5, 0.0), (math.nan, 0, 1.0, 0.0), (1.0, -4, 1.5, -1.0), (1.0, 0, math.nan, math.nan),
                  (math.inf, 0, 0.9, 0.0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 4097, 33000])
def test_filters(zc, vocab, dtype):
    settings = _settings()
    g = torch.Generator().manual_seed(vocab)
    _check(zc, _logits(len(settings), vocab, vocab + 1, dtype=dtype), settings, torch.rand(len(settings), generator=g).tolist())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 3, 12])
def test_large_vocabularies(zc, rows, dtype):
    settings = [((0, 50)[r % 2], (1.0, 0.9)[r % 3 == 0]) for r in range(rows)]
    settings = [(0.8, k, p, 0.0) for k, p in settings]
    g = torch.Generator().manual_seed(rows)
    _check(zc, _logits(rows, 151669, rows, dtype=dtype), settings, torch.rand(rows, generator=g).tolist())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_largest_vocabulary(zc, dtype):
    _check(zc, _logits(2, zc.MAX_VOCAB, 5, dtype=dtype), [(1.0, 100, 0.95, 0.0), (1.0, 0, 0.5, 0.0)], [0.3, 0.999])


@pytest.mark.parametrize("vocab", [3000, 40000])
def test_equal_logits_take_the_lowest_ids(zc, vocab):
    """All equal, two levels, and a few distinct values: bins hold far more tokens than are ranked directly."""
    flat = torch.zeros((3, vocab), device="cuda")
    flat[1, ::2] = 1.0
    flat[2] = torch.arange(vocab, device="cuda") % 3
    settings = [(1.0, 1500, 1.0, 0.0), (1.0, 0, 0.6, 0.0), (0.7, vocab // 2 + 1, 0.9, 0.0)]
    for u in (0.0, 0.5, 0.99999994):
        _check(zc, flat, settings, [u] * 3)


def test_clustered_logits(zc):
    """Values a few units of the last place apart, next to one far away: every bin but one is empty."""
    x = torch.full((2, 20000), 100.0, device="cuda")
    x += (torch.arange(20000, device="cuda") * 7919 % 20000) * 2.0**-17
    x[:, 77] = -1e9
    _check(zc, x, [(1.0, 3000, 1.0, 0.0), (0.5, 0, 0.4, 0.0)], [0.25, 0.75])


def test_edges_of_the_uniform_number(zc):
    x = _logits(7, 500, 3)
    _check(zc, x, [(1.0, 0, 0.95, 0.0)] * 7, [0.0, 1.0, 2.0, -1.0, math.nan, 1e-30, 0.99999994])


def test_infinities_nan_and_masks(zc):
    low = torch.finfo(torch.float32).min
    x = _logits(7, 3000, 4)
    x[0, 1:] = -math.inf
    x[1, ::3] = math.nan
    x[2] = -math.inf
    x[3, [5, 99, 2000]] = math.inf
    x[4, 10:] = low
    x[5] = low
    x[6] = math.nan
    _check(zc, x, [(0.9, 20, 0.9, 0.0)] * 7, [0.7] * 7)
    _check(zc, x, [(1.0, 0, 1.0, 0.0)] * 7, [0.99] * 7)
    _check(zc, x, [(0.0, 0, 1.0, 0.0)] * 7, [0.5] * 7)


def test_signed_zeros_tie(zc):
    x = torch.tensor([[-0.0, 0.0, -0.0, 0.0, -5.0]], device="cuda")
    for k in (1, 2, 3):
        _check(zc, x, [(1.0, k, 1.0, 0.0)], [0.999])
    _check(zc, x, [(0.0, 0, 1.0, 0.0)], [0.0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_strided_and_unaligned_rows(zc, dtype):
    wide = _logits(5, 5003, 8, dtype=dtype)
    _check(zc, wide[:, 1:5000], [(0.9, 30, 0.9, 0.01)] * 5, [0.1, 0.3, 0.5, 0.7, 0.9])


def test_without_settings_and_on_another_stream(zc):
    x = _logits(4, 1000, 11)
    u = torch.tensor([0.1, 0.4, 0.6, 0.95], device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    out = (torch.empty(4, dtype=torch.int32, device="cuda"), torch.empty(4, device="cuda"))
    zc.sample(x, u, out=out, stream=side)
    side.synchronize()
    for r in range(4):
        token, logprob = ref.sample_reference(x[r].cpu(), 1.0, 0, 1.0, 0.0, float(u[r]))
        assert int(out[0][r]) == token and math.isclose(float(out[1][r]), logprob, rel_tol=1e-6)


def test_frequencies_follow_the_weights(zc):
    """An even grid of uniform numbers draws each token as often as its share of the weight says, within one grid step."""
    x = torch.tensor([0.0, 1.0, -2.0, 0.5, 3.0]).repeat(4096, 1).cuda()
    u = (torch.arange(4096, device="cuda") + 0.5) / 4096
    tokens, _ = zc.sample(x, u.float())
    share = torch.bincount(tokens.long(), minlength=5).double() / 4096
    want = torch.softmax(x[0].double(), 0)
    assert bool(((share - want).abs() <= 1 / 4096).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("k", [255, 256, 257, 1000, 5000])
def test_top_k_around_the_list_that_is_taken_at_once(zc, k, dtype):
    settings = [(0.9, k, 1.0, 0.0), (1.3, k, 0.97, 0.0), (2.0, k, 0.6, 0.01)]
    _check(zc, _logits(3, 50000, k, dtype=dtype), settings, [0.2, 0.93, 0.5])


@pytest.mark.parametrize("spread", [0.001, 0.3, 30.0, 1000.0])
def test_flat_and_steep_distributions(zc, spread):
    settings = [(1.0, 0, 0.9, 0.0), (0.1, 0, 0.5, 0.001), (5.0, 0, 0.999, 0.0), (1.0, 400, 0.9, 0.0)]
    for dtype in (torch.float32, torch.bfloat16):
        _check(zc, _logits(4, 30000, 7, spread=spread, dtype=dtype), settings, [0.1, 0.6, 0.99, 0.4])


def test_extreme_temperatures(zc):
    settings = [(1e-30, 0, 0.9, 0.0), (1e-4, 0, 0.9, 0.0), (1e30, 0, 0.3, 0.0), (1e10, 20, 0.5, 0.0), (1e-40, 7, 1.0, 0.0)]
    _check(zc, _logits(5, 9000, 12), settings, [0.5] * 5)


def test_quotients_are_correctly_rounded(zc):
    """Two tokens at a chosen distance: the drawn token turns at the weight of the correctly rounded quotient, so the
    logarithm of its probability equals the definition's to the last bit of its fp32 value."""
    g = torch.Generator().manual_seed(0)
    rows = 4000
    distance = torch.rand(rows, generator=g) * 20
    temperature = (torch.rand(rows, generator=g) + 0.05).float()
    x = torch.zeros((rows, 2))
    x[:, 1] = -distance
    tokens, logprobs = zc.sample(x.cuda(), torch.full((rows,), 0.99999994).cuda(), temperature=temperature.cuda(),
                                 top_p=torch.full((rows,), 0.99999994).cuda())
    e = torch.exp((x.cuda()[:, 1] / temperature.cuda()))
    w = (e.double() * 2.0**40).round()
    total = w + 2.0**40
    kept = 2.0**40 < 0.9999999403953552 * total  # whether top-p keeps the second token
    second = tokens == 1
    assert bool((second <= kept).all())
    want = torch.log(torch.where(second, w, torch.full_like(w, 2.0**40)) / torch.where(kept, total, torch.full_like(w, 2.0**40))).float()
    assert torch.equal(logprobs, want)
