"""Drawn tokens against the rule in 64 bits.  Weights there are doubles, here whole multiples of 2^-45 or finer of the
power of 2^(1/16) that is nearest to them, and so within 2^-45 of themselves; the sum of those of one power is brought to multiples of 2^-45 of the largest.  A running sum
is off by 2^-45 of itself and 2^10 halves of such a step at most, and a token differs where a uniform number's place lies that near to a border, which is to say (borders up to
2^17, sums of one or more) in one draw of 2^45 / (1 + 2^9) / 2^17, some 2^18, at the worst.  Logits and numbers here are fixed."""
import math

import numpy as np
import pytest
import torch

import sspmm_amd

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16, torch.float32]
INF = float("inf")


def _draw(x, u, temperature, top_k, top_p, min_p):
    """(token, probability) of one row of doubles."""
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.lexsort((np.arange(x.size), -x))
    y = x[order]
    y = y[y > -np.inf]
    if y.size == 0:
        return -1, 0.0
    if not temperature > 0:
        return int(order[0]), 1.0
    w = np.ones_like(y)
    below = y < y[0]
    with np.errstate(over="ignore"):
        w[below] = np.exp((y[below] - y[0]) / temperature) if y[0] < np.inf else 0.0
    w = w[(w >= min(min_p, 1.0)) & (w > 0)] if min_p > 0 else w[w > 0]
    if top_k > 0:
        w = w[:top_k]
    if top_p < 1:
        sums = np.cumsum(w)
        w = w[:max(1, int(np.searchsorted(sums, top_p * sums[-1], side="left")) + 1)]
    sums = np.cumsum(w)
    at = min(int(np.searchsorted(sums, u * sums[-1], side="right")), w.size - 1)
    return int(order[at]), float(w[at] / sums[-1])


def _check(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    got, chances = sspmm_amd.sample_tokens(logits, uniform, temperature, top_k, top_p, min_p, probabilities=True)
    assert got.dtype is torch.int32 and chances.dtype is torch.float32
    x = logits.double().cpu().numpy()
    columns = []
    for value in (uniform, temperature, top_k, top_p, min_p):
        columns.append(value.double().tolist() if isinstance(value, torch.Tensor) else [float(np.float32(value))] * x.shape[0])
    for i, (u, t, k, p, m) in enumerate(zip(*columns)):
        token, chance = _draw(x[i], u, t, int(k), p, m)
        assert int(got[i]) == token, (i, int(got[i]), token, u, t, k, p, m)
        # (a step of 2^-45 of the largest in the weight, 2^-28 of the sum in all; half a step of 32 bits of the quotient)
        assert abs(float(chances[i]) - chance) <= chance * (2.0 ** -24 + 2.0 ** -27) + 2.0 ** -45, (i, float(chances[i]), chance)


def _logits(rows, vocab, dtype, seed, spread=3.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g, device="cuda") * spread).to(dtype), torch.rand(rows, generator=g, device="cuda")


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 0, 1.0, 0.0), (1.3, 5, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.1), (0.8, 40, 0.95, 0.02), (0.0, 3, 0.5, 0.5), (2.0, 1, 1.0, 0.0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 2, 3, 5, 8, 31, 64, 257, 1000, 4099, 8192, 50001])
def test_against_the_rule(built_library, vocab, dtype):
    for i, settings in enumerate(SETTINGS):
        logits, uniform = _logits(9, vocab, dtype, seed=17 * vocab + i)
        print(vocab, dtype, settings, flush=True)
        _check(logits, uniform, *settings)


@pytest.mark.parametrize("dtype", TYPES)
def test_every_row_its_own_settings(built_library, dtype):
    rows = 61
    logits, uniform = _logits(rows, 3001, dtype, seed=1)
    i = torch.arange(rows, device="cuda")
    temperature = torch.tensor([0.0, 0.3, 0.7, 1.0, 1.5, 5.0], device="cuda")[i % 6]
    top_k = torch.tensor([0, 1, 2, 50, 5000, -1, 700], dtype=torch.int32, device="cuda")[i % 7]
    top_p = torch.tensor([1.0, 0.9, 0.5, 0.01, 0.0], device="cuda")[i % 5]
    min_p = torch.tensor([0.0, 0.05, 1.0], device="cuda")[i % 3]
    _check(logits, uniform, temperature, top_k, top_p, min_p)
    _check(logits, uniform, temperature, 50, top_p, 0.0)
    _check(logits, uniform, 1.0, top_k, 0.9, min_p)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [131072, 130999])
def test_large_vocabularies(built_library, vocab, dtype):
    logits, uniform = _logits(6, vocab, dtype, seed=vocab)
    for settings in ((1.0, 0, 1.0, 0.0), (1.0, 1000, 0.9, 0.0), (3.0, 0, 0.99, 0.0), (30.0, 100000, 0.9, 1e-4)):
        _check(logits, uniform, *settings)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [7, 4096, 70000])
def test_equal_logits_go_by_their_index(built_library, vocab, dtype):
    """All weights are the same, and every sum is exact: the token is floor(u * kept)."""
    rows = 33
    logits = torch.full((rows, vocab), 2.5, dtype=dtype, device="cuda")
    uniform = (torch.arange(rows, device="cuda") / rows).float()
    for top_k, top_p in ((0, 1.0), (5, 1.0), (0, 0.5), (6, 0.5), (vocab, 1.0), (0, 0.0)):
        kept = vocab if top_k == 0 else min(top_k, vocab)
        kept = kept if top_p == 1.0 else max(1, math.ceil(top_p * kept))
        got, chances = sspmm_amd.sample_tokens(logits, uniform, 0.5, top_k, top_p, probabilities=True)
        want = torch.tensor([int(math.floor(u * kept)) for u in uniform.double().tolist()], dtype=torch.int32)
        assert torch.equal(got.cpu(), want), (top_k, top_p)
        assert torch.equal(chances.cpu(), torch.full((rows,), np.float32(1.0 / kept)))


@pytest.mark.parametrize("dtype", TYPES)
def test_few_levels_many_tokens(built_library, dtype):
    """Thousands of tokens of each logit: borders fall among equals."""
    rows, vocab = 40, 20011
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    logits = torch.randint(0, 4, (rows, vocab), generator=g, device="cuda").to(dtype) * 0.5
    uniform = torch.rand(rows, generator=g, device="cuda")
    for settings in ((1.0, 0, 1.0, 0.0), (1.0, 6000, 1.0, 0.0), (0.5, 0, 0.8, 0.0), (1.0, 9000, 0.7, 0.0), (1.0, 0, 1.0, 0.5), (1.0, 12000, 0.97, 0.3)):
        _check(logits, uniform, *settings)


@pytest.mark.parametrize("dtype", TYPES)
def test_what_is_not_finite(built_library, dtype):
    x = torch.tensor([[1.0, -INF, 2.0, float("nan"), 0.5], [-INF] * 5, [float("nan")] * 5, [INF, 1.0, INF, -INF, INF], [-INF, -INF, -3.0, -INF, -INF], [0.0, -0.0, 0.0, -0.0, -INF],
                      [INF, INF, INF, INF, INF], [torch.finfo(dtype).min] * 5, [torch.finfo(dtype).max, torch.finfo(dtype).min, 0.0, 1.0, -INF]], device="cuda").to(dtype)
    for u in (0.0, 0.25, 0.34, 0.5, 0.75, 0.999):
        for settings in ((1.0, 0, 1.0, 0.0), (1.0, 2, 1.0, 0.0), (0.7, 0, 0.5, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.3), (1e30, 0, 1.0, 0.0), (1e-30, 0, 1.0, 0.0)):
            _check(x, torch.full((x.size(0),), u, device="cuda"), *settings)


def test_settings_that_only_the_device_knows(built_library):
    """NaN and numbers out of their range, in tensors."""
    x, _ = _logits(6, 100, torch.float32, seed=3)
    one = torch.ones(6, device="cuda")
    half = 0.5 * one
    nan = float("nan") * one
    plain = sspmm_amd.sample_tokens(x, half)
    greedy = x.argmax(1).int()
    for call, want in (((half, nan), greedy), ((half, -one), greedy), ((half, one, torch.full((6,), -7, dtype=torch.int32, device="cuda")), plain), ((half, one, 0, nan), plain),
                       ((half, one, 0, 2 * one), plain), ((half, one, 0, -one), greedy), ((half, one, 0, 1.0, nan), plain), ((half, one, 0, 1.0, -one), plain),
                       ((half, one, 0, 1.0, 3 * one), greedy)):
        assert torch.equal(sspmm_amd.sample_tokens(x, *call), want)
    last = sspmm_amd.sample_tokens(x, one - 2.0 ** -24)
    assert torch.equal(sspmm_amd.sample_tokens(x, one), last) and torch.equal(sspmm_amd.sample_tokens(x, 5 * one), last)
    first = sspmm_amd.sample_tokens(x, 0 * one)
    assert torch.equal(first, greedy) and torch.equal(sspmm_amd.sample_tokens(x, -one), first) and torch.equal(sspmm_amd.sample_tokens(x, nan), first)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("order", ["padded", "odd start", "turned", "one row for all", "every other row"])
def test_other_orders_in_memory(built_library, order, dtype):
    rows, vocab = 7, 1003
    base, uniform = _logits(2 * rows, vocab + 30, dtype, seed=8)
    if order == "padded":
        logits = base[:rows, 5:5 + vocab]
    elif order == "odd start":
        logits = base.flatten()[3:3 + rows * vocab].view(rows, vocab)
    elif order == "turned":
        logits = base.t()[:rows, :2 * rows]
    elif order == "one row for all":
        logits = base[3:4, 1:1 + vocab].expand(rows, vocab)
    else:
        logits = base[::2, :vocab]
    uniform = uniform[:rows].contiguous()
    _check(logits, uniform, 0.9, 30, 0.9)
    _check(logits, uniform)
    _check(logits, uniform, 0.0)


def test_nothing_is_read_beside_the_row(built_library):
    """Neighbours of the row, in the same 16 bytes, are larger than anything in it."""
    for dtype in TYPES:
        for start in range(9):
            for vocab in (1, 2, 7, 8, 9, 1025):
                base = torch.full((vocab + 40,), INF, dtype=dtype, device="cuda")
                base[16 + start:16 + start + vocab] = torch.arange(vocab, device="cuda").to(dtype) * 0.01
                _check(base[16 + start:16 + start + vocab][None], torch.tensor([0.7], device="cuda"), 1.0, 0, 0.9)


def test_captured_streams_and_twice_the_same(built_library):
    logits, uniform = _logits(50, 32003, torch.bfloat16, seed=10)
    settings = (0.8, 100, 0.95, 0.01)
    want = sspmm_amd.sample_tokens(logits, uniform, *settings)
    assert all(torch.equal(sspmm_amd.sample_tokens(logits, uniform, *settings), want) for _ in range(5))
    x, u = logits.clone(), uniform.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, chances = sspmm_amd.sample_tokens(x, u, *settings, probabilities=True)
    for turn in range(4):
        fresh, numbers = _logits(50, 32003, torch.bfloat16, seed=20 + turn)
        x.copy_(fresh)
        u.copy_(numbers)
        eager = sspmm_amd.sample_tokens(x, u, *settings, probabilities=True)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(tokens, eager[0]) and torch.equal(chances, eager[1])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        beside = sspmm_amd.sample_tokens(logits, uniform, *settings)
    stream.synchronize()
    assert torch.equal(beside, want)


@pytest.mark.parametrize("dtype", TYPES)
def test_first_ones_at_any_place(built_library, dtype):
    """Settings that list few logits of a row: rows that begin and end at any element, their first ones at the edges and in the middle, values of both signs."""
    for vocab in (1025, 5003, 33001):
        base = _logits(1, vocab + 40, dtype, seed=vocab)[0][0]
        for start in range(9):
            x = base.clone()
            row = x[16 + start:16 + start + vocab]
            x[:16 + start] = INF
            x[16 + start + vocab:] = INF
            row -= 14  # (all below zero)
            row[0], row[vocab - 1], row[vocab // 2] = 3.0, 2.5, 2.75
            for top_k in (1, 3, 20, 128):
                _check(row[None], torch.tensor([0.93], device="cuda"), 4.0, top_k, 0.99)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("alike", [1, 2, 255, 256, 257, 511, 513, 1500])
def test_equal_logits_among_others(built_library, dtype, alike):
    """So many equal ones, far apart in the row, at the place that is drawn; and logits about zero, whose order the signs decide."""
    vocab = 20000
    logits = _logits(3, vocab, dtype, seed=alike, spread=0.01)[0].float()
    at = torch.randperm(vocab, device="cuda", generator=torch.Generator(device="cuda").manual_seed(alike))[:alike]
    logits[0, at] = 1.5
    logits[1, at] = -0.0
    logits[2, at] = 0.0
    logits = logits.to(dtype)
    for u in (0.0, 0.3, 0.999):
        _check(logits, torch.full((3,), u, device="cuda"), 1.0)
        _check(logits, torch.full((3,), u, device="cuda"), 0.05, 0, 0.9)
        _check(logits, torch.full((3,), u, device="cuda"), 1.0, max(1, alike // 2))


def test_frequencies_are_the_probabilities(built_library):
    """A number for each of n equal parts of [0, 1): a token of probability p is drawn n p times, give or take one (its run has two ends)."""
    n, vocab = 4096, 37
    logits, _ = _logits(1, vocab, torch.float32, seed=12, spread=1.5)
    uniform = (torch.arange(n, device="cuda") + 0.5) / n
    tokens, chances = sspmm_amd.sample_tokens(logits.expand(n, vocab), uniform, 1.0, 0, 0.9, probabilities=True)
    counts = torch.bincount(tokens.long(), minlength=vocab).double()
    p = torch.zeros(vocab, dtype=torch.float64, device="cuda")
    p[tokens.long()] = chances.double()
    assert ((counts - n * p).abs() <= 1.001).all() and abs(float(p.sum()) - 1) < 1e-5


def test_rows_beyond_32_bits(built_library):
    rows, stride = 3, 1100000000
    base = torch.zeros(rows * stride, dtype=torch.bfloat16, device="cuda")
    logits = base.view(rows, stride)[:, stride - 500:]
    logits.copy_(_logits(rows, 500, torch.bfloat16, seed=13)[0])
    _check(logits, torch.tensor([0.1, 0.5, 0.9], device="cuda"), 1.0, 20, 0.9)


def test_refusals(built_library):
    x, u = _logits(4, 50, torch.float16, seed=2)
    sample = sspmm_amd.sample_tokens
    one = torch.ones(4, device="cuda")
    for call, kind in (((x.double(), u), TypeError), ((x.cpu(), u), TypeError), ((x[0], u), ValueError), ((x[:, :0], u), ValueError), ((x, u[:3]), ValueError), ((x, u.double()), TypeError),
                       ((x, u.cpu()), TypeError), ((x, torch.stack([u, u], 1)[:, 0]), TypeError), ((x, u, -1.0), ValueError), ((x, u, INF), ValueError), ((x, u, float("nan")), ValueError),
                       ((x, u, 1.0, -1), ValueError), ((x, u, 1.0, 1 << 31), ValueError), ((x, u, 1.0, 0, 1.5), ValueError), ((x, u, 1.0, 0, -0.1), ValueError),
                       ((x, u, 1.0, 0, 1.0, 2.0), ValueError), ((x, u, 1.0, 0, 1.0, float("nan")), ValueError), ((x, u, one.double()), TypeError), ((x, u, one[:2]), ValueError),
                       ((x, u, one, one), TypeError), ((x, u, one[:, None]), TypeError), ((x, u, one.cpu()), TypeError)):
        with pytest.raises(kind):
            sample(*call)
    with pytest.raises(RuntimeError, match="gradients"):
        sample(x.float().requires_grad_(), u)
    with pytest.raises(RuntimeError, match="gradients"):
        sample(x, u, one.clone().requires_grad_())
    assert sample(x[:0], u[:0]).shape == (0,)
