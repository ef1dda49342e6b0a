"""Drawn tokens of few rows of large vocabularies, which several workgroups share, against the rule in 64 bits: the same bounds as in test_sample_gpu.py."""
import pytest
import torch

import sspmm_amd
from sspmm_amd import _lib
from test_sample_gpu import INF, TYPES, _check, _logits

pytestmark = pytest.mark.gpu

# (rows, vocab): five parts of a row at the least vocabulary that has them and of as many rows as have them, six, seven, eight
SIZES = [(23, 81920), (102, 90001), (19, 98309), (21, 114689), (25, 131072)]


def _in_parts(logits):
    """Whether the call has a workspace, which only rows in parts want."""
    return _lib.lib().sspmm_sample_tokens_workspace_bytes(*logits.shape) > 0


def _mixed(rows):
    """Settings of every kind beside each other: rows that are listed, rows with bins, temperature 0."""
    i = torch.arange(rows, device="cuda")
    temperature = torch.tensor([0.7, 1.0, 0.0, 1.5, 0.3], device="cuda")[i % 5]
    top_k = torch.tensor([0, 50, 1, 1000, 1200, 1201, 60000, 7], dtype=torch.int32, device="cuda")[i % 8]
    top_p = torch.tensor([1.0, 0.9, 0.5], device="cuda")[i % 3]
    min_p = torch.tensor([0.0, 0.0, 0.05, 1e-4, 0.0, 1.0, 0.0], device="cuda")[i % 7]
    return temperature, top_k, top_p, min_p


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_every_row_its_own_settings(built_library, rows, vocab, dtype):
    logits, uniform = _logits(rows, vocab, dtype, seed=vocab)
    assert _in_parts(logits)
    _check(logits, uniform, *_mixed(rows))


@pytest.mark.parametrize("dtype", TYPES)
def test_settings_for_all_rows(built_library, dtype):
    """What the host knows decides how many launches there are."""
    logits, uniform = _logits(5, 81921, dtype, seed=1)
    for settings in ((0.0, 0, 1.0, 0.0), (0.0, 3, 0.5, 0.5), (2.0, 1, 1.0, 0.0), (1.0, 128, 1.0, 0.0), (1.0, 129, 0.9, 0.0), (0.8, 1200, 0.95, 0.02), (0.8, 1201, 0.95, 0.02), (1.0, 81921, 1.0, 0.0),
                     (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0), (1.0, 0, 1.0, 0.0), (1.0, 0, 0.9, 0.05)):
        _check(logits, uniform, *settings)
    cold = torch.tensor([0.0, 1.0, 0.0, 0.5, 2.0], device="cuda")
    _check(logits, uniform, cold)
    _check(logits, uniform, cold, 300)
    _check(logits, uniform, 0.0, torch.tensor([0, 5, 1, 2000, 90000], dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("falling", [True, False])
@pytest.mark.parametrize("vocab", [81920, 131072 - 5])
def test_sorted_rows(built_library, vocab, falling, dtype):
    """The first tokens side by side, at either end of the row."""
    logits, uniform = _logits(6, vocab, dtype, seed=vocab + falling)
    logits = logits.float().sort(1, descending=falling).values.to(dtype)
    assert _in_parts(logits)
    for settings in ((1.0, 1, 1.0, 0.0), (1.0, 60, 1.0, 0.0), (1.5, 100, 0.95, 0.0), (1.0, 500, 0.9, 0.0), (2.0, 1000, 1.0, 0.01), (1.0, 1200, 0.99, 0.0), (1.0, 0, 0.9, 0.0), (0.7, 5000, 1.0, 0.0)):
        _check(logits, uniform, *settings)
    _check(logits, uniform, *_mixed(6))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("start", [0, 40000, 81920 - 700])
def test_first_ones_in_one_place(built_library, start, dtype):
    """700 logits above all others, side by side in the middle or at an end: with a top_k below, of, and above as many."""
    logits, uniform = _logits(4, 81920, dtype, seed=start)
    logits[:, start:start + 700] += 40.0
    for top_k in (60, 350, 699, 700, 701, 1100):
        _check(logits, uniform, 3.0, top_k, 0.97)


@pytest.mark.parametrize("dtype", TYPES)
def test_equal_logits(built_library, dtype):
    """One logit everywhere, few levels with thousands of each, a level that only one stretch of the row has: lists that have no room, of a part and of all."""
    vocab = 98304
    g = torch.Generator(device="cuda").manual_seed(5)
    logits = torch.full((8, vocab), 2.5, dtype=dtype, device="cuda")
    logits[1] = torch.randint(0, 4, (vocab,), generator=g, device="cuda").to(dtype) * 0.5
    logits[2] = torch.randint(0, 40, (vocab,), generator=g, device="cuda").to(dtype) * 0.125
    logits[3, 20000:29000] = 4.0
    logits[4, :] = -1.0
    logits[4, 5::19] = 4.0
    logits[5, ::2] = -0.0
    logits[5, 1::2] = 0.0
    logits[6, vocab - 7000:] = 2.75
    logits[7, 90000] = 9.0
    assert _in_parts(logits)
    for u in (0.0, 0.41, 0.9999):
        uniform = torch.full((8,), u, device="cuda")
        for settings in ((1.0, 0, 1.0, 0.0), (1.0, 1, 1.0, 0.0), (1.0, 90, 1.0, 0.0), (1.0, 1200, 0.5, 0.0), (0.5, 9000, 0.7, 0.0), (1.0, 0, 0.5, 0.3), (0.0, 0, 1.0, 0.0)):
            _check(logits, uniform, *settings)


@pytest.mark.parametrize("dtype", TYPES)
def test_what_is_not_finite(built_library, dtype):
    """Rows of -infinity or NaN, stretches of these longer than a part, infinities in one place and in many, a row with one token."""
    vocab = 90112
    logits, _ = _logits(10, vocab, dtype, seed=6)
    logits[0] = -INF
    logits[1] = float("nan")
    logits[2, :40000] = -INF
    logits[3, 30000:] = float("nan")
    logits[4, 77777] = INF
    logits[5, 500::6001] = INF
    logits[6] = INF
    logits[7] = -INF
    logits[7, 60001] = -3.0
    logits[8, 1::2] = -INF
    logits[9, ::3] = float("nan")
    logits[9, 45000] = torch.finfo(dtype).max
    logits[9, 45001] = torch.finfo(dtype).min
    assert _in_parts(logits)
    for u in (0.0, 0.5, 0.999):
        uniform = torch.full((10,), u, device="cuda")
        for settings in ((1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 70, 1.0, 0.0), (1.0, 1000, 0.9, 0.0), (1.0, 5000, 0.9, 0.01), (1e30, 0, 1.0, 0.0), (1e-30, 0, 1.0, 0.0)):
            _check(logits, uniform, *settings)
        _check(logits, uniform, *_mixed(10))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("order", ["padded", "odd start", "one row for all", "every other row"])
def test_other_orders_in_memory(built_library, order, dtype):
    """Rows that begin at any element, with larger logits beside them."""
    rows, vocab = 9, 81931
    base, uniform = _logits(2 * rows, vocab + 30, dtype, seed=8)
    if order == "padded":
        base[:, :5] = INF
        base[:, 5 + vocab:] = INF
        logits = base[:rows, 5:5 + vocab]
    elif order == "odd start":
        logits = base.flatten()[3:3 + rows * vocab].view(rows, vocab)
    elif order == "one row for all":
        logits = base[3:4, 1:1 + vocab].expand(rows, vocab)
    else:
        logits = base[::2, :vocab]
    uniform = uniform[:rows].contiguous()
    _check(logits, uniform, *_mixed(rows))
    _check(logits, uniform, 0.9, 30, 0.9)
    for i in range(rows):  # (the first and last elements are the row's first ones)
        logits[i, 0], logits[i, vocab - 1] = 30.0, 29.5
    _check(logits, uniform, 1.0, 2)
    _check(logits, uniform)


def test_captured_streams_and_twice_the_same(built_library):
    """Two graphs and two streams have workspaces of their own, and a call the same result every time."""
    rows, vocab = 16, 90001
    sets = [_logits(rows, vocab, torch.bfloat16, seed=10 + i) for i in range(2)]
    settings = _mixed(rows)
    assert _in_parts(sets[0][0])
    want = [sspmm_amd.sample_tokens(x, u, *settings, probabilities=True) for x, u in sets]
    for turn in range(5):
        for (x, u), (tokens, chances) in zip(sets, want):
            again = sspmm_amd.sample_tokens(x, u, *settings, probabilities=True)
            assert torch.equal(again[0], tokens) and torch.equal(again[1], chances)
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in sets], []
    for (x, u), g in zip(sets, graphs):
        with torch.cuda.graph(g):
            outs.append(sspmm_amd.sample_tokens(x, u, *settings, probabilities=True))
    for turn in range(4):
        for i, (x, u) in enumerate(sets):
            fresh, numbers = _logits(rows, vocab, torch.bfloat16, seed=30 + 2 * turn + i)
            x.copy_(fresh.sort(1, descending=True).values if turn % 2 else fresh)
            u.copy_(numbers)
        want = [sspmm_amd.sample_tokens(x, u, *settings, probabilities=True) for x, u in sets]
        for g in graphs if turn % 2 else graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        for out, (tokens, chances) in zip(outs, want):
            assert torch.equal(out[0], tokens) and torch.equal(out[1], chances)
    _check(*sets[0], *settings)
    streams, got = [torch.cuda.Stream() for _ in sets], []
    torch.cuda.synchronize()
    for turn in range(6):
        for s, (x, u) in zip(streams, sets):
            with torch.cuda.stream(s):
                got.append(sspmm_amd.sample_tokens(x, u, *settings, probabilities=True))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert torch.equal(out[0], want[i % 2][0]) and torch.equal(out[1], want[i % 2][1])


def _in_turn(*calls):
    """us of each call: medians of captured runs of 20, timed in turn."""
    graphs, times = [], [[] for _ in calls]
    for call in calls:
        call()
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            for _ in range(20):
                call()
    for turn in range(9):
        for graph, took in zip(graphs, times):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            graph.replay()
            end.record()
            end.synchronize()
            took.append(begin.elapsed_time(end) * 1e3 / 20)
    return [sorted(took)[len(took) // 2] for took in times]


@pytest.mark.parametrize("order", ["likely ones first", "sorted"])
@pytest.mark.parametrize("top_k", [100, 200, 1000])
def test_likely_tokens_side_by_side_take_no_longer(built_library, top_k, order):
    """The parts' lists suffice, wherever a row's first tokens lie: in less than three times the time of the same logits in any order (the lists are up to eight times as long
    where they are sorted, 1.05 to 1.75 times the time; the whole row by one workgroup takes 3.9 to 13 times)."""
    rows, vocab = 64, 131072
    x, uniform = _logits(rows, vocab, torch.float32, seed=top_k, spread=2.0)
    x = x.sort(1, descending=True).values if order == "sorted" else x - 0.8 * torch.log(1.0 + torch.arange(vocab, device="cuda"))
    anywhere = x[:, torch.randperm(vocab, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")]
    x, anywhere = x.bfloat16(), anywhere.bfloat16().contiguous()
    for logits in (x, anywhere):
        _check(logits[:2], uniform[:2], 0.8, top_k)
    first, other = _in_turn(lambda: sspmm_amd.sample_tokens(x, uniform, 0.8, top_k), lambda: sspmm_amd.sample_tokens(anywhere, uniform, 0.8, top_k))
    assert first < 3 * other, "%.1f us, in any order %.1f" % (first, other)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(40, 20000), (12, 131072)])
def test_tokens_ruled_out_by_a_low_number(built_library, rows, vocab, dtype):
    """Few tokens are left, fewer than top_k, and the others have the type's lowest value, or one that is far enough below: as if it were -infinity, also in its time (with lists that overflow eight
    times as long)."""
    logits, uniform = _logits(rows, vocab, dtype, seed=vocab)
    out = torch.rand(rows, vocab, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda") >= 20 / vocab
    out[:, 7] = False
    never = logits.masked_fill(out, -INF)
    for low in (torch.finfo(dtype).min, -1e4):
        lowest = logits.masked_fill(out, low)
        for settings in ((0.8, 10, 1.0, 0.0), (0.8, 50, 0.9, 0.0), (0.8, 1000, 1.0, 0.01), (0.0, 0, 1.0, 0.0), (0.8, 0, 1.0, 0.0)):
            _check(lowest, uniform, *settings)
            assert torch.equal(sspmm_amd.sample_tokens(lowest, uniform, *settings), sspmm_amd.sample_tokens(never, uniform, *settings))
        for temperature in (1e4, 1e38):  # (where they count again)
            _check(lowest, uniform, temperature, 50)
        for top_k in (10, 50, 1000) if _in_parts(lowest) else ():
            took, other = _in_turn(lambda: sspmm_amd.sample_tokens(lowest, uniform, 0.8, top_k), lambda: sspmm_amd.sample_tokens(never, uniform, 0.8, top_k))
            assert took < 4 * other, "top_k %d: %.1f us, with -infinity %.1f" % (top_k, took, other)
