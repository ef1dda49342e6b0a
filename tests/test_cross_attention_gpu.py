"""Attention of packed queries over packed states of other lengths, against the formula in 64 bits."""
import math

import pytest
import torch

import sspmm_amd
from serving_util import attention, check, offsets_of

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16]


def _randn(shape, seed, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _inputs(lengths, sources, heads, kv, d, dtype, seed=0):
    kvs = _randn((sum(sources), 2, kv, d), seed + 1, dtype)
    return _randn((sum(lengths), heads, d), seed, dtype), kvs[:, 0], kvs[:, 1]


def _check(got, q, k, v, lengths, sources, scale, what=""):
    group, i, j = q.size(1) // k.size(1), 0, 0
    for n, m in zip(lengths, sources):
        for h in range(q.size(1) if n else 0):
            if m == 0:
                assert not got[i:i + n, h].any(), "%s: queries at %d have no states" % (what, i)
                continue
            want, off = attention(q[i:i + n, h], k[j:j + m, h // group], v[j:j + m, h // group], torch.full((n,), m, device="cuda"), scale, q.dtype, q.dtype)
            check(got[i:i + n, h], want, off, "%s %d queries at %d on %d states, head %d" % (what, n, i, m, h))
        i, j = i + n, j + m


def _run(lengths, sources, heads, kv, d, dtype, seed=0, **more):
    q, k, v = _inputs(lengths, sources, heads, kv, d, dtype, seed)
    print(lengths, sources, heads, kv, d, dtype, flush=True)
    got = sspmm_amd.cross_attention(q, k, v, offsets_of(lengths), offsets_of(sources), **more)
    _check(got, q, k, v, lengths, sources, more.get("scaling") or d ** -0.5)
    return q, k, v, got


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,sources,heads,kv", [([1], [1], 1, 1), ([1], [700], 4, 2), ([2, 0, 65, 1], [5, 9, 0, 64], 4, 2), ([63, 33, 31], [1, 65, 300], 3, 1), ([300], [3], 2, 2),
                                                      ([129, 1, 7], [128, 129, 31], 6, 2), ([1] * 9, [0, 1, 2, 63, 64, 65, 200, 0, 31], 8, 1), ([5] * 4, [90, 0, 17, 256], 16, 2),
                                                      ([17, 3], [513, 1025], 24, 1)])
def test_against_the_formula(built_library, lengths, sources, heads, kv, dtype, d):
    _run(lengths, sources, heads, kv, d, dtype, seed=len(lengths) + d)


@pytest.mark.parametrize("lengths,sources,heads,kv,d", [([1], [20011], 8, 2, 128), ([3], [9001], 4, 4, 64), ([1] * 70, [(37 * i * i) % 900 for i in range(70)], 8, 8, 64),
                                                        ([1, 1, 400, 1], [2000, 10, 1500, 3000], 8, 2, 128), ([1500, 900], [1100, 2500], 4, 2, 128), ([16] * 3, [4000, 1, 5000], 8, 8, 32),
                                                        ([2000], [40], 2, 1, 64), ([1] * 300, [11] * 300, 4, 2, 64)])
def test_longer_and_more(built_library, lengths, sources, heads, kv, d):
    _run(lengths, sources, heads, kv, d, torch.bfloat16, seed=3)


def test_thousands_of_single_tokens(built_library):
    n = 3000
    lengths, sources = [1 if i % 7 else 0 for i in range(n)], [(13 * i) % 50 for i in range(n)]
    q, k, v = _inputs(lengths, sources, 2, 1, 32, torch.float16, seed=4)
    got = sspmm_amd.cross_attention(q, k, v, offsets_of(lengths), offsets_of(sources))
    at = [i for i in range(n) if lengths[i]]
    for row in list(range(0, len(at), 97)) + [len(at) - 1]:
        i = at[row]
        j = sum(sources[:i])
        for h in range(2):
            if sources[i] == 0:
                assert not got[row, h].any()
                continue
            want, off = attention(q[row:row + 1, h], k[j:j + sources[i], 0], v[j:j + sources[i], 0], torch.tensor([sources[i]], device="cuda"), 32 ** -0.5, q.dtype, q.dtype)
            check(got[row:row + 1, h], want, off, "sequence %d" % i)


@pytest.mark.parametrize("n", [33000, 300000])
def test_more_sequences_than_a_batch(built_library, n):
    """One token each, of tens and hundreds of thousands of sequences with up to four states."""
    heads, kv, d = 16, 8, 32
    sources = torch.arange(n, device="cuda") % 5
    offsets, source_offsets = torch.arange(n + 1, dtype=torch.int32, device="cuda"), torch.cat([sources.new_zeros(1), sources.cumsum(0)]).int()
    q = _randn((n, heads, d), 1, torch.float16)
    kvs = _randn((int(source_offsets[-1]), 2, kv, d), 2, torch.float16)
    got = sspmm_amd.cross_attention(q, kvs[:, 0], kvs[:, 1], offsets, source_offsets)
    assert not got[sources == 0].any()
    for i in list(range(0, n, n // 40)) + list(range(n - 6, n)):
        at, m = int(source_offsets[i]), int(sources[i])
        for h in range(heads) if m else ():
            want, off = attention(q[i:i + 1, h], kvs[at:at + m, 0, h // 2], kvs[at:at + m, 1, h // 2], torch.tensor([m], device="cuda"), d ** -0.5, q.dtype, q.dtype)
            check(got[i:i + 1, h], want, off, "sequence %d" % i)


@pytest.mark.parametrize("scaling", [1e-3, 0.125, 3.0, 100.0])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,sources", [([1, 3], [300, 77]), ([150, 20], [300, 77])])
def test_scores_small_and_large(built_library, dtype, scaling, lengths, sources):
    _run(lengths, sources, 4, 2, 64, dtype, seed=6, scaling=scaling)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 140])
def test_maxima_that_grow_along_the_states(built_library, dtype, n):
    lengths, sources, d = [n], [900], 64
    q, k, v = _inputs(lengths, sources, 2, 1, d, dtype, seed=7)
    q = q.abs()
    k = (k.abs() * torch.linspace(0.1, 6.0, 900, device="cuda")[:, None, None]).to(dtype)
    got = sspmm_amd.cross_attention(q, k, v, offsets_of(lengths), offsets_of(sources))
    _check(got, q, k, v, lengths, sources, d ** -0.5)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 3, 130])
def test_a_neighbour_that_is_not_finite(built_library, dtype, bad, n):
    """States of the sequences in front and behind, in the same tiles, are seen by nobody else."""
    lengths, sources, d = [n, n, n], [45, 77, 60], 64
    q, k, v = _inputs(lengths, sources, 4, 2, d, dtype, seed=9)
    k, v = k.clone(), v.clone()
    for t in (k, v):
        t[:45] = bad
        t[45 + 77:] = bad
    got = sspmm_amd.cross_attention(q, k, v, offsets_of(lengths), offsets_of(sources))
    group = 2
    for h in range(4):
        want, off = attention(q[n:2 * n, h], k[45:122, h // group], v[45:122, h // group], torch.full((n,), 77, device="cuda"), d ** -0.5, dtype, dtype)
        check(got[n:2 * n, h], want, off, "head %d" % h)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 130])
def test_infinities_in_the_values_of_the_sequence(built_library, dtype, n):
    """An infinite value reaches every query of its sequence, however small its probability."""
    lengths, sources, d = [n, n], [200, 90], 64
    q, k, v = _inputs(lengths, sources, 2, 1, d, dtype, seed=10)
    v = v.clone()
    v[3, 0, 5], v[150, 0, 7], v[250, 0, 9] = float("inf"), float("-inf"), float("nan")
    got = sspmm_amd.cross_attention(q, k, v, offsets_of(lengths), offsets_of(sources))
    _check(got, q, k, v, lengths, sources, d ** -0.5)


@pytest.mark.parametrize("n", [1, 130])
def test_scores_of_minus_infinity_only_are_zeros(built_library, n):
    q, k, v = _inputs([n], [70], 2, 2, 32, torch.float16, seed=11)
    q = q.abs() + 0.1
    k = torch.full_like(k, float("-inf"))
    assert not sspmm_amd.cross_attention(q, k, v, offsets_of([n]), offsets_of([70])).any()


@pytest.mark.parametrize("lengths", [[4, 3], [140, 30]])
def test_rows_of_no_sequence_stay_as_they_were(built_library, lengths):
    total = sum(lengths)
    q, k, v = _inputs([total + 9], [100], 4, 2, 64, torch.float16, seed=12)
    offsets = offsets_of(lengths) + 5
    out = torch.full_like(q, 7.0)
    got = sspmm_amd.cross_attention(q, k, v, offsets, torch.tensor([0, 60, 90], dtype=torch.int32, device="cuda"), out=out)
    assert got is out and (out[:5] == 7).all() and (out[5 + total:] == 7).all()
    _check(out[5:5 + total], q[5:5 + total], k, v, lengths, [60, 30], 0.125)


@pytest.mark.parametrize("n", [2, 90])
def test_offsets_outside_are_taken_to_the_ends(built_library, n):
    q, k, v = _inputs([2 * n], [100], 2, 1, 64, torch.float16, seed=13)
    offsets = torch.tensor([-5, n, 5000], dtype=torch.int32, device="cuda")
    sources = torch.tensor([-9, 30, 1 << 30], dtype=torch.int32, device="cuda")
    got = sspmm_amd.cross_attention(q, k, v, offsets, sources)
    _check(got, q, k, v, [n, n], [30, 70], 0.125)
    falling = torch.tensor([60, 20, 100], dtype=torch.int32, device="cuda")  # (the first sequence has no states)
    got = sspmm_amd.cross_attention(q, k, v, offsets, falling)
    assert not got[:n].any()
    _check(got[n:], q[n:], k[20:], v[20:], [n], [80], 0.125)


@pytest.mark.parametrize("order", ["fused projections", "heads in front", "features apart", "odd start"])
@pytest.mark.parametrize("lengths,sources", [([1, 2], [300, 70]), ([140, 3], [300, 70])])
def test_other_orders_in_memory(built_library, order, lengths, sources):
    heads, kv, d, n, m = 4, 2, 64, sum(lengths), sum(sources)
    if order == "fused projections":
        q = _randn((n, heads * d + 32), 1, torch.float16)[:, 32:].view(n, heads, d)
        k, v = _randn((m, 3, kv, d), 2, torch.float16)[:, 1:].unbind(1)
        out = torch.zeros(n, heads * d + 64, device="cuda", dtype=torch.float16)[:, 64:].view(n, heads, d)
    elif order == "heads in front":
        q, k, v = _randn((heads, n, d), 1, torch.float16).transpose(0, 1), _randn((kv, m, d), 2, torch.float16).transpose(0, 1), _randn((kv, m, d), 3, torch.float16).transpose(0, 1)
        out = torch.zeros(heads, n, d, device="cuda", dtype=torch.float16).transpose(0, 1)
    elif order == "features apart":
        q, k, v = (_randn((heads * d, n), 1, torch.float16).t().view(n, heads, d), _randn((kv * d, m), 2, torch.float16).t().view(m, kv, d),
                   _randn((kv * d, m), 3, torch.float16).t().view(m, kv, d))
        out = None
    else:
        q, k, v = (_randn((rows * width * d + 5,), seed, torch.float16)[5:].view(rows, width, d) for rows, width, seed in ((n, heads, 1), (m, kv, 2), (m, kv, 3)))
        out = None
    got = sspmm_amd.cross_attention(q, k, v, offsets_of(lengths), offsets_of(sources), out=out)
    _check(got, q, k, v, lengths, sources, 0.125)


@pytest.mark.parametrize("lengths", [[1, 1, 1], [3, 0, 5], [200, 1, 31]])
def test_in_place(built_library, lengths):
    sources = [50, 80, 4000]
    q, k, v = _inputs(lengths, sources, 8, 2, 64, torch.bfloat16, seed=15)
    want = sspmm_amd.cross_attention(q, k, v, offsets_of(lengths), offsets_of(sources))
    got = sspmm_amd.cross_attention(q, k, v, offsets_of(lengths), offsets_of(sources), out=q)
    assert got is q and torch.equal(got, want)


@pytest.mark.parametrize("lengths,sources", [([1, 1], [3000, 1700]), ([150, 9], [700, 100])])
def test_captured_streams_and_twice_the_same(built_library, lengths, sources):
    """The graph reads the lists when it is replayed; two graphs, and calls on two streams at once, have workspaces of their own."""
    heads, kv, d = 8, 2, 128
    q, k, v = _inputs(lengths, sources, heads, kv, d, torch.bfloat16, seed=16)
    qs, offsets, states = [q, q.flip(0).contiguous()], offsets_of(lengths), offsets_of(sources)
    first = sspmm_amd.cross_attention(q, k, v, offsets, states)
    assert all(torch.equal(sspmm_amd.cross_attention(q, k, v, offsets, states), first) for _ in range(3))
    torch.cuda.synchronize()
    outs, graphs = [torch.zeros_like(q) for _ in qs], [torch.cuda.CUDAGraph() for _ in qs]
    for x, out, g in zip(qs, outs, graphs):
        with torch.cuda.graph(g):
            sspmm_amd.cross_attention(x, k, v, offsets, states, out=out)
    for turn in range(4):
        states.copy_(offsets_of([sources[0] - 100 * turn, sources[1] + 100 * turn]))
        for i, x in enumerate(qs):
            x.copy_(_randn(x.shape, 50 + 2 * turn + i, x.dtype))
        want = [sspmm_amd.cross_attention(x, k, v, offsets, states) for x in qs]
        for g in graphs if turn % 2 else graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for turn in range(6):
        for s, x in zip(streams, qs):
            with torch.cuda.stream(s):
                got.append(sspmm_amd.cross_attention(x, k, v, offsets, states))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i % 2]) for i, x in enumerate(got))


@pytest.mark.parametrize("n", [1, 130])
def test_states_further_apart_than_32_bits_reach(built_library, n):
    m, pitch = 300, (1 << 23) - 64
    base = torch.zeros(m * pitch, dtype=torch.float16, device="cuda")
    kv = base.view(m, pitch)[:, :256].view(m, 2, 2, 64)
    kv.copy_(_randn((m, 2, 2, 64), 17, torch.float16))
    k, v = kv.unbind(1)
    q = _randn((n, 4, 64), 18, torch.float16)
    got = sspmm_amd.cross_attention(q, k, v, offsets_of([n]), offsets_of([m]))
    _check(got, q, k.contiguous(), v.contiguous(), [n], [m], 0.125)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 130])
def test_scores_far_beyond_what_32_bits_resolve(built_library, dtype, n):
    """Scores near 2^27 that differ by a few thousand: the largest probability is one and the others nothing, wherever the reference point is rounded to."""
    m, d = 600, 64
    q = torch.full((n, 2, d), 64.0, device="cuda", dtype=dtype)
    k = torch.full((m, 1, d), 128.0, device="cuda", dtype=dtype)
    k[77, 0, :8] = 129.0
    v = _randn((m, 1, d), 19, dtype)
    got = sspmm_amd.cross_attention(q, k, v, offsets_of([n]), offsets_of([m]), scaling=256.0)
    assert torch.equal(got, v[77].expand(n, 2, d))


@pytest.mark.parametrize("n", [1, 130])
def test_values_at_the_end_of_the_range(built_library, n):
    m, d = 200, 64
    q, k, v = _inputs([n], [m], 2, 1, d, torch.bfloat16, seed=20)
    v = (torch.sign(v.float()) * 3.0e38).to(torch.bfloat16)
    v[:, 0, 0] = 3.0e38
    got = sspmm_amd.cross_attention(q, k, v, offsets_of([n]), offsets_of([m]))
    assert torch.isfinite(got).all()
    _check(got, q, k, v, [n], [m], 0.125)


def test_refusals(built_library):
    q, k, v = _inputs([5], [9], 4, 2, 64, torch.float16)
    a, b = offsets_of([5]), offsets_of([9])
    cross = sspmm_amd.cross_attention
    for call, kind in (((q.float(), k, v, a, b), TypeError), ((q, k.bfloat16(), v, a, b), TypeError), ((q, k, v.cpu(), a, b), TypeError), ((q[None], k, v, a, b), ValueError),
                       ((q, k, v[:8], a, b), ValueError), ((q, k[..., :32], v[..., :32], a, b), ValueError), ((q[:, :3], k, v, a, b), ValueError), ((q, k, v, a.long(), b), TypeError),
                       ((q, k, v, a, b.cpu()), TypeError), ((q, k, v, a, b[:1]), ValueError), ((q, k, v, a[:0], b[:0]), ValueError), ((q, k, v, a, b, 0.0), ValueError),
                       ((q, k, v, a, b, float("inf")), ValueError), ((q, k, v, a, b, None, q[:4]), ValueError), ((q, k, v, a, b, None, q.expand(5, 4, 64)[:, :1].expand(5, 4, 64)), ValueError)):
        with pytest.raises(kind):
            cross(*call)
    with pytest.raises(RuntimeError, match="gradients"):
        cross(q.clone().requires_grad_(), k, v, a, b)
    with pytest.raises(RuntimeError, match="gradients"):
        cross(q, k, v.clone().requires_grad_(), a, b)
    # nothing to do, and nothing to see
    assert cross(q[:0], k, v, offsets_of([0]), b).shape == (0, 4, 64)
    assert not cross(q, k[:0], v[:0], a, offsets_of([0])).any()
    same = q.clone()
    assert torch.equal(cross(q, k, v, a[:1], b[:1], out=same), q)  # no sequence: nothing is written
