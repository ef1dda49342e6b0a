"""Attention over packed prompts against the formula in 64 bits."""
import math

import pytest
import torch

import sspmm_amd
from serving_util import attention, check, check_prompt, offsets_of

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16]


def _projection(tokens, heads, kv, d, dtype, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(tokens, (heads + 2 * kv) * d, generator=g, device="cuda").to(dtype)
    return (x[:, :heads * d].view(tokens, heads, d), x[:, heads * d:(heads + kv) * d].view(tokens, kv, d), x[:, (heads + kv) * d:].view(tokens, kv, d))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,heads,kv", [([1], 1, 1), ([2, 0, 65, 1], 4, 2), ([63, 64, 31, 32, 33], 3, 1), ([127, 128, 129], 2, 2), ([300, 5], 6, 2),
                                              ([257, 0, 0, 96], 8, 8), ([150], 16, 8), ([700], 2, 1)])
def test_against_the_formula(built_library, lengths, heads, kv, dtype, d, causal):
    q, k, v = _projection(sum(lengths), heads, kv, d, dtype, seed=len(lengths) + d)
    print(lengths, heads, kv, dtype, d, causal, flush=True)
    got = sspmm_amd.prompt_attention(q, k, v, offsets_of(lengths), causal=causal)
    check_prompt(got, q, k, v, lengths, causal, 1 / math.sqrt(d))


@pytest.mark.parametrize("lengths,heads,kv,causal", [([2500, 1100], 4, 1, True), ([3001], 8, 8, True), ([1900, 2300], 2, 2, False)])
def test_longer_ones(built_library, lengths, heads, kv, causal):
    q, k, v = _projection(sum(lengths), heads, kv, 128, torch.bfloat16, seed=3)
    got = sspmm_amd.prompt_attention(q, k, v, offsets_of(lengths), causal=causal)
    check_prompt(got, q, k, v, lengths, causal, 128 ** -0.5)


def test_hundreds_of_short_sequences(built_library):
    lengths = [(7 * i * i + 3) % 40 for i in range(300)]
    q, k, v = _projection(sum(lengths), 4, 4, 64, torch.float16, seed=5)
    got = sspmm_amd.prompt_attention(q, k, v, offsets_of(lengths))
    check_prompt(got, q, k, v, lengths, True, 0.125)


@pytest.mark.parametrize("scaling", [1e-3, 0.125, 3.0, 100.0])
@pytest.mark.parametrize("dtype", TYPES)
def test_scores_small_and_large(built_library, dtype, scaling):
    lengths = [200, 77]
    q, k, v = _projection(sum(lengths), 2, 1, 64, dtype, seed=6)
    got = sspmm_amd.prompt_attention(q, k, v, offsets_of(lengths), scaling=scaling)
    check_prompt(got, q, k, v, lengths, True, scaling)


@pytest.mark.parametrize("causal", [True, False])
def test_maxima_that_grow_along_the_sequence(built_library, causal):
    """Every tile's maximum is far above the one before: the reference point moves each time."""
    n = 500
    q, k, v = _projection(n, 2, 2, 64, torch.float16, seed=7)
    k = (k * torch.linspace(0.1, 8, n, device="cuda")[:, None, None]).half()
    got = sspmm_amd.prompt_attention(q, k, v, offsets_of([n]), causal=causal, scaling=1.0)
    check_prompt(got, q, k, v, [n], causal, 1.0)


def test_many_small_probabilities_beside_a_large_one(built_library):
    """The sum is of the exponentials, not of what fp16 makes of them: 8000 keys of 2^-26 are together a part in 8000 of the one that is 1."""
    n, d = 8000, 64
    q = torch.zeros(n, 1, d, device="cuda", dtype=torch.float16)
    k = torch.zeros_like(q)
    q[-1, 0, 0], k[0, 0, 0] = 1.0, 26.0 * math.log(2)
    v = torch.ones_like(q)
    v[0] = 0.0
    got = sspmm_amd.prompt_attention(q, k, v, offsets_of([n]), scaling=1.0)
    want, off = attention(q[-1:, 0], k[:, 0], v[:, 0], torch.tensor([n], device="cuda"), 1.0, torch.float16, torch.float16)
    check(got[-1:, 0], want, off)
    v[0] = 1.0  # all ones: the result is one, whatever was rounded on the way, to what fp16 leaves out of these keys
    got = sspmm_amd.prompt_attention(q, k, v, offsets_of([n]), scaling=1.0)
    assert (got[-1].float() - 1).abs().max() <= n * 2.0 ** -26 + 2.0 ** -11


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [32, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_nothing_comes_from_masked_places(built_library, dtype, d, bad):
    """NaN and infinities in k and v of tokens that a query does not see: later ones, other sequences', and rows behind the last."""
    lengths = [130, 70, 1, 40]
    q, k, v = (t.clone() for t in _projection(sum(lengths) + 30, 4, 2, d, dtype, seed=8))
    k[sum(lengths):], v[sum(lengths):] = bad, bad
    q[sum(lengths):] = bad
    for at in (100, 129, 195, 200 + 1 + 5):  # tokens of three of the sequences
        v[at, 0, 3] = bad
        k[at, 1] = bad if bad != bad else k[at, 1]
    got = sspmm_amd.prompt_attention(q, k, v, offsets_of(lengths))
    # keys that are NaN: whoever sees one gets NaN, all others a finite result
    group, at = 2, 0
    for n in lengths:
        for h in range(4):
            qq, kk, vv = q[at:at + n, h], k[at:at + n, h // group], v[at:at + n, h // group]
            nan_key = torch.isnan(kk).any(-1)
            sees_nan = torch.cumsum(nan_key.int(), 0) > 0
            visible = torch.arange(1, n + 1, device="cuda")
            want, off = attention(qq, torch.where(nan_key[:, None], 0.0, kk.double()), vv, visible, d ** -0.5, dtype, dtype)
            rows = ~sees_nan
            check(got[at:at + n, h][rows], want[rows], off[rows], "head %d at %d" % (h, at))
            assert torch.isnan(got[at:at + n, h][sees_nan]).all()
        at += n


def test_both_infinities_in_the_last_tile(built_library):
    n = 40
    q, k, v = (t.clone() for t in _projection(n, 1, 1, 64, torch.bfloat16, seed=9))
    v[10, 0, 0], v[20, 0, 0], v[15, 0, 1], v[12, 0, 40] = float("inf"), float("-inf"), float("-inf"), float("nan")
    got = sspmm_amd.prompt_attention(q, k, v, offsets_of([n]))[:, 0]
    assert torch.isfinite(got[:10]).all() and (got[10:20, 0] == float("inf")).all() and torch.isnan(got[20:, 0]).all()
    assert (got[15:, 1] == float("-inf")).all() and torch.isfinite(got[:15, 1]).all() and torch.isnan(got[12:, 40]).all() and torch.isfinite(got[:, 2:40]).all()


def test_scores_of_minus_infinity_only_are_zeros(built_library):
    q = torch.full((3, 1, 32), float("-inf"), device="cuda", dtype=torch.float16)
    k = torch.ones_like(q)
    got = sspmm_amd.prompt_attention(q, k, torch.ones_like(q), offsets_of([3]))
    assert not got.any()


def test_rows_of_no_sequence_stay_as_they_were(built_library):
    lengths = [50, 0, 30]
    q, k, v = _projection(100, 2, 1, 64, torch.float16, seed=10)
    out = torch.full((100, 2, 64), 7.0, device="cuda", dtype=torch.float16)
    offsets = offsets_of(lengths) + 5  # tokens 0 .. 4 and 85 .. belong to nobody
    got = sspmm_amd.prompt_attention(q, k, v, offsets, out=out)
    assert got is out and (out[:5] == 7).all() and (out[85:] == 7).all()
    check_prompt(out[5:85], q[5:85], k[5:85], v[5:85], lengths, True, 0.125)


def test_offsets_outside_the_tokens_are_taken_to_their_ends(built_library):
    q, k, v = _projection(60, 2, 2, 32, torch.float16, seed=11)
    out = torch.full((60, 2, 32), 7.0, device="cuda", dtype=torch.float16)
    offsets = torch.tensor([-9, 20, 10, 50, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    # 0 .. 19; 20 .. 9, nothing; 10 .. 49; 50 .. 59
    sspmm_amd.prompt_attention(q, k, v, offsets[[0, 1]].contiguous(), out=out)
    check_prompt(out[:20], q[:20], k[:20], v[:20], [20], True, 32 ** -0.5)
    sspmm_amd.prompt_attention(q, k, v, offsets[[1, 2]].contiguous(), out=out)
    sspmm_amd.prompt_attention(q, k, v, offsets[[2, 3, 4]].contiguous(), out=out)
    check_prompt(out[10:], q[10:], k[10:], v[10:], [40, 10], True, 32 ** -0.5)


@pytest.mark.parametrize("order", ["heads first", "features first", "odd start", "out"])
def test_other_orders_in_memory(built_library, order):
    lengths, heads, kv, d = [90, 33], 4, 2, 64
    q, k, v = _projection(123, heads, kv, d, torch.bfloat16, seed=12)
    want = sspmm_amd.prompt_attention(q, k, v, offsets_of(lengths))
    out = None
    if order == "heads first":
        q, k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    elif order == "features first":  # as the SpMM leaves projections
        q, k, v = (t.permute(1, 2, 0).contiguous().permute(2, 0, 1) for t in (q, k, v))
    elif order == "odd start":
        q, k, v = (torch.nn.functional.pad(t.reshape(-1), (3, 0))[3:].view(t.shape) for t in (q, k, v))
        assert q.data_ptr() % 16
    else:
        out = torch.zeros(heads, 123, d + 8, device="cuda", dtype=torch.bfloat16)[:, :, :d].transpose(0, 1)
    got = sspmm_amd.prompt_attention(q, k, v, offsets_of(lengths), out=out)
    assert torch.equal(got, want)


def test_rows_further_apart_than_32_bits_reach(built_library):
    n, pitch = 520, 1 << 22  # 4.4 GB
    room = torch.empty(n * pitch, dtype=torch.float16, device="cuda")
    x = room.view(n, pitch)
    g = torch.Generator(device="cuda")
    g.manual_seed(13)
    q, k, v = (x[:, i * 64:(i + 1) * 64].view(n, 1, 64) for i in range(3))
    for t in (q, k, v):
        t.copy_(torch.randn(n, 1, 64, generator=g, device="cuda"))
    out = x[:, 1024:1088].view(n, 1, 64)
    sspmm_amd.prompt_attention(q, k, v, offsets_of([n]), out=out)
    check_prompt(out, q, k, v, [n], True, 0.125)


def test_captured_replayed_and_called_beside_it(built_library):
    lengths = [300, 77]
    q, k, v = (t.clone() for t in _projection(377, 8, 8, 128, torch.bfloat16, seed=14))
    offsets, out = offsets_of(lengths), torch.zeros(377, 8, 128, device="cuda", dtype=torch.bfloat16)
    eager = sspmm_amd.prompt_attention(q, k, v, offsets)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sspmm_amd.prompt_attention(q, k, v, offsets, out=out)
    for seed in range(4):
        q.copy_(_projection(377, 8, 8, 128, torch.bfloat16, seed=20 + seed)[0])
        offsets.copy_(offsets_of([100 + seed, 277 - seed]))  # (the graph reads them anew)
        want = sspmm_amd.prompt_attention(q, k, v, offsets)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert eager.shape == out.shape


def test_on_another_stream(built_library):
    q, k, v = _projection(200, 4, 2, 64, torch.float16, seed=15)
    offsets = offsets_of([200])
    want = sspmm_amd.prompt_attention(q, k, v, offsets)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = sspmm_amd.prompt_attention(q, k, v, offsets)
    s.synchronize()
    assert torch.equal(got, want)


def test_refusals(built_library):
    q, k, v = _projection(10, 4, 2, 64, torch.float16)
    offsets = offsets_of([10])
    call = sspmm_amd.prompt_attention
    for bad, kind in (((q.float(), k, v, offsets), TypeError), ((q, k.bfloat16(), v, offsets), TypeError), ((q, k, v, offsets.long()), TypeError),
                      ((q, k, v, offsets.cpu()), TypeError), ((q.cpu(), k.cpu(), v.cpu(), offsets), TypeError), ((q[:, :3], k, v, offsets), ValueError),
                      ((q, k[:, :, :32], v[:, :, :32], offsets), ValueError), ((q[:, :, :48], k[:, :, :48], v[:, :, :48], offsets), ValueError),
                      ((q, k[:9], v[:9], offsets), ValueError), ((q[0], k[0], v[0], offsets), ValueError), ((q, k, v, offsets[None]), ValueError),
                      ((q, k, v, offsets[:0]), ValueError), ((q, k[:, :0], v[:, :0], offsets), ValueError)):
        with pytest.raises(kind):
            call(*bad)
    for scaling in (0.0, -1.0, float("nan"), float("inf"), 3e38):
        with pytest.raises(ValueError):
            call(q, k, v, offsets, scaling=scaling)
    with pytest.raises(ValueError):
        call(q, k, v, offsets, out=torch.empty(10, 4, 64, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        call(q, k, v, offsets, out=torch.empty(10, 64, 4, device="cuda", dtype=torch.float16).transpose(1, 2))
    with pytest.raises(RuntimeError):
        call(q.clone().requires_grad_(), k, v, offsets)
    with torch.no_grad():
        assert not call(q.clone().requires_grad_(), k, v, offsets).requires_grad
    assert call(q[:0], k[:0], v[:0], offsets_of([])).shape == (0, 4, 64)


def test_few_workgroups_share_their_keys_between_groups(built_library):
    """Long sequences and few heads: the other launch shape, with every width, empty and one-token sequences beside them."""
    for d, dtype, causal in ((32, torch.float16, True), (64, torch.bfloat16, False), (128, torch.float16, False), (64, torch.float16, True)):
        for lengths in ([2049, 1600], [1, 3333, 0], [1664]):
            q, k, v = _projection(sum(lengths), 3, 1, d, dtype, seed=d)
            print(d, dtype, causal, lengths, flush=True)
            got = sspmm_amd.prompt_attention(q, k, v, offsets_of(lengths), causal=causal)
            check_prompt(got, q, k, v, lengths, causal, d ** -0.5)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_masked_places_where_groups_share_the_keys(built_library, bad):
    n = 1500
    q, k, v = (t.clone() for t in _projection(n, 2, 1, 128, torch.bfloat16, seed=31))
    at = 1210
    v[at, 0, 5] = bad
    got = sspmm_amd.prompt_attention(q, k, v, offsets_of([n]))
    check_prompt(got, q, k, v, [n], True, 128 ** -0.5)
    assert torch.isfinite(got[:at]).all() and not torch.isfinite(got[at:, :, 5]).any()


def test_prompts_of_many_thousand_tokens(built_library):
    """More than 6000 tokens with 128 features take a launch of their own."""
    lengths = [8003, 6500]
    q, k, v = _projection(sum(lengths), 8, 2, 128, torch.bfloat16, seed=32)
    for causal in (True, False):
        got = sspmm_amd.prompt_attention(q, k, v, offsets_of(lengths), causal=causal)
        check_prompt(got, q, k, v, lengths, causal, 128 ** -0.5)


def test_more_sequences_than_a_wave_has_lanes(built_library):
    """The longest tiles of 64 sequences go first, then the next 64's: every tile of every sequence is found, whatever their order."""
    for lengths in ([300] + [0] * 130 + [5, 257], list(range(0, 400, 3)), [128] * 65, [1] * 129 + [700]):
        for causal in (True, False):
            q, k, v = _projection(sum(lengths), 2, 2, 32, torch.float16, seed=len(lengths))
            got = sspmm_amd.prompt_attention(q, k, v, offsets_of(lengths), causal=causal)
            check_prompt(got, q, k, v, lengths, causal, 32 ** -0.5)


def test_twice_the_same_bits(built_library):
    q, k, v = _projection(3000, 8, 8, 64, torch.bfloat16, seed=33)
    first = sspmm_amd.prompt_attention(q, k, v, offsets_of([1200, 1800]))
    for _ in range(3):
        assert torch.equal(sspmm_amd.prompt_attention(q, k, v, offsets_of([1200, 1800])), first)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,heads", [([200, 90], 2), ([1700], 1)])
def test_infinities_beside_probabilities_that_underflow(built_library, causal, lengths, heads):
    """A key whose probability is far below what 16 bits hold is seen all the same: what is infinite in its v is infinite in the result."""
    n = sum(lengths)
    q, k, v = (t.clone() for t in _projection(n, heads, heads, 64, torch.float16, seed=34))
    q[:, :, 0], k[:, :, 0] = 8.0, 0.0
    for at, what in ((3, float("inf")), (70, float("-inf")), (n - 2, float("nan"))):
        k[at, :, 0] = -40.0  # 2^-58 beside the others
        v[at, 0, 7 + at % 5] = what
    got = sspmm_amd.prompt_attention(q, k, v, offsets_of(lengths), causal=causal)
    check_prompt(got, q, k, v, lengths, causal, 0.125)


def _randn(shape, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda")


@pytest.mark.parametrize("causal", [True, False])
def test_thousands_of_sequences(built_library, causal):
    """Sequences that are found by way of more than 64 groups of 64, empty ones and tokens in front of the first among them: the bits of a few at a time."""
    g = torch.Generator()
    g.manual_seed(5)
    counts = torch.randint(0, 4, (4500,), generator=g)
    counts[1000:1200] = 0
    counts[[64, 3000, 4499]] = 300
    offsets = (torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)]) + 200).int().cuda()
    tokens = int(offsets[-1]) + 70
    q, k, v = (_randn((tokens, h, 32), i).half() for i, h in ((1, 4), (2, 2), (3, 2)))
    out = torch.full_like(q, 7.0)
    sspmm_amd.prompt_attention(q, k, v, offsets, causal=causal, out=out)
    want = torch.full_like(q, 7.0)
    for b in range(0, 4500, 60):
        sspmm_amd.prompt_attention(q, k, v, offsets[b:b + 61].clone(), causal=causal, out=want)
    assert torch.equal(out, want)


def test_thousands_of_small_probabilities_in_fp16(built_library):
    """Probabilities below half of fp16's smallest number beside one of 1, together as large as what the result's type resolves: v is 1 there.  They are
    rounded as multiples of 2^-24 / 2^7: off by 2^-32 each at most, and the sum and the result by 2^-11 of it."""
    n = 16384
    q = torch.zeros(n, 1, 64, device="cuda", dtype=torch.float16)
    k, v = torch.zeros_like(q), torch.ones_like(q)
    q[..., 0] = 1.0
    k[1:, :, 0] = -25.5 * math.log(2.0)
    v[0] = 0.0
    out = sspmm_amd.prompt_attention(q, k, v, offsets_of([n]), scaling=1.0, causal=False)
    p = math.exp(k[1, 0, 0].item())
    want = (n - 1) * p / (1 + (n - 1) * p)
    assert (out.double() - want).abs().max().item() <= (n - 1) * 2.0 ** -32 + want * 2.0 ** -10


def test_in_place(built_library):
    lengths, heads, kv, d = [700, 1, 130, 2000], 8, 2, 128
    x = _randn((sum(lengths), (heads + 2 * kv) * d), 3).to(torch.bfloat16)
    q, k, v = x[:, :heads * d].view(-1, heads, d), x[:, heads * d:(heads + kv) * d].view(-1, kv, d), x[:, (heads + kv) * d:].view(-1, kv, d)
    for parts in (lengths, [2831]):  # (one sequence: two groups share the keys)
        kept = x.clone()
        want = sspmm_amd.prompt_attention(q, k, v, offsets_of(parts))
        assert sspmm_amd.prompt_attention(q, k, v, offsets_of(parts), out=q) is q
        assert torch.equal(q, want) and torch.equal(x[:, heads * d:], kept[:, heads * d:])
        x.copy_(kept)


def test_out_that_overlaps_itself_is_refused(built_library):
    q, k, v = (_randn((16, 4, 64), i).half() for i in range(3))
    narrow = torch.zeros(16, 1, 64, device="cuda", dtype=torch.float16)
    close = torch.zeros(16 * 128 + 256, device="cuda", dtype=torch.float16).as_strided((16, 4, 64), (128, 64, 1))
    for out in (narrow.expand(16, 4, 64), close):
        with pytest.raises(ValueError):
            sspmm_amd.prompt_attention(q, k, v, offsets_of([16]), out=out)


def test_more_sequences_than_a_launch_holds_are_refused(built_library):
    q, k, v = (torch.zeros(1, h, 32, device="cuda", dtype=torch.float16) for h in (32, 8, 8))
    with pytest.raises(RuntimeError):
        sspmm_amd.prompt_attention(q, k, v, torch.zeros(2 ** 18 + 1, dtype=torch.int32, device="cuda"))
    offsets = torch.ones(2 ** 18 - 1, dtype=torch.int32, device="cuda")
    offsets[0] = 0
    assert not sspmm_amd.prompt_attention(q, k, v, offsets).any()


@pytest.mark.parametrize("tokens,heads,kv", [(6100, 4, 1), (6100, 12, 4), (6100, 20, 4)])
def test_long_prompts_in_one_round_of_workgroups_and_more(built_library, tokens, heads, kv):
    q, k, v = _projection(tokens, heads, kv, 128, torch.bfloat16, seed=heads)
    for causal in (True, False):
        got = sspmm_amd.prompt_attention(q, k, v, offsets_of([tokens]), causal=causal)
        for h in (0, heads - 1):  # (each pair of a head of q and of k and v is a prompt of its own)
            pair = slice(h, h + 1), slice(h * kv // heads, h * kv // heads + 1)
            check_prompt(got[:, pair[0]], q[:, pair[0]], k[:, pair[1]], v[:, pair[1]], [tokens], causal, 1 / math.sqrt(128))



@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,heads,kv,d,causal", [([70, 1, 200], 2, 1, 64, True), ([131], 3, 3, 32, False), ([900, 5], 1, 1, 128, True), ([6100], 6, 6, 128, False)])
@pytest.mark.parametrize("scaling", [0.125, 1.0, 2.0 ** 40, 2.0e38])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scores_far_beyond_what_32_bits_resolve(built_library, dtype, lengths, heads, kv, d, causal, scaling, sign):
    """Scores of sign * 2^30 + 128 t, each exact in 32 bits, t a small whole number: softmax does not know of the 2^30.  Each probability is rounded to 16 bits (in
    fp16 below the normal numbers: half of 2^-24 where the largest is 2^7), its exponent, 48 scaling log2(e) or next to nothing, to a few times 2^-24; the result
    is rounded once."""
    n = sum(lengths)
    q, k = torch.zeros(n, heads, d, device="cuda", dtype=dtype), torch.zeros(n, kv, d, device="cuda", dtype=dtype)
    q[..., 0], k[..., 0] = 2.0 ** 15, sign * 2.0 ** 15
    t = torch.randint(0, 4, (n, kv), generator=torch.Generator().manual_seed(n)).cuda()
    q[..., 1], k[..., 1] = 128.0, t.to(dtype)
    q[::5] = 1.0  # queries of ordinary scores beside them: 0 .. 2^15 + 3
    v = _randn((n, kv, d), 3).to(dtype)
    got = sspmm_amd.prompt_attention(q, k, v, offsets_of(lengths), scaling=scaling, causal=causal)
    half = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    at = 0
    for count in lengths:
        part = slice(at, at + count)
        visible = torch.ones(count, count, device="cuda", dtype=torch.bool)
        visible = visible.tril() if causal else visible
        far = torch.arange(at, at + count, device="cuda") % 5 != 0
        for h in range(heads):
            key = t[part, h * kv // heads]
            most = torch.where(visible, key, -1).amax(1, keepdim=True)
            p = torch.exp(128 * scaling * (key - most).double()).masked_fill(~visible, 0.0)
            p /= p.sum(1, keepdim=True)
            x = v[part, h * kv // heads].double()
            off = (p @ x.abs()) * (half + 2.0 ** -16) + (p @ x).abs() * half + count * 2.0 ** -32 * x.abs().max() + 2.0 ** -25
            check(got[part, h][far], (p @ x)[far], off[far] * 1.01, "sequence at %d, head %d" % (at, h))
        at += count
    assert torch.isfinite(got).all()



@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_large_queries_and_keys(built_library, dtype, causal):
    """Normal values of size 12000: a query whose largest score is ahead of all others by more than both may be off, and 40, takes that key's v."""
    n, d = 300, 64
    q, k, v = (_randn((n, 2, d), i) for i in range(3))
    q, k, v = (q * 12000).to(dtype), (k * 12000).to(dtype), v.to(dtype)
    got = sspmm_amd.prompt_attention(q, k, v, offsets_of([n]), causal=causal)
    assert torch.isfinite(got).all()
    decided = 0
    for h in range(2):
        s = (q[:, h].double() @ k[:, h].double().t().contiguous()) / 8
        size = (q[:, h].double().abs() @ k[:, h].double().abs().t().contiguous()).amax(1) / 8
        if causal:
            s = s.masked_fill(torch.ones(n, n, device="cuda", dtype=torch.bool).triu(1), float("-inf"))
        two = s.topk(2, 1)
        sure = two.values[:, 0] - two.values[:, 1] > 40 + 2 * size * (d + 8) * 2.0 ** -24
        want = v[two.indices[:, 0], h].double()
        half = 2.0 ** -11 if dtype is torch.float16 else 2.0 ** -8
        off = want.abs() * (2 * half + 2.0 ** -17) + 1e-15
        check(got[:, h][sure], want[sure], off[sure])
        decided += int(sure.sum())
    assert decided > n  # (of 2 n)



def test_values_at_the_end_of_the_range(built_library):
    """Means of values whose sum is still a number of 32 bits, where later tiles' scores are some powers of two larger than the first one's."""
    n, d = 192, 64
    q = torch.ones(n, 1, d, device="cuda", dtype=torch.bfloat16)
    k = torch.zeros_like(q)
    k[64:, :, 0] = 7.5
    v = (1e36 * (1 + 0.5 * torch.rand(n, 1, d, generator=torch.Generator().manual_seed(4)))).cuda().bfloat16()
    for causal in (True, False):
        got = sspmm_amd.prompt_attention(q, k, v, offsets_of([n]), scaling=math.log(2.0), causal=causal)
        check_prompt(got, q, k, v, [n], causal, math.log(2.0))



@pytest.mark.parametrize("n,causal", [(200, True), (200, False), (1700, True), (1700, False)])
@pytest.mark.parametrize("below", [100.0, 140.0, 200.0, 500.0])
@pytest.mark.parametrize("first", [0, 64, 128])
def test_large_values_of_small_probability(built_library, n, causal, below, first):
    """v of 1e38 at 64 keys whose scores lie `below` powers of two under the others': their share is there as long as it is a number, and nothing else of them."""
    d, large = 64, slice(first, first + 64)
    q = torch.zeros(n, 1, d, device="cuda", dtype=torch.bfloat16)
    k, v = torch.zeros_like(q), torch.ones_like(q)
    q[..., 0], k[..., 0] = 1.0, below
    k[large], v[large] = 0.0, 1e38
    got = sspmm_amd.prompt_attention(q, k, v, offsets_of([n]), scaling=math.log(2.0), causal=causal)[:, 0]
    big, p = v[first, 0, 0].double(), 2.0 ** -below
    seen = torch.arange(1, n + 1, device="cuda")[:, None].double() if causal else torch.full((n, 1), n, device="cuda").double()
    low = (seen - first).clamp(0, 64)
    high = seen - low
    want = (high + low * p * big) / (high + low * p)
    # half a step of each probability (bf16), what scaling and its product with log2(e) are off by, the result's half step; a probability below 2^-126 may be nothing
    off = want * (2.0 ** -8 + 2.0 ** -18 + below * 2.0 ** -22) + want * 2.0 ** -8 + torch.where(high > 0, low * p * big if below > 110 else 0.0, 0.0)
    check(got, want.expand(-1, d), (off * 1.01).expand(-1, d))
