"""The paged cache in 8 bits: writing it, bit for bit, and attention over it against the formula in 64 bits."""
import math

import pytest
import torch

import sspmm_amd
from serving_util import attention, check, check_step, codes_for, offsets_of, row_of_cache, scale_for, write

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16]
FORMATS = [torch.int8, torch.float8_e4m3fn]


def _randn(shape, seed, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda") * scale


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _filled(pages, kv, page, d, dtype, seed):
    """A pool of quantised normal values, blocks of different size."""
    keys, values, scales = sspmm_amd.new_cache(pages, kv, page, d, dtype)
    for i, pool in enumerate((keys, values)):
        x = _randn(pool.shape, seed + i) * torch.exp(_randn((pages, kv, 1, 1), seed + 10 + i))
        s = scale_for(x.abs().amax((2, 3)), dtype)
        pool.view(torch.int8).copy_(codes_for(x, s[:, :, None, None], dtype))
        scales[:, i] = s
    return keys, values, scales


def _table(lengths, page, seed, spare=3):
    g = torch.Generator()
    g.manual_seed(seed)
    held = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(held) + spare, generator=g)
    table = torch.full((len(lengths), max(held + [1]) + 1), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(held):
        table[i, :n] = order[at:at + n]
        at += n
    return table.cuda(), sum(held) + spare


# ---- writing

@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page,d,kv", [(32, 64, 3), (64, 128, 2), (128, 32, 1), (128, 128, 2), (64, 32, 5)])
def test_writes_bit_for_bit(built_library, page, d, kv, dtype, form):
    starts = [0, 5, page - 1, page, 3 * page + 7, 0, 11, 2 * page - 3]
    counts = [1, 1, 2, page, 2 * page + 9, 3 * page, 0, 3]
    table, pages = _table([s + n for s, n in zip(starts, counts)], page, seed=page)
    keys, values, scales = _filled(pages, kv, page, d, form, seed=d)
    tokens = sum(counts)
    x = (_randn((tokens, 2, kv, d), 5) * torch.exp(_randn((tokens, 1, kv, 1), 6))).to(dtype)
    k, v = x.unbind(1)
    host = [t.cpu().clone() for t in (keys, values, scales)]
    write(k.cpu(), v.cpu(), offsets_of(counts).cpu(), starts, table.cpu(), *host)
    print(page, d, kv, dtype, form, flush=True)
    sspmm_amd.cache_write(k, v, offsets_of(counts), _ints(starts), table, keys, values, scales)
    for name, got, want in zip(("keys", "values", "scales"), (keys, values, scales), host):
        same = got.cpu().view(torch.int8 if got.dtype in FORMATS else torch.int32) == want.view(torch.int8 if want.dtype in FORMATS else torch.int32)
        assert same.all(), "%s: %d of %d differ" % (name, (~same).sum(), same.numel())


@pytest.mark.parametrize("form", FORMATS)
def test_token_by_token_is_as_the_rule_says(built_library, form):
    """A page filled one token at a time, sizes rising and falling: each growth of the scale brings the codes to it once more."""
    page, kv, d = 32, 2, 64
    keys, values, scales = _filled(4, kv, page, d, form, seed=1)
    host = [t.cpu().clone() for t in (keys, values, scales)]
    table = _ints([[2, 0]])
    for i in range(40):
        x = (_randn((1, 2, kv, d), 100 + i) * 2.0 ** ((7 * i) % 11 - 5)).half()
        k, v = x.unbind(1)
        write(k.cpu(), v.cpu(), [0, 1], [i], table.cpu(), *host)
        sspmm_amd.cache_write(k, v, offsets_of([1]), _ints([i]), table, keys, values, scales)
    for got, want in zip((keys, values, scales), host):
        assert torch.equal(got.cpu().view(torch.int8), want.view(torch.int8))
    # what was written is there: within half a step of the block's scale for each time it was brought to a larger one, and its own rounding
    k, v = row_of_cache(table[0], keys, values, scales, 40)
    x = torch.stack([(_randn((1, 2, kv, d), 100 + i) * 2.0 ** ((7 * i) % 11 - 5)).half() for i in range(40)]).double()[:, 0]
    step = 0.5 if form is torch.int8 else 0.0
    for i, got in enumerate((k, v)):
        s = scales[table[0].long(), i].double().repeat_interleave(page, 0)[:40, :, None]  # [40, kv, 1]
        # e4m3: 2^-4 of the value, or half of the smallest step, which is 2^-9 of the scale.  Scales grow by powers of two, so codes that stay
        # normal numbers move without a rounding, and those that do not are off by half a smallest step of each scale they had in turn,
        # the last one's and at most half of it, a quarter, ...: 2^-9 of the scale in all.
        near = 12 * s * step if step else x[:, i].abs() * 2.0 ** -4 + s * 2.0 ** -9
        assert ((got - x[:, i]).abs() <= near).all()


def test_every_e4m3_code_and_every_tie(built_library):
    """All halves below 448 against torch's conversion (the block's largest is 448, so its scale is one)."""
    bits = torch.arange(0, 0x6000, dtype=torch.int32, device="cuda").to(torch.int16)
    x = bits.view(torch.float16)
    x = x[x <= 448]
    x = torch.cat([x, -x])
    d, page = 128, 128
    n = -(-x.numel() // (d - 1))
    x = torch.nn.functional.pad(x, (0, n * (d - 1) - x.numel())).view(n, 1, d - 1)
    x = torch.cat([torch.full((n, 1, 1), 448.0, device="cuda", dtype=torch.float16), x], 2)
    pages = -(-n // page)
    keys, values, scales = sspmm_amd.new_cache(pages, 1, page, d, torch.float8_e4m3fn)
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    sspmm_amd.cache_write(x, x, offsets_of([n]), _ints([0]), table, keys, values, scales)
    assert (scales == 1).all()
    want = x[:, 0].to(torch.float8_e4m3fn).view(torch.int8)
    assert torch.equal(keys.view(torch.int8).view(-1, d)[:n], want)
    assert torch.equal(values.view(torch.int8).transpose(2, 3).reshape(-1, d)[:n], want)


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("most", [2.0 ** -126, 3e-39, 1e-45, 0.0, 3.0e38, 1.75 * 2.0 ** 20, 1.7578125 * 2.0 ** 20])
def test_sizes_at_the_ends_of_the_range(built_library, form, most):
    keys, values, scales = _filled(1, 1, 32, 32, form, seed=2)
    x = torch.zeros(3, 1, 32, device="cuda", dtype=torch.bfloat16)
    x[1, 0, 5], x[2, 0, 7] = most, -most / 2
    host = [t.cpu().clone() for t in (keys, values, scales)]
    write(x.cpu(), x.cpu(), [0, 3], [0], torch.zeros(1, 1, dtype=torch.int32), *host)
    sspmm_amd.cache_write(x, x, offsets_of([3]), _ints([0]), _ints([[0]]), keys, values, scales)
    for got, want in zip((keys, values, scales), host):
        assert torch.equal(got.cpu().view(torch.int8), want.view(torch.int8))


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_what_is_not_finite_marks_its_block(built_library, form, bad):
    page, kv, d = 32, 2, 32
    keys, values, scales = _filled(3, kv, page, d, form, seed=3)
    before = scales.clone()
    k, v = _randn((4, kv, d), 1).half(), _randn((4, kv, d), 2).half()
    k[1, 0, 3] = bad
    table = _ints([[1, 2]])
    sspmm_amd.cache_write(k, v, offsets_of([4]), _ints([10]), table, keys, values, scales)
    assert torch.isnan(scales[1, 0, 0]) and torch.isfinite(scales[1, 0, 1]) and torch.isfinite(scales[1, 1]).all()
    assert torch.equal(scales[[0, 2]], before[[0, 2]])
    out = sspmm_amd.cache_attention(_randn((1, 1, 4, d), 3).half(), table, _ints([14]), keys, values, scales)
    assert torch.isnan(out[0, 0, :2]).all() and torch.isfinite(out[0, 0, 2:]).all()
    # it stays so until the page begins anew
    ok = _randn((1, kv, d), 4).half()
    sspmm_amd.cache_write(ok, ok, offsets_of([1]), _ints([14]), table, keys, values, scales)
    assert torch.isnan(scales[1, 0, 0])
    sspmm_amd.cache_write(ok, ok, offsets_of([1]), _ints([0]), table, keys, values, scales)
    assert torch.isfinite(scales).all()


def test_tokens_without_a_page_are_dropped(built_library):
    page, kv, d = 32, 2, 32
    keys, values, scales = _filled(4, kv, page, d, torch.int8, seed=4)
    host = [t.cpu().clone() for t in (keys, values, scales)]
    table = _ints([[-1, 1], [4, 2], [0, 2 ** 31 - 1], [3, -7]])
    counts, starts = [40, 50, 5, 90], [0, 0, -3, 20]  # (a start below zero: nothing; the last row runs out of its slots)
    k, v = _randn((sum(counts), kv, d), 5).half(), _randn((sum(counts), kv, d), 6).half()
    write(k.cpu(), v.cpu(), offsets_of(counts).cpu(), starts, table.cpu(), *host)
    sspmm_amd.cache_write(k, v, offsets_of(counts), _ints(starts), table, keys, values, scales)
    for got, want in zip((keys, values, scales), host):
        assert torch.equal(got.cpu().view(torch.int8), want.view(torch.int8))


@pytest.mark.parametrize("order", ["heads first", "features first", "odd start"])
def test_write_from_other_orders_in_memory(built_library, order):
    k, v = _randn((70, 2, 64), 7).half(), _randn((70, 2, 64), 8).half()
    table = _ints([[3, 0, 1]])
    want = _filled(4, 2, 32, 64, torch.int8, seed=9)
    sspmm_amd.cache_write(k, v, offsets_of([70]), _ints([9]), table, *want)
    if order == "heads first":
        k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (k, v))
    elif order == "features first":
        k, v = (t.permute(1, 2, 0).contiguous().permute(2, 0, 1) for t in (k, v))
    else:
        k, v = (torch.nn.functional.pad(t.reshape(-1), (5, 0))[5:].view(t.shape) for t in (k, v))
    got = _filled(4, 2, 32, 64, torch.int8, seed=9)
    sspmm_amd.cache_write(k, v, offsets_of([70]), _ints([9]), table, *got)
    assert all(torch.equal(a.view(torch.int8), b.view(torch.int8)) for a, b in zip(got, want))


# ---- attention

@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page,d", [(32, 128), (64, 128), (128, 128), (32, 64), (64, 64), (128, 32), (32, 32), (64, 32)])
@pytest.mark.parametrize("n,heads,kv", [(1, 4, 1), (1, 3, 3), (5, 8, 4), (3, 16, 2), (11, 6, 2)])
def test_attention_against_the_formula(built_library, n, heads, kv, page, d, dtype, form):
    lengths = [1, 0, 2, page - 1, page, page + 1, 5 * page + 17, 333]
    table, pages = _table(lengths, page, seed=n)
    pool = _filled(pages, kv, page, d, form, seed=d + n)
    q = _randn((len(lengths), n, heads, d), 11, 1.5).to(dtype)
    print(n, heads, kv, page, d, dtype, form, flush=True)
    got = sspmm_amd.cache_attention(q, table, _ints(lengths), *pool)
    check_step(got, q, table, lengths, *pool, 1 / math.sqrt(d))


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("lengths,n,heads,kv,page,d", [([9001], 1, 8, 2, 64, 128), ([20000, 17], 2, 4, 4, 128, 64), ([4096, 5000, 1], 9, 4, 1, 32, 128),
                                                       ([7777], 1, 64, 1, 64, 64)])
def test_long_rows_are_split_and_joined(built_library, lengths, n, heads, kv, page, d, form):
    table, pages = _table(lengths, page, seed=1)
    pool = _filled(pages, kv, page, d, form, seed=2)
    q = _randn((len(lengths), n, heads, d), 12, 1.5).bfloat16()
    got = sspmm_amd.cache_attention(q, table, _ints(lengths), *pool)
    check_step(got, q, table, lengths, *pool, 1 / math.sqrt(d))


@pytest.mark.parametrize("size", [1e-30, 1e-4, 1.0, 3e4, 1e30])
def test_queries_of_any_size(built_library, size):
    lengths, d = [200, 65], 64
    table, pages = _table(lengths, 64, seed=3)
    pool = _filled(pages, 2, 64, d, torch.int8, seed=4)
    q = _randn((2, 1, 4, d), 13, size).bfloat16()
    scaling = 1 / (8 * size)
    got = sspmm_amd.cache_attention(q, table, _ints(lengths), *pool, scaling=scaling)
    check_step(got, q, table, lengths, *pool, scaling)


def test_blocks_of_very_different_scales(built_library):
    """One block of large values that the queries ignore beside small ones that they do not: nothing of the small ones is lost."""
    page, d = 32, 64
    keys, values, scales = _filled(4, 1, page, d, torch.int8, seed=5)
    keys.zero_()
    keys[0, 0, :, 0] = -127
    scales[0], scales[1:] = 1.0, 1.0
    scales[0, 1], scales[1:, 1] = 1e6, 1e-3
    table, lengths = _ints([[0, 1, 2, 3]]), [4 * page]
    q = torch.zeros(1, 1, 1, d, device="cuda", dtype=torch.float16)
    q[..., 0] = 1.0
    got = sspmm_amd.cache_attention(q, table, _ints(lengths), keys, values, scales, scaling=1.0)
    k, v = row_of_cache(table[0], keys, values, scales, 128)
    want, off = attention(q[0, 0], k[:, 0], v[:, 0], torch.tensor([128], device="cuda"), 1.0, torch.float16, torch.float16)
    # (the first block's probabilities are 2^-183: neither they nor their rounding reach the result)
    _, off = attention(q[0, 0], k[page:, 0], v[page:, 0], torch.tensor([96], device="cuda"), 1.0, torch.float16, torch.float16)
    check(got[0, 0], want, off)


@pytest.mark.parametrize("form", FORMATS)
def test_nothing_comes_from_behind_the_row(built_library, form):
    """Codes of NaN and scales of NaN in the rest of the last page, in pages behind it, and where a draft's earlier queries do not see."""
    page, d, lengths = 32, 64, [40, 1, 33, 64]
    table, pages = _table(lengths, page, seed=6)
    pool = _filled(pages, 2, page, d, form, seed=7)
    q = _randn((4, 3, 4, d), 14).half()
    want = sspmm_amd.cache_attention(q, table, _ints(lengths), *pool)
    nan = 0x7f if form is torch.float8_e4m3fn else -128
    keys, values, scales = (t.clone() for t in pool)
    kb, vb = keys.view(torch.int8), values.view(torch.int8)
    for b, n in enumerate(lengths):
        if n % page:
            p = int(table[b, n // page])
            kb[p, :, n % page:] = nan
            vb[p, :, :, n % page:] = nan
    free = [p for p in range(pages) if not (table == p).any()]
    kb[free], vb[free], scales[free] = nan, nan, float("nan")
    table2 = table.clone()
    for b, n in enumerate(lengths):  # pages behind the row's end
        table2[b, -(-n // page):] = free[0]
    got = sspmm_amd.cache_attention(q, table2, _ints(lengths), keys, values, scales)
    assert torch.equal(got, want)
    # queries 0 of the row of 33 (sees 31) and 1 (sees 32): its second page is not theirs
    p = int(table[2, 1])
    scales[p] = float("nan")
    got = sspmm_amd.cache_attention(q, table2, _ints(lengths), keys, values, scales)
    assert torch.equal(got[2, :2], want[2, :2]) and torch.isnan(got[2, 2]).all() and torch.equal(got[[0, 1, 3]], want[[0, 1, 3]])


def test_positions_without_a_page_are_masked(built_library):
    page, d = 32, 64
    pool = _filled(6, 1, page, d, torch.int8, seed=8)
    table = _ints([[4, -1, 2], [6, 1, 2 ** 31 - 1], [-1, -1, -1]])
    q = _randn((3, 1, 2, d), 15).half()
    got = sspmm_amd.cache_attention(q, table, _ints([96, 96, 50]), *pool)
    want = sspmm_amd.cache_attention(q, _ints([[4, 2], [1, 0], [0, 0]]), _ints([64, 32, 0]), *pool)
    assert not got[2].any()
    for b, part in ((0, [4, 2]), (1, [1])):
        k, v = row_of_cache(_ints(part), *pool, 32 * len(part))
        for h in range(2):
            ref, off = attention(q[b, :, h], k[:, 0], v[:, 0], torch.tensor([32 * len(part)], device="cuda"), 0.125, torch.float16, torch.float16)
            check(got[b, :, h], ref, off)
            check(want[b, :, h], ref, off)
    # lengths beyond the table end with it, lengths below zero are empty
    got = sspmm_amd.cache_attention(q, table, _ints([2 ** 31 - 1, -5, 0]), *pool)
    assert not got[1:].any()
    check(got[0, :, 0], *attention(q[0, :, 0], *(t[:, 0] for t in row_of_cache(_ints([4, 2]), *pool, 64)), torch.tensor([64], device="cuda"), 0.125,
                                   torch.float16, torch.float16))


@pytest.mark.parametrize("order", ["heads first", "features first", "odd start", "out"])
def test_attention_of_other_orders_in_memory(built_library, order):
    lengths, d = [100, 31], 64
    table, pages = _table(lengths, 32, seed=9)
    pool = _filled(pages, 2, 32, d, torch.int8, seed=10)
    q = _randn((2, 3, 4, d), 16).bfloat16()
    want = sspmm_amd.cache_attention(q, table, _ints(lengths), *pool)
    out = None
    if order == "heads first":
        q = q.transpose(1, 2).contiguous().transpose(1, 2)
    elif order == "features first":
        q = q.permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)
    elif order == "odd start":
        q = torch.nn.functional.pad(q.reshape(-1), (1, 0))[1:].view(q.shape)
    else:
        out = torch.full((2, 5, 4, d + 8), 7.0, device="cuda", dtype=torch.bfloat16)[:, 1:4, :, :d]
    got = sspmm_amd.cache_attention(q, table, _ints(lengths), *pool, out=out)
    assert torch.equal(got, want)
    if out is not None:
        assert (out._base[:, 0] == 7).all() and (out._base[:, 4] == 7).all() and (out._base[..., d:] == 7).all()


def test_a_pool_beyond_32_bits(built_library):
    """Pages whose bytes lie past 2^32."""
    page, kv, d = 128, 8, 128
    pages = (1 << 32) // (kv * page * d) + 40
    keys = torch.empty(pages, kv, page, d, dtype=torch.int8, device="cuda")
    values = torch.empty(pages, kv, d, page, dtype=torch.int8, device="cuda")
    scales = torch.zeros(pages, 2, kv, device="cuda")
    table = torch.arange(pages - 3, pages, dtype=torch.int32, device="cuda")[None].contiguous()
    k, v = _randn((300, kv, d), 17).half(), _randn((300, kv, d), 18).half()
    sspmm_amd.cache_write(k, v, offsets_of([300]), _ints([0]), table, keys, values, scales)
    q = _randn((1, 1, kv, d), 19).half()
    got = sspmm_amd.cache_attention(q, table, _ints([300]), keys, values, scales)
    last = table[0].long()
    small = keys[last].contiguous(), values[last].contiguous(), scales[last].contiguous()
    want = sspmm_amd.cache_attention(q, _ints([[0, 1, 2]]), _ints([300]), *small)
    assert torch.equal(got, want)
    check_step(got, q, _ints([[0, 1, 2]]), [300], *small, 128 ** -0.5)


def test_two_graphs_and_two_streams(built_library):
    """Each call has a workspace of its own: two captured steps replayed one after the other, calls on two streams at once."""
    lengths, d = [3000, 1700], 128
    table, pages = _table(lengths, 64, seed=11)
    pool = _filled(pages, 2, 64, d, torch.int8, seed=12)
    n = _ints(lengths)
    qs = [_randn((2, 1, 8, d), 30 + i).bfloat16() for i in range(2)]
    outs, graphs = [torch.zeros_like(q) for q in qs], [torch.cuda.CUDAGraph() for _ in qs]
    sspmm_amd.cache_attention(qs[0], table, n, *pool)
    torch.cuda.synchronize()
    for q, out, g in zip(qs, outs, graphs):
        with torch.cuda.graph(g):
            sspmm_amd.cache_attention(q, table, n, *pool, out=out)
    for turn in range(4):
        n.copy_(_ints([3000 - 500 * turn, 100 + turn]))
        for i, q in enumerate(qs):
            q.copy_(_randn((2, 1, 8, d), 40 + 2 * turn + i))
        want = [sspmm_amd.cache_attention(q, table, n, *pool) for q in qs]
        for g in graphs if turn % 2 else graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    torch.cuda.synchronize()
    for turn in range(6):
        for s, q in zip(streams, qs):
            with torch.cuda.stream(s):
                got.append(sspmm_amd.cache_attention(q, table, n, *pool))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i % 2]) for i, x in enumerate(got))


def test_refusals(built_library):
    keys, values, scales = sspmm_amd.new_cache(4, 2, 32, 64)
    table, n, q = _ints([[0, 1]]), _ints([40]), _randn((1, 1, 4, 64), 1).half()
    k = _randn((3, 2, 64), 2).half()
    step, put = sspmm_amd.cache_attention, sspmm_amd.cache_write
    for bad, kind in (((q.float(), table, n, keys, values, scales), TypeError), ((q, table.long(), n, keys, values, scales), TypeError),
                      ((q, table, n.cpu(), keys, values, scales), TypeError), ((q, table, n, keys.float(), values, scales), TypeError),
                      ((q, table, n, keys, values.view(torch.float8_e4m3fn), scales), TypeError), ((q, table, n, keys, values, scales.half()), TypeError),
                      ((q[0], table, n, keys, values, scales), ValueError), ((q[..., :32], table, n, keys, values, scales), ValueError),
                      ((q[:, :, :3], table, n, keys, values, scales), ValueError), ((q, table[0], n, keys, values, scales), ValueError),
                      ((q, _ints([[0], [1]]), n, keys, values, scales), ValueError), ((q, table, _ints([1, 2]), keys, values, scales), ValueError),
                      ((q, table, n, keys, values.transpose(2, 3).contiguous(), scales), ValueError), ((q, table, n, keys, values, scales[:, :, :1].contiguous()), ValueError),
                      ((q, table, n, keys[1:3, :, ::2].contiguous(), values[1:3, :, :, ::2].contiguous(), scales[1:3]), ValueError),
                      ((q, table, n, keys.transpose(0, 1), values, scales), ValueError), ((q, table[:, :0], n, keys, values, scales), ValueError)):
        with pytest.raises(kind):
            step(*bad)
    with pytest.raises(ValueError):
        step(q, table, n, keys, values, scales, scaling=float("inf"))
    with pytest.raises(RuntimeError):
        step(q.clone().requires_grad_(), table, n, keys, values, scales)
    with pytest.raises(ValueError):
        step(q, table, n, keys, values, scales, out=q[:, :, :2])
    off, start = offsets_of([3]), _ints([0])
    for bad, kind in (((k.float(), k, off, start, table, keys, values, scales), TypeError), ((k, k.bfloat16(), off, start, table, keys, values, scales), TypeError),
                      ((k[:, :1], k[:, :1], off, start, table, keys, values, scales), ValueError), ((k, k[:2], off, start, table, keys, values, scales), ValueError),
                      ((k, k, off[:1], start, table, keys, values, scales), ValueError), ((k, k, off, start.long(), table, keys, values, scales), TypeError),
                      ((k, k, off, start, _ints([[0], [1]]), keys, values, scales), ValueError)):
        with pytest.raises(kind):
            put(*bad)
    with pytest.raises(TypeError):
        sspmm_amd.new_cache(4, 2, 32, 64, torch.float16)
    for page, d in ((16, 64), (48, 64), (32, 80)):
        with pytest.raises(ValueError):
            sspmm_amd.new_cache(4, 2, page, d)
    assert step(q[:0], table[:0], n[:0], keys, values, scales).shape == (0, 1, 4, 64)


def test_more_rows_than_a_wave_has_lanes(built_library):
    """Rows of all lengths, the longest of every 64 first; more queries than a tile of rows; writes of as many sequences."""
    lengths = [(97 * i * i + 13 * i) % 700 for i in range(150)]
    table, pages = _table(lengths, 64, seed=21)
    pool = _filled(pages, 3, 64, 64, torch.int8, seed=22)
    q = _randn((150, 1, 6, 64), 23).half()
    got = sspmm_amd.cache_attention(q, table, _ints(lengths), *pool)
    check_step(got, q, table, lengths, *pool, 0.125)
    counts = [(3 * i) % 7 for i in range(150)]
    starts = [max(0, n - c) for n, c in zip(lengths, counts)]
    x = _randn((sum(counts), 2, 3, 64), 24).half()
    k, v = x.unbind(1)
    host = [t.cpu().clone() for t in pool]
    write(k.cpu(), v.cpu(), offsets_of(counts).cpu(), starts, table.cpu(), *host)
    sspmm_amd.cache_write(k, v, offsets_of(counts), _ints(starts), table, *pool)
    for a, b in zip(pool, host):
        assert torch.equal(a.cpu().view(torch.int8), b.view(torch.int8))


@pytest.mark.parametrize("n,heads,kv", [(70, 4, 1), (129, 3, 3), (33, 16, 1)])
def test_a_piece_of_a_prompt_over_the_cache(built_library, n, heads, kv):
    """Many queries at once: a prompt's later part over what is in the cache, its own tokens among it."""
    lengths, page, d = [n, 3 * n + 5, n - 3, 700], 64, 64
    table, pages = _table(lengths, page, seed=25)
    pool = _filled(pages, kv, page, d, torch.float8_e4m3fn, seed=26)
    q = _randn((4, n, heads, d), 27).bfloat16()
    got = sspmm_amd.cache_attention(q, table, _ints(lengths), *pool)
    check_step(got, q, table, lengths, *pool, 0.125)


@pytest.mark.parametrize("form", FORMATS)
def test_a_captured_decoding_step(built_library, form):
    """Pages, writing and attention of the next token in one graph, replayed token after token with the program's own work in between; the cache and
    every result as in a program that calls them one by one."""
    rows, kv, heads, d, page, pages = 3, 2, 4, 64, 32, 24
    state = []
    for _ in range(2):
        keys, values, scales = sspmm_amd.new_cache(pages, kv, page, d, form)
        state.append(dict(cache=(keys, values, scales), refs=_ints([0] * pages), table=torch.full((rows, 6), -1, dtype=torch.int32, device="cuda"),
                          starts=_ints([0, 30, 63]), lengths=_ints([1, 31, 64]), out=torch.zeros(rows, 1, heads, d, device="cuda", dtype=torch.float16)))
    offsets = offsets_of([1] * rows)
    k, v, q = (torch.zeros(rows, n, d, device="cuda", dtype=torch.float16) for n in (kv, kv, heads))
    for s in state:  # what came before
        x = _randn((93, 2, kv, d), 50).half()
        first = _ints([0, 0, 30, 93])
        sspmm_amd.reserve_pages(s["refs"], s["table"], _ints([0, 0, 0]), first, page)
        sspmm_amd.cache_write(x[:, 0], x[:, 1], first, _ints([0, 0, 0]), s["table"], *s["cache"])

    def step(s):
        sspmm_amd.reserve_pages(s["refs"], s["table"], s["starts"], offsets, page)
        sspmm_amd.cache_write(k, v, offsets, s["starts"], s["table"], *s["cache"])
        sspmm_amd.cache_attention(q[:, None], s["table"], s["lengths"], *s["cache"], out=s["out"])

    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(state[0])
    for token in range(70):
        for i, t in enumerate((k, v, q)):
            t.copy_(_randn(t.shape, 100 + 3 * token + i) * 2.0 ** (token % 5))
        g.replay()
        step(state[1])
        torch.cuda.synchronize()
        assert torch.equal(state[0]["out"], state[1]["out"]), token
        for s in state:
            s["starts"] += 1
            s["lengths"] += 1
    for a, b in zip(state[0]["cache"] + (state[0]["table"], state[0]["refs"]), state[1]["cache"] + (state[1]["table"], state[1]["refs"])):
        assert torch.equal(a.view(torch.int8), b.view(torch.int8))
    check_step(state[0]["out"], q[:, None], state[0]["table"], [70, 100, 133], *state[0]["cache"], 0.125)


def test_thousands_of_rows_are_written(built_library):
    """Rows found by way of more than 64 groups of 64, by their tokens (most of one) and by their pages: the bytes of a few rows at a time."""
    g = torch.Generator()
    g.manual_seed(6)
    for most in (2, 90):
        counts = torch.randint(0, most, (4500,), generator=g)
        counts[700:900] = 0
        starts = torch.randint(0, 40, (4500,), generator=g)
        slots = -(-(most + 40) // 32)
        offsets = torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)]).int().cuda()
        starts = starts.int().cuda()
        table = torch.randperm(4500 * slots, generator=g).int().cuda().view(4500, slots)
        k, v = (_randn((int(offsets[-1]), 2, 32), i).half() for i in (1, 2))
        caches = [sspmm_amd.new_cache(4500 * slots, 2, 32, 32) for _ in range(2)]
        sspmm_amd.cache_write(k, v, offsets, starts, table, *caches[0])
        for b in range(0, 4500, 60):
            sspmm_amd.cache_write(k, v, offsets[b:b + 61].clone(), starts[b:b + 60].clone(), table[b:b + 60].clone(), *caches[1])
        for x, y in zip(*caches):
            assert torch.equal(x, y)


def test_thousands_of_small_probabilities(built_library):
    """As with prompts: off by 2^-32 a key at most, and 2^-11 of the sum and of the result."""
    n, page = 16384, 64
    keys, values, scales = sspmm_amd.new_cache(n // page, 1, page, 64)
    keys[..., 0] = -127
    keys[0, 0, 0, 0] = 0
    values.fill_(127)
    values[0, :, :, 0] = 0
    scales[:, 0], scales[:, 1] = 25.5 * math.log(2.0) / 127, 1.0 / 127
    q = torch.zeros(1, 1, 1, 64, device="cuda", dtype=torch.float16)
    q[..., 0] = 1.0
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").view(1, -1)
    out = sspmm_amd.cache_attention(q, table, _ints([n]), keys, values, scales, scaling=1.0)
    p = math.exp(-127 * scales[0, 0, 0].item())
    want = (n - 1) * p / (1 + (n - 1) * p)
    assert (out.double() - want).abs().max().item() <= (n - 1) * 2.0 ** -32 + want * 2.0 ** -10


@pytest.mark.parametrize("lengths,heads,kv", [([700, 33, 0, 200], 8, 2), ([9000], 40, 2)])
def test_attention_in_place(built_library, lengths, heads, kv):
    table, pages = _table(lengths, 64, seed=3)
    cache = _filled(pages, kv, 64, 64, torch.int8, seed=4)
    q = _randn((len(lengths), 2, heads, 64), 5).half()
    want = sspmm_amd.cache_attention(q, table, _ints(lengths), *cache)
    assert sspmm_amd.cache_attention(q, table, _ints(lengths), *cache, out=q) is q
    assert torch.equal(q, want)


def test_attention_into_rows_that_overlap_is_refused(built_library):
    table, pages = _table([40], 64, seed=3)
    cache = _filled(pages, 1, 64, 64, torch.int8, seed=4)
    q = _randn((1, 2, 4, 64), 5).half()
    for out in (q[:, :, :1].expand(1, 2, 4, 64), q.view(-1)[:320].as_strided((1, 2, 4, 64), (512, 64, 64, 1))):
        with pytest.raises(ValueError):
            sspmm_amd.cache_attention(q, table, _ints([40]), *cache, out=out)



@pytest.mark.parametrize("form", FORMATS)
def test_values_at_the_end_of_the_range(built_library, form):
    """Values of up to 6e36 and keys whose scores grow by some powers of two along the row: probabilities are large numbers before they are divided by their sum."""
    lengths, d, page = [700, 40, 5000], 64, 64
    table, pages = _table(lengths, page, seed=31)
    keys, values, scales = _filled(pages, 2, page, d, form, seed=32)
    scales[:, 1] *= 6e36 / (127 if form is torch.int8 else 448) / scales[:, 1].max()
    q = _randn((3, 2, 4, d), 33).bfloat16()
    for rows in (slice(0, 2), slice(0, 3)):
        got = sspmm_amd.cache_attention(q[rows], table[rows].contiguous(), _ints(lengths[rows]), keys, values, scales)
        check_step(got, q[rows], table[rows], lengths[rows], keys, values, scales, 0.125)


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("size", [1e-36, 1e-30, 1e-6])
def test_values_near_the_smallest(built_library, form, size):
    """Tiny values come back as far as 32 bits hold them: a scale in units of 2^16 is off by half of 2^-149, which is 2^-134 of the scale, and 2^-127 with the largest
    code; 2^-125 is allowed."""
    lengths, d, page = [300, 40], 64, 64
    table, pages = _table(lengths, page, seed=36)
    keys, values, scales = _filled(pages, 2, page, d, form, seed=37)
    scales[:, 1] *= size / scales[:, 1].max()
    if form is torch.float8_e4m3fn:
        scales[:, 1] = torch.ldexp(torch.ones(()), scales[:, 1].log2().round().cpu()).cuda()
    q = _randn((2, 1, 4, d), 38).bfloat16()
    got = sspmm_amd.cache_attention(q, table, _ints(lengths), keys, values, scales).double()
    for b, n in enumerate(lengths):
        k, v = row_of_cache(table[b], keys, values, scales, n)
        for h in range(4):
            want, off = attention(q[b, :, h], k[:, h // 2], v[:, h // 2], torch.tensor([n], device="cuda"), 0.125, torch.float16, torch.bfloat16)
            check(got[b, :, h], want, off + 2.0 ** -125)



@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("splits", [False, True])
@pytest.mark.parametrize("place,below", [(0, 100.0), (0, 140.0), (0, 200.0), (700, 140.0), (1100, 200.0), (1100, 500.0)])
def test_large_values_of_small_probability(built_library, form, splits, place, below):
    """v of 1e38 in a page whose keys' scores lie `below` powers of two under the others': its share is there as long as 2^-below of it is, and nothing else of it."""
    page, d, n = 32, 64, 1200
    slots = 2048 // page + (40 if splits else 0)
    keys, values, scales = sspmm_amd.new_cache(n // page + 1, 1, page, d, form)
    largest = 127.0 if form is torch.int8 else 448.0
    table = torch.full((1, slots), -1, dtype=torch.int32, device="cuda")
    table[0, :-(-n // page)] = torch.arange(-(-n // page))
    values.view(torch.int8).copy_(torch.full(values.shape, largest, device="cuda").to(form).view(torch.int8))
    scales[:, 1] = 1.0 / largest
    low = place // page
    keys.view(torch.int8)[low, :, :, 0] = torch.tensor(-largest, device="cuda").to(form).view(torch.int8)
    scales[:, 0] = below / largest
    scales[low, 1] = 1e38 / largest
    q = torch.zeros(1, 1, 1, d, device="cuda", dtype=torch.bfloat16)
    q[..., 0] = 1.0
    got = sspmm_amd.cache_attention(q, table, _ints([n]), keys, values, scales, scaling=math.log(2.0))
    big, p = scales[low, 1, 0].double() * largest, 2.0 ** (-largest * scales[low, 0, 0].double())
    count = min(page, n - low * page)
    want = ((n - count) + count * p * big) / (n - count + count * p)
    # a probability's half step in fp16, what scaling and the scales of 32 bits are off by, the result's half step; behind larger ones the page's
    # probabilities are nothing in fp16
    off = want * (2.0 ** -11 + 2.0 ** -18 + below * 2.0 ** -21 + 2.0 ** -8) + (count * p * big / (n - count) if place else 0.0)
    check(got.flatten(), want.expand(d), (off * 1.01).expand(d))



def test_rows_longer_than_their_table(built_library):
    """Tokens for which the table has no slot were dropped, and count all the same: query i sees positions 0 .. length - n + i, those behind the table masked."""
    page, d, n = 32, 64, 4
    pool = _filled(6, 1, page, d, torch.int8, seed=34)
    table = _ints([[4, 0], [1, 2], [3, 5], [0, 1], [2, 3]])
    lengths = [64, 65, 66, 90, 2 ** 31 - 1]
    q = _randn((5, n, 2, d), 35).half()
    got = sspmm_amd.cache_attention(q, table, _ints(lengths), *pool)
    for b, length in enumerate(lengths):
        k, v = row_of_cache(table[b], *pool, 64)
        visible = torch.tensor([min(64, length - n + 1 + i) for i in range(n)], device="cuda")
        for h in range(2):
            check(got[b, :, h], *attention(q[b, :, h], k[:, 0], v[:, 0], visible, 0.125, torch.float16, torch.float16), "row %d" % b)


@pytest.mark.parametrize("n,heads,kv,lengths", [(70, 4, 4, [70, 500, 1000]), (33, 8, 8, [800] * 20), (21, 6, 2, [64, 1900, 40]), (17, 8, 4, [300] * 40), (49, 4, 4, [9000])])
def test_in_place_with_several_tiles_of_queries(built_library, n, heads, kv, lengths):
    """Queries that fill more than a workgroup's places, the last tile in part: written over q they are the bits that they are beside it, however often."""
    table, pages = _table(lengths, 64, seed=39)
    cache = _filled(pages, kv, 64, 64, torch.int8, seed=40)
    q = (_randn((len(lengths), n, heads, 64), 41) * 2.0 ** torch.arange(n, device="cuda").view(1, n, 1, 1).remainder(5)).half()
    want = sspmm_amd.cache_attention(q, table, _ints(lengths), *cache)
    check_step(want, q, table, lengths, *cache, 0.125)
    for _ in range(10):
        x = q.clone()
        assert sspmm_amd.cache_attention(x, table, _ints(lengths), *cache, out=x) is x
        assert torch.equal(x, want)



def test_whatever_wants_gradients_is_refused(built_library):
    """Gradients backward and forward, of activations and of scales: none is dropped without a word."""
    from torch.autograd import forward_ad
    cache = sspmm_amd.new_cache(4, 2, 32, 64)
    table, n, off, start = _ints([[0, 1]]), _ints([40]), offsets_of([3]), _ints([0])
    q, k = _randn((1, 1, 4, 64), 1).half(), _randn((3, 2, 64), 2).half()

    def calls(wrap):
        keys, values, scales = cache
        return (lambda: sspmm_amd.prompt_attention(wrap(k), k, k, off), lambda: sspmm_amd.prompt_attention(k, wrap(k), k, off),
                lambda: sspmm_amd.prompt_attention(k, k, wrap(k), off), lambda: sspmm_amd.prompt_attention(k, k, k, off, out=wrap(k.clone())),
                lambda: sspmm_amd.cache_attention(wrap(q), table, n, *cache), lambda: sspmm_amd.cache_attention(q, table, n, keys, values, wrap(scales)),
                lambda: sspmm_amd.cache_attention(q, table, n, *cache, out=wrap(q.clone())),
                lambda: sspmm_amd.cache_write(wrap(k), k, off, start, table, *cache), lambda: sspmm_amd.cache_write(k, wrap(k), off, start, table, *cache),
                lambda: sspmm_amd.cache_write(k, k, off, start, table, keys, values, wrap(scales)))

    for call in calls(lambda t: t.detach().clone().requires_grad_()):
        with pytest.raises(RuntimeError, match="gradients"):
            call()
    with forward_ad.dual_level():
        for call in calls(lambda t: forward_ad.make_dual(t, torch.ones_like(t))):
            with pytest.raises(RuntimeError, match="gradients"):
                call()
        sspmm_amd.cache_write(k, k, off, start, table, *cache)  # (others than these, while a level is open, are as ever)
        assert torch.isfinite(sspmm_amd.cache_attention(q, table, n, *cache)).all()
    for f in (lambda x: sspmm_amd.prompt_attention(x, k, k, off), lambda x: sspmm_amd.prompt_attention(k, k, x, off)):
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (k,), (torch.ones_like(k),))
        with pytest.raises(RuntimeError):
            torch.func.vjp(f, k)
        with pytest.raises(RuntimeError):
            torch.func.vmap(f)(k.expand(2, 3, 2, 64))
    refs, length = _ints([1, 1, 0, 0]), _ints([40])
    for wanting in (cache[2].clone().requires_grad_(), None):
        with forward_ad.dual_level():
            scales = forward_ad.make_dual(cache[2], torch.ones_like(cache[2])) if wanting is None else wanting
            for call in (lambda: sspmm_amd.fork_pages(refs, table, length, _ints([0]), _ints([0]), *cache[:2], scales),
                         lambda: sspmm_amd.compact_pages(refs, table, *cache[:2], scales)):
                with pytest.raises(RuntimeError, match="gradients"):
                    call()
