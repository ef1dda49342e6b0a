"""Attention over the paged cache for rows that share leading pages, against the formula in 64 bits, and what a plan finds."""
import pytest
import torch

import sspmm_amd
from serving_util import check_step, offsets_of

pytestmark = pytest.mark.gpu

FORMATS = [torch.int8, torch.float8_e4m3fn]
UNIT = 32  # positions that a plan counts as one


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _randn(shape, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda")


def _pool(pages, kv, page, d, form, seed):
    """A pool of codes of every size and scales between 1/200 and 1/50."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    keys, values, scales = sspmm_amd.new_cache(pages, kv, page, d, form)
    for t in (keys, values):
        if form is torch.int8:
            t.copy_(torch.randint(-127, 128, t.shape, generator=g, device="cuda"))
        else:
            t.copy_((torch.randn(t.shape, generator=g, device="cuda") * 40).clamp(-448, 448).to(form))
    scales.copy_(torch.rand(scales.shape, generator=g, device="cuda") * 0.015 + 0.005)
    return keys, values, scales


def _tables(groups, page, seed=0):
    """(page_table, lengths, pages) of rows as forks leave them: groups of (shared tokens, [tokens of its own for each row])."""
    rows = sorted((j, i) for i, (_, each) in enumerate(groups) for j in range(len(each)))
    lengths = [groups[i][0] + groups[i][1][j] for j, i in rows]
    need = sum(s // page for s, _ in groups) + sum(-(-n // page) - groups[i][0] // page for n, (_, i) in zip(lengths, rows))
    g = torch.Generator()
    g.manual_seed(seed)
    at = torch.randperm(need + 3, generator=g).to(torch.int32)
    table = torch.full((len(rows), max(max(-(-n // page) for n in lengths), 1)), -1, dtype=torch.int32)
    taken, fronts = 0, []
    for shared, _ in groups:
        fronts.append(at[taken:taken + shared // page])
        taken += shared // page
    for row, (n, (_, i)) in enumerate(zip(lengths, rows)):
        front, more = fronts[i], -(-n // page) - fronts[i].numel()
        table[row, :front.numel()] = front
        table[row, front.numel():front.numel() + more] = at[taken:taken + more]
        taken += more
    return table.cuda(), _ints(lengths), need + 3


def _units(plan):
    """Units of all jobs, which is what the workgroups of a head of the cache go over."""
    words = plan.data
    jobs = words[4:4 + 12 * int(words[0])].view(-1, 12)
    return int((jobs[:, 2] - jobs[:, 1]).sum())


def _run(groups, n, heads, kv, page, d, dtype, form, seed=0):
    table, lengths, pages = _tables(groups, page, seed)
    pool = _pool(pages, kv, page, d, form, seed + 1)
    q = _randn((lengths.numel(), n, heads, d), seed + 2).to(dtype)
    print(groups, n, heads, kv, page, d, dtype, form, flush=True)
    plan = sspmm_amd.plan_prefixes(table, lengths, n, heads, kv, page)
    got = sspmm_amd.prefix_attention(q, table, plan, *pool)
    check_step(got, q, table, lengths, *pool, d ** -0.5)
    return table, lengths, pool, q, plan, got


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("groups,n,heads,kv,page,d", [
    ([(70, [5, 1])], 1, 4, 2, 32, 64), ([(1, [1])], 1, 1, 1, 32, 32), ([(0, [1, 33, 64])], 1, 2, 2, 64, 64), ([(128, [1, 2, 3, 60, 70])], 1, 8, 2, 128, 128),
    ([(333, [5, 40]), (0, [77])], 3, 12, 12, 32, 64), ([(640, [1] * 9)], 1, 8, 2, 64, 128), ([(200, [3, 7, 11]), (97, [1, 50]), (64, [9])], 2, 6, 1, 32, 32),
    ([(1000, [1, 100, 30, 77]), (500, [20, 1, 3])], 1, 16, 2, 64, 64), ([(300, [2, 8])], 7, 8, 1, 32, 128), ([(96, [1] * 20)], 5, 4, 4, 32, 64)])
def test_against_the_formula(built_library, groups, n, heads, kv, page, d, dtype, form):
    _run(groups, n, heads, kv, page, d, dtype, form, seed=len(groups) + d)


@pytest.mark.parametrize("form", FORMATS)
def test_many_rows_and_long_prefixes(built_library, form):
    _run([(5000, [(31 * i * i) % 300 + 1 for i in range(70)])], 1, 4, 2, 64, 64, torch.bfloat16, form, seed=3)
    _run([(20001, [5, 400, 77])], 1, 8, 2, 128, 128, torch.float16, form, seed=4)
    _run([(64 * i, [1 + i, 2]) for i in range(40)], 1, 2, 1, 64, 32, torch.float16, form, seed=5)


def test_as_many_rows_as_a_plan_takes(built_library):
    page, d = 32, 32
    groups = [(96, [1 + (7 * i) % 50 for i in range(500)]), (40, [1 + i % 20 for i in range(24)])] + [(33 + i % 3, [1 + i % 9]) for i in range(500)]
    table, lengths, pages = _tables(groups, page)
    assert lengths.numel() == 1024
    pool = _pool(pages, 1, page, d, torch.int8, 1)
    q = _randn((1024, 1, 2, d), 2).half()
    plan = sspmm_amd.plan_prefixes(table, lengths, 1, 2, 1, page)
    # three pages once for 500 rows, one for 24, and what every row has behind
    tokens = lengths.tolist()
    shared = [0] * 1024
    where = sorted((j, i) for i, (_, each) in enumerate(groups) for j in range(len(each)))
    for r, (_, i) in enumerate(where):
        shared[r] = 96 if i == 0 else 32 if i == 1 else 0
    assert _units(plan) == 3 * -(-500 * 2 // 32) + 1 * -(-24 * 2 // 32) + sum(-(-(n - s) // UNIT) for n, s in zip(tokens, shared))
    got = sspmm_amd.prefix_attention(q, table, plan, *pool)
    want = sspmm_amd.cache_attention(q, table, lengths, *pool)
    at = list(range(0, 1024, 53)) + [1023]
    check_step(got[at], q[at], table[at], lengths[at], *pool, d ** -0.5)
    # both are within the formula's bounds; so the largest distance of the two is within twice the bound of values up to 1.3 * 127 / 50
    assert (got.float() - want.float()).abs().max() < 0.02


@pytest.mark.parametrize("groups,heads,kv,page", [([(0, [4096 + 120 * i]) for i in range(32)], 16, 16, 32), ([(0, [22000 + 900 * i]) for i in range(8)], 64, 64, 64),
                                                  ([(3200, [3000 + 5 * i, 3500]) for i in range(200)], 2, 1, 64), ([(30000, [500, 9000, 20000]), (25000, [4000] * 5)], 32, 32, 64)])
def test_more_tiles_than_places_and_long_rows(built_library, groups, heads, kv, page):
    """Jobs are no more than the plan has room for, where their number grows with the root of the rows' lengths, and where it is bounded."""
    table, lengths, pages = _tables(groups, page)
    rows, d = lengths.numel(), 32
    pool = _pool(pages, kv, page, d, torch.int8, 1)
    q = _randn((rows, 1, heads, d), 2).half()
    plan = sspmm_amd.plan_prefixes(table, lengths, 1, heads, kv, page)
    assert rows < int(plan.data[0]) <= (plan.data.numel() - 4 - 12 * rows) // 12
    got = sspmm_amd.prefix_attention(q, table, plan, *pool)
    at = list(range(0, rows, 1 + rows // 9)) + [rows - 1]
    check_step(got[at], q[at], table[at], lengths[at], *pool, d ** -0.5)
    want = sspmm_amd.cache_attention(q, table, lengths, *pool)
    assert (got.float() - want.float()).abs().max() < 0.02


@pytest.mark.parametrize("rows,n,heads,kv", [(1024, 128, 32, 1), (1024, 1, 4096, 512), (3, 32768, 32, 4)])
def test_the_largest_sizes(built_library, rows, n, heads, kv):
    """As many queries and heads as a plan is for, of many rows and of few."""
    page, d = 32, 32
    groups = [(130, [n + 1 + (7 * i) % 50 for i in range(rows // 2)]), (64, [n + 3 + (5 * i) % 70 for i in range(rows - rows // 2)])]
    table, lengths, pages = _tables(groups, page)
    pool = _pool(pages, kv, page, d, torch.int8, 1)
    q = _randn((rows, n, heads, d), 2).half()
    plan = sspmm_amd.plan_prefixes(table, lengths, n, heads, kv, page)
    assert rows <= int(plan.data[0]) <= (plan.data.numel() - 4 - 12 * rows) // 12
    got = sspmm_amd.prefix_attention(q, table, plan, *pool)
    want = sspmm_amd.cache_attention(q, table, lengths, *pool)
    assert (got.float() - want.float()).abs().max() < 0.02


def test_what_a_plan_shares(built_library):
    page, rows = 32, 6
    table = _ints([[1, 2, 3, 4, 5], [1, 2, 3, 9, 8], [1, 2, 3, 4, 7], [1, 10, 11, 12, 13], [20, 21, -1, -1, -1], [-1, 2, 3, 4, 5]])
    lengths = _ints([150, 130, 160, 129, 40, 150])
    plan = sspmm_amd.plan_prefixes(table, lengths, 1, 2, 1, page)
    # rows 0, 1 and 2 share three pages with row 0, row 3 one: three for three save six pages, one for four three
    own = [150 - 96, 130 - 96, 160 - 96, 129, 40, 150]
    assert _units(plan) == 3 + sum(-(-n // UNIT) for n in own)
    # a row's pages are shared as far as they lie whole in front of its first query
    for n, tokens, shared in ((1, 97, 3), (1, 96, 3), (1, 95, 2), (2, 97, 3), (3, 97, 2), (40, 97, 1), (97, 97, 0), (200, 97, 0)):
        two = sspmm_amd.plan_prefixes(table[:1].expand(2, 5).contiguous(), _ints([tokens, tokens]), n, 1, 1, page)
        tiles, own_units = -(-2 * n // 32), -(-n // 32) * -(-(tokens - 32 * shared) // UNIT)
        assert _units(two) == tiles * shared + 2 * own_units, (n, tokens, shared)
    # the same, made anew in place
    again = sspmm_amd.plan_prefixes(table, lengths - 32, 1, 2, 1, page, plan=plan)
    assert again is plan and _units(plan) == 3 + sum(-(-(n - 32) // UNIT) for n in (150, 130, 160, 129 + 0, 40, 150)) - 3 * 3
    empty = sspmm_amd.plan_prefixes(table, 0 * lengths, 1, 2, 1, page)
    assert _units(empty) == 0


@pytest.mark.parametrize("others", [0, 9])
def test_where_long_rows_part(built_library, others):
    """Rows of thousands of pages, as far as they are the same; alone, and among others without a token."""
    slots = 5000
    base = torch.arange(slots, dtype=torch.int32, device="cuda")
    for shared in (1, 63, 64, 511, 512, 513, 1536, 2047, 2048, 2049, 4095, 4096, 4097, 4999, 5000):
        table = torch.stack([base, base])
        table[1, shared:] += slots
        if shared + 1 < slots:
            table[1, shared + 1] -= slots  # (the same again behind it)
        table = torch.cat([table, table[:1].expand(others, slots)])
        plan = sspmm_amd.plan_prefixes(table, _ints([32 * slots + 1, 32 * slots] + [0] * others), 1, 1, 1, 32)
        assert _units(plan) == shared + 2 * (slots - shared), shared


@pytest.mark.parametrize("form", FORMATS)
def test_short_empty_and_overlong_rows(built_library, form):
    """Rows without a token, with fewer tokens than queries, and with more than their table has room for; queries that see nothing are zeros."""
    page, d, heads, kv, n = 32, 64, 4, 2, 3
    table = _ints([[1, 2, 3], [1, 2, 4], [1, 2, 5], [1, 6, 7], [1, 2, 3]])
    pool = _pool(9, kv, page, d, form, 1)
    for lengths in ([70, 0, 65, 2, 96], [1, 2, 3, 0, 0], [0, 0, 0, 0, 0], [96, 96, 64, 33, 96]):
        q = _randn((5, n, heads, d), 2).half()
        m = _ints(lengths)
        got = sspmm_amd.prefix_attention(q, table, sspmm_amd.plan_prefixes(table, m, n, heads, kv, page), *pool)
        check_step(got, q, table, m, *pool, d ** -0.5, lengths)
    long = _ints([97, 98, 150, 1 << 30, 99])
    q = _randn((5, n, heads, d), 3).half()
    got = sspmm_amd.prefix_attention(q, table, sspmm_amd.plan_prefixes(table, long, n, heads, kv, page), *pool)
    want = sspmm_amd.cache_attention(q, table, long, *pool)
    assert torch.isfinite(got).all() and (got.float() - want.float()).abs().max() < 0.02


@pytest.mark.parametrize("form", FORMATS)
def test_positions_without_a_page_are_masked(built_library, form):
    """Slots without a page, and entries that name none of the pool's, in what is shared and behind: as cache_attention has them."""
    page, d, kv, heads = 32, 64, 2, 4
    pool = _pool(12, kv, page, d, form, 5)
    q = _randn((4, 1, heads, d), 6).half()
    lengths = _ints([150, 140, 130, 40])
    for rows in ([[1, 2, 3, 4, 5], [1, 2, -1, 4, 6], [1, 2, 3, -1, -1], [-1, 2, 0, 0, 0]], [[1, 99, 3, 4, 5], [1, 99, 3, 4, 6], [1, 99, 3, 4, 7], [1, 99, 3, 4, 5]],
                 [[99, 2, 3, 4, 5], [99, 2, 3, 4, 6], [99, 2, 3, 4, 7], [99, 2, 0, 0, 0]], [[-1] * 5] * 4):
        table = _ints(rows)
        got = sspmm_amd.prefix_attention(q, table, sspmm_amd.plan_prefixes(table, lengths, 1, heads, kv, page), *pool)
        want = sspmm_amd.cache_attention(q, table, lengths, *pool)
        assert torch.isfinite(got).all() and (got.float() - want.float()).abs().max() < 0.02, rows
        assert torch.equal(got == 0, want == 0)


@pytest.mark.parametrize("form", FORMATS)
def test_nothing_comes_from_behind_a_row(built_library, form):
    """What lies behind the rows in their last pages, and pages of no row, may be anything: codes, and in e4m3 NaN."""
    groups, n, heads, kv, page, d = [(100, [5, 20, 33]), (0, [3])], 2, 4, 2, 64, 64
    table, lengths, pages = _tables(groups, page)
    keys, values, scales = _pool(pages, kv, page, d, form, 7)
    q = _randn((4, n, heads, d), 8).half()
    plan = sspmm_amd.plan_prefixes(table, lengths, n, heads, kv, page)
    want = sspmm_amd.prefix_attention(q, table, plan, keys, values, scales)
    used = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    for b in range(4):
        for slot in range(-(-int(lengths[b]) // page)):
            used[int(table[b, slot]), :min(page, int(lengths[b]) - slot * page)] = True
    for fill in (127, -127) if form is torch.int8 else (0x7F, -1):  # (e4m3: NaN of either sign)
        k, v = keys.clone(), values.clone()
        k.view(torch.int8).masked_fill_(~used[:, None, :, None], fill)
        v.view(torch.int8).masked_fill_(~used[:, None, None, :], fill)
        assert torch.equal(sspmm_amd.prefix_attention(q, table, plan, k, v, scales), want)


@pytest.mark.parametrize("order", ["projection", "rows apart", "features apart", "in place"])
def test_other_orders_in_memory(built_library, order):
    groups, n, heads, kv, page, d = [(150, [5, 20, 33])], 2, 8, 2, 32, 64
    table, lengths, pages = _tables(groups, page)
    pool = _pool(pages, kv, page, d, torch.int8, 9)
    out = None
    if order == "projection":
        q = _randn((3, n, (heads + 4) * d), 1).half()[..., 2 * d:(heads + 2) * d].view(3, n, heads, d)
    elif order == "rows apart":
        q = _randn((n, 3, heads, d), 1).half().transpose(0, 1)
        out = torch.zeros(n, 3, heads + 1, d, device="cuda", dtype=torch.float16)[:, :, 1:].transpose(0, 1)
    elif order == "features apart":
        q = _randn((d, 3, n, heads), 1).half().permute(1, 2, 3, 0)
    else:
        out = q = _randn((3, n, heads, d), 1).half()
    copy = q.clone()
    got = sspmm_amd.prefix_attention(q, table, sspmm_amd.plan_prefixes(table, lengths, n, heads, kv, page), *pool, out=out)
    assert out is None or got is out
    check_step(got, copy, table, lengths, *pool, d ** -0.5)


def test_a_pool_beyond_32_bits(built_library):
    page, kv, d, pages = 128, 8, 128, 36000
    keys, values = (torch.zeros(s, dtype=torch.int8, device="cuda") for s in ((pages, kv, page, d), (pages, kv, d, page)))
    scales = torch.full((pages, 2, kv), 0.01, device="cuda")
    table = _ints([[35990, 3, 35991, 35999], [35990, 3, 35992, -1], [35990, 3, 35993, -1]])
    lengths = _ints([500, 300, 290])
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    for p in set(table.flatten().tolist()) - {-1}:
        for t in (keys, values):
            t[p] = torch.randint(-127, 128, t[p].shape, generator=g, device="cuda")
    q = _randn((3, 1, 16, d), 3).bfloat16()
    plan = sspmm_amd.plan_prefixes(table, lengths, 1, 16, kv, page)
    check_step(sspmm_amd.prefix_attention(q, table, plan, keys, values, scales), q, table, lengths, keys, values, scales, d ** -0.5)


def test_graphs_streams_and_twice_the_same(built_library):
    """A plan made in place inside a graph and outside of it, two graphs replayed in either order, calls on two streams at once."""
    groups, n, heads, kv, page, d = [(3000, [5, 700, 33]), (100, [9, 4])], 1, 8, 2, 64, 128
    table, lengths, pages = _tables(groups, page)
    pool = _pool(pages, kv, page, d, torch.int8, 11)
    qs = [_randn((5, n, heads, d), 30 + i).bfloat16() for i in range(2)]
    plan = sspmm_amd.plan_prefixes(table, lengths, n, heads, kv, page)
    first = sspmm_amd.prefix_attention(qs[0], table, plan, *pool)
    assert all(torch.equal(sspmm_amd.prefix_attention(qs[0], table, sspmm_amd.plan_prefixes(table, lengths, n, heads, kv, page), *pool), first) for _ in range(3))
    torch.cuda.synchronize()
    outs, graphs = [torch.zeros_like(q) for q in qs], [torch.cuda.CUDAGraph() for _ in qs]
    with torch.cuda.graph(graphs[0]):  # (its own plan, made each time)
        sspmm_amd.prefix_attention(qs[0], table, sspmm_amd.plan_prefixes(table, lengths, n, heads, kv, page), *pool, out=outs[0])
    with torch.cuda.graph(graphs[1]):  # (one made outside)
        sspmm_amd.prefix_attention(qs[1], table, plan, *pool, out=outs[1])
    start = lengths.clone()
    for turn in range(4):
        lengths.copy_(start - 40 * turn)
        for i, q in enumerate(qs):
            q.copy_(_randn(q.shape, 40 + 2 * turn + i))
        sspmm_amd.plan_prefixes(table, lengths, n, heads, kv, page, plan=plan)
        want = [sspmm_amd.prefix_attention(q, table, plan, *pool) for q in qs]
        for g in graphs if turn % 2 else graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
        check_step(want[0], qs[0], table, lengths.clamp(min=0), *pool, d ** -0.5)
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for turn in range(6):
        for s, q in zip(streams, qs):
            with torch.cuda.stream(s):
                got.append(sspmm_amd.prefix_attention(q, table, plan, *pool))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i % 2]) for i, x in enumerate(got))


@pytest.mark.parametrize("size", [2.0 ** -12, 1.0, 300.0])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_queries_of_any_size(built_library, size, dtype):
    groups, n, heads, kv, page, d = [(200, [5, 60])], 1, 4, 2, 32, 64
    table, lengths, pages = _tables(groups, page)
    pool = _pool(pages, kv, page, d, torch.int8, 12)
    q = (_randn((2, n, heads, d), 13) * size).to(dtype)
    got = sspmm_amd.prefix_attention(q, table, sspmm_amd.plan_prefixes(table, lengths, n, heads, kv, page), *pool)
    check_step(got, q, table, lengths, *pool, d ** -0.5)


def test_what_forks_leave(built_library):
    """Rows forked by fork_pages, forked again, and written to: the plan finds what they share."""
    page, kv, d, heads = 32, 2, 64, 4
    keys, values, scales = sspmm_amd.new_cache(40, kv, page, d)
    refs, table, lengths = torch.zeros(40, dtype=torch.int32, device="cuda"), torch.full((6, 6), -1, dtype=torch.int32, device="cuda"), _ints([110, 0, 0, 0, 0, 40])
    starts, counts = _ints([0] * 6), [110, 0, 0, 0, 0, 40]
    x = _randn((150, 2, kv, d), 1).half()
    sspmm_amd.reserve_pages(refs, table, starts, offsets_of(counts), page)
    sspmm_amd.cache_write(x[:, 0], x[:, 1], offsets_of(counts), starts, table, keys, values, scales)
    sspmm_amd.fork_pages(refs, table, lengths, _ints([0, 0]), _ints([1, 2]), keys, values, scales)
    for step in range(40):
        counts = [1, 1, 1, 0, 0, 1] if step < 20 else [1] * 6
        if step == 20:
            sspmm_amd.fork_pages(refs, table, lengths, _ints([2, 2]), _ints([3, 4]), keys, values, scales)
        new = _randn((sum(counts), 2, kv, d), 100 + step).half()
        sspmm_amd.reserve_pages(refs, table, lengths, offsets_of(counts), page)
        sspmm_amd.cache_write(new[:, 0], new[:, 1], offsets_of(counts), lengths, table, keys, values, scales)
        lengths += _ints(counts)
        if step % 13 == 0 or step == 39:
            q = _randn((6, 1, heads, d), 200 + step).half()
            plan = sspmm_amd.plan_prefixes(table, lengths, 1, heads, kv, page)
            check_step(sspmm_amd.prefix_attention(q, table, plan, keys, values, scales), q, table, lengths, keys, values, scales, d ** -0.5, step)
    # rows 0 to 4 share three pages (110 tokens when they were forked)
    assert _units(plan) == 3 + sum(-(-(n - s) // UNIT) for n, s in zip(lengths.tolist(), (96, 96, 96, 96, 96, 0)))


def test_refusals(built_library):
    page, d, heads, kv = 32, 64, 4, 2
    pool = sspmm_amd.new_cache(4, kv, page, d)
    table, lengths, q = _ints([[0, 1], [0, 2]]), _ints([40, 50]), _randn((2, 1, heads, d), 1).half()
    plan_of, attend = sspmm_amd.plan_prefixes, sspmm_amd.prefix_attention
    plan = plan_of(table, lengths, 1, heads, kv, page)
    for call, kind in (((table.long(), lengths, 1, heads, kv, page), TypeError), ((table, lengths.cpu(), 1, heads, kv, page), TypeError), ((table.cpu(), lengths, 1, heads, kv, page), TypeError),
                       ((table[0], lengths, 1, heads, kv, page), ValueError), ((table, lengths[:1], 1, heads, kv, page), ValueError), ((table, lengths, 1, 3, kv, page), ValueError),
                       ((table, lengths, 1, heads, 0, page), ValueError), ((table, lengths, -1, heads, kv, page), ValueError), ((table, lengths, 1, heads, kv, 48), ValueError),
                       ((table[:, :0], lengths, 1, heads, kv, page), ValueError), ((table, lengths, 1 << 19, heads, kv, page), ValueError),
                       ((table[:1].expand(1025, 2).contiguous(), lengths[:1].expand(1025).contiguous(), 1, heads, kv, page), ValueError),
                       ((table, lengths, 2, heads, kv, page, plan), ValueError), ((table, lengths, 1, heads, kv, 64, plan), ValueError)):
        with pytest.raises(kind):
            plan_of(*call)
    for call, kind in (((q.float(), table, plan, *pool), TypeError), ((q[:1], table, plan, *pool), ValueError), ((q, table[:1], plan, *pool), ValueError),
                       ((q, table[:, :1].contiguous(), plan, *pool), ValueError), ((q, table.t(), plan, *pool), TypeError), ((q[:, :, :2], table, plan, *pool), ValueError),
                       ((q.expand(2, 3, heads, d), table, plan, *pool), ValueError), ((q[..., :32], table, plan, *pool), ValueError), ((q, table, plan, pool[0].float(), *pool[1:]), TypeError),
                       ((q, table, plan, *sspmm_amd.new_cache(4, 4, page, d)), ValueError), ((q, table, plan, *sspmm_amd.new_cache(4, kv, 64, d)), ValueError),
                       ((q, table, plan, *pool, 0.0), ValueError), ((q, table, plan, *pool, None, q[:1]), ValueError)):
        with pytest.raises(kind):
            attend(*call)
    with pytest.raises(RuntimeError, match="gradients"):
        attend(q.clone().requires_grad_(), table, plan, *pool)
    # nothing to do
    none = plan_of(table[:0], lengths[:0], 1, heads, kv, page)
    assert attend(q[:0], table[:0], none, *pool).shape == (0, 1, heads, d)
    none = plan_of(table, lengths, 0, heads, kv, page)
    assert attend(q[:, :0], table, none, *pool).shape == (2, 0, heads, d)
