"""Attention over shared pages where a plan, a scale or the sizes are at an end of what the interface allows."""
import pytest
import torch

import sspmm_amd
from serving_util import attention, check, check_step, row_of_cache
from test_prefix_attention_gpu import FORMATS, _ints, _pool, _randn, _tables

pytestmark = pytest.mark.gpu


def test_a_plan_whose_memory_is_not_what_its_sizes_say(built_library):
    """The words are counted before a kernel writes or reads them."""
    page, d, heads, kv = 32, 64, 4, 2
    table, lengths = _ints([[0, 1], [0, 2]]), _ints([40, 50])
    pool, q = _pool(4, kv, page, d, torch.int8, 1), _randn((2, 1, heads, d), 1).half()
    plan = sspmm_amd.plan_prefixes(table, lengths, 1, heads, kv, page)
    sizes = (plan.rows, plan.slots, plan.queries, plan.heads, plan.kv_heads, plan.page_size)
    words = plan.data.numel()
    for data in (plan.data[:words - 4].clone(), plan.data[:0].clone(), plan.data.view(torch.uint8)[:words].clone(), torch.zeros(2 * words, dtype=torch.int32, device="cuda")[::2],
                 plan.data[:1].expand(words)):
        other = sspmm_amd.PrefixPlan(*sizes, data)
        with pytest.raises(ValueError, match="plan"):
            sspmm_amd.plan_prefixes(table, lengths, 1, heads, kv, page, plan=other)
        with pytest.raises((TypeError, RuntimeError)):
            sspmm_amd.prefix_attention(q, table, other, *pool)
    # more than it needs is as good
    more = sspmm_amd.PrefixPlan(*sizes, torch.zeros(words + 100, dtype=torch.int32, device="cuda"))
    assert sspmm_amd.plan_prefixes(table, lengths, 1, heads, kv, page, plan=more) is more
    assert torch.equal(sspmm_amd.prefix_attention(q, table, more, *pool), sspmm_amd.prefix_attention(q, table, plan, *pool)) and not more.data[words:].any()


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("page", [32, 64, 128])
def test_scales_of_nan_where_nobody_looks(built_library, page, form):
    """Scales of NaN in free pages, the first among them, which slots without a page and entries outside the pool must not show; and in a last page that only the
    last of three drafted queries sees."""
    d, heads, kv, n = 64, 4, 2, 3
    #  page 0 and the pages 20 on are free; rows 0 to 2 share two pages
    table = _ints([[1, 2, 3, 4, -1], [1, 2, 5, 6, -1], [1, 2, 7, -1, -1], [8, -1, 9, 10, -1], [11, 999, 12, 13, -1], [14, 15, -1, -1, -1]])
    lengths = _ints([3 * page + 1, 4 * page, 2 * page + 5, 3 * page + 1, 3 * page + 7, page + 2])
    keys, values, scales = _pool(24, kv, page, d, form, 1)
    q = _randn((6, n, heads, d), 2).half()
    plan = sspmm_amd.plan_prefixes(table, lengths, n, heads, kv, page)
    want = sspmm_amd.prefix_attention(q, table, plan, keys, values, scales)
    check_step(want[[0, 1, 2, 5]], q[[0, 1, 2, 5]], table[[0, 1, 2, 5]], lengths[[0, 1, 2, 5]], keys, values, scales, d ** -0.5)
    assert torch.isfinite(want).all()
    scales[0], scales[16:] = float("nan"), float("nan")
    behind = table.clone()
    behind[:, 4] = 20  # (behind every row's end)
    behind[2, 3], behind[5, 2:] = 21, 0
    for t in (table, behind):
        assert torch.equal(sspmm_amd.prefix_attention(q, t, plan, keys, values, scales), want)
        assert torch.equal(sspmm_amd.prefix_attention(q, t, sspmm_amd.plan_prefixes(t, lengths, n, heads, kv, page), keys, values, scales), want)
    # the last pages of rows 0 and 3 have one token, that of row 5 two
    for row, last, blind in ((0, 4, 2), (3, 10, 2), (5, 15, 1)):
        for which in (0, 1):  # of keys, of values
            bad = scales.clone()
            bad[last, which] = float("nan")
            got = sspmm_amd.prefix_attention(q, behind, plan, keys, values, bad)
            others = [r for r in range(6) if r != row]
            assert torch.equal(got[others], want[others]) and torch.equal(got[row, :blind], want[row, :blind]) and torch.isnan(got[row, blind:]).all(), (row, which)


@pytest.mark.parametrize("rows,n,heads,kv", [(1024, 128, 32, 1), (1024, 1, 4096, 512), (3, 32768, 32, 4)])
def test_every_page_once_at_the_largest_sizes(built_library, rows, n, heads, kv):
    """As many queries and heads as a plan is for.

    Queries of zeros: all probabilities are one power of two, and so are the scales, so that sums of the codes are whole numbers below 2^24 of a unit, and exact.  What is left
    are the quotient (three roundings of 32 bits) and half a step of fp16.  Feature f has values in the pages of slots f, f + 32, ...: of at most 33 in a row, so that
    one that is lost or counted twice is 3 % of it.  And queries here and there against the formula, with others of any size."""
    page, d = 32, 32
    groups = [(130, [n + 1 + (7 * i) % 50 for i in range(rows // 2)]), (64, [n + 3 + (5 * i) % 70 for i in range(rows - rows // 2)])]
    table, lengths, pages = _tables(groups, page)
    keys, values, scales = _pool(pages, kv, page, d, torch.int8, 1)
    values.copy_(values.abs().clamp(min=1))
    slot_of = torch.zeros(pages, dtype=torch.int64, device="cuda")
    slots = torch.arange(table.size(1), device="cuda").expand(rows, -1)
    slot_of[table[table >= 0].long()] = slots[table >= 0]
    feature = torch.arange(d, device="cuda")
    values *= (feature == (slot_of % d)[:, None])[:, None, :, None]
    scales.fill_(2.0 ** -6)
    plan = sspmm_amd.plan_prefixes(table, lengths, n, heads, kv, page)
    got = sspmm_amd.prefix_attention(torch.zeros(rows, n, heads, d, dtype=torch.float16, device="cuda"), table, plan, keys, values, scales)
    for b in range(rows):
        length = int(lengths[b])
        _, v = row_of_cache(table[b], keys, values, scales, length)
        seen = torch.arange(length - n + 1, length + 1, device="cuda")
        want = (v.cumsum(0)[seen - 1] / seen[:, None, None].double()).repeat_interleave(heads // kv, 1)
        off = want * (2.0 ** -11 + 3 * 2.0 ** -24) * 1.01 + 2.0 ** -25
        far = ((got[b].double() - want).abs() - off).max().item()
        assert far <= 0, "row %d of %d off by %.3g more" % (b, length, far)
    q = _randn((rows, n, heads, d), 2).half()
    got = sspmm_amd.prefix_attention(q, table, plan, keys, values, scales)
    for b in sorted({0, 1, 2, rows // 2, rows - 1}):
        if b >= rows:
            continue
        length = int(lengths[b])
        k, v = row_of_cache(table[b], keys, values, scales, length)
        at = torch.tensor(sorted({0, n // 3, n - 2, n - 1} & set(range(n))), device="cuda")
        for h in range(0, heads, max(1, heads // 5)):
            want, off = attention(q[b, at, h], k[:, h // (heads // kv)], v[:, h // (heads // kv)], length - n + 1 + at, d ** -0.5, torch.float16, q.dtype)
            check(got[b, at, h], want, off, "row %d of %d, head %d" % (b, length, h))


@pytest.mark.parametrize("form", FORMATS)
def test_equal_scores_near_the_lowest(built_library, form):
    """-104 * 2^121 * 0.8 log2(e), about -3.19e38, for every position: finite and equal, each has the same share."""
    page, d, heads, kv = 32, 32, 2, 1
    table, lengths = _ints([[1, 2, 3, 4], [1, 2, 5, -1], [6, 7, 8, 0]]), _ints([100, 70, 128])
    keys, values, scales = sspmm_amd.new_cache(9, kv, page, d, form)
    keys[..., 0] = -104
    values.fill_(52)
    scales[:, 0], scales[:, 1] = 2.0 ** 121, 0.25
    q = torch.zeros(3, 1, heads, d, dtype=torch.float16, device="cuda")
    q[..., 0] = 1.0
    plan = sspmm_amd.plan_prefixes(table, lengths, 1, heads, kv, page)
    for got in (sspmm_amd.prefix_attention(q, table, plan, keys, values, scales, scaling=0.8), sspmm_amd.cache_attention(q, table, lengths, keys, values, scales, scaling=0.8)):
        assert (got == 13).all()
