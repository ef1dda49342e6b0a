"""Attention over shared pages where a plan, a scale or the sizes are at an end of what the interface allows."""
import pytest
import torch

import sspmm_amd
from test_prefix_attention_gpu import _ints, _pool, _randn

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
