"""Draws whose uniform number lies on a border between two tokens: the first whose running sum EXCEEDS its share of all is the one behind the border."""
import pytest
import torch

import sspmm_amd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("level", [2.5, float("inf")])
@pytest.mark.parametrize("vocab", [64, 1024, 4096, 65536, 98304, 131072])
def test_borders_between_equal_logits(built_library, vocab, level):
    """Weights are all the same, sums whole numbers and borders multiples of 1 / kept: u * kept is exact, and so is the token."""
    rows = 64
    logits = torch.full((rows, vocab), level, dtype=torch.bfloat16, device="cuda")
    uniform = torch.arange(rows, device="cuda") / rows  # (exact)
    for top_k, top_p, kept in ((0, 1.0, vocab), (0, 0.5, vocab // 2), (vocab // 4, 1.0, vocab // 4), (vocab // 2, 0.75, 3 * vocab // 8)):
        tokens = sspmm_amd.sample_tokens(logits, uniform, 0.5, top_k, top_p)
        assert torch.equal(tokens.cpu(), torch.tensor([int(u * kept) for u in uniform.double().tolist()], dtype=torch.int32)), (top_k, top_p)


@pytest.mark.parametrize("vocab", [20000, 90000])
def test_borders_among_the_first_of_many(built_library, vocab):
    """The same of 4096 equal logits among others that weigh nothing beside them."""
    rows, kept = 64, 4096
    logits = torch.full((rows, vocab), -200.0, dtype=torch.float32, device="cuda")
    at = torch.randperm(vocab, generator=torch.Generator(device="cuda").manual_seed(vocab), device="cuda")[:kept].sort().values
    logits[:, at] = 1.0
    uniform = torch.arange(rows, device="cuda") / rows
    tokens = sspmm_amd.sample_tokens(logits, uniform)
    assert torch.equal(tokens.long(), at[(uniform.double() * kept).long()])
