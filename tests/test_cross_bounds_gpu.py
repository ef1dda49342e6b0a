"""Attention over an encoder's states where scores are at the end of the range."""
import pytest
import torch

import sspmm_amd
from serving_util import offsets_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sources", [1, 70, 3000, 20011])
@pytest.mark.parametrize("n", [1, 140])
def test_equal_scores_near_the_lowest(built_library, n, sources):
    """-2^127 - 1.75 * 2^126, about -3.19e38, for every state: finite and equal, so that each has the same share, and the result is the value that they all have."""
    d = 64
    q, k = torch.zeros(n, 2, d, dtype=torch.bfloat16, device="cuda"), torch.zeros(sources, 1, d, dtype=torch.bfloat16, device="cuda")
    q[..., 0], q[..., 40] = 2.0 ** 64, 2.0 ** 64
    k[..., 0], k[..., 40] = -2.0 ** 63, -1.75 * 2.0 ** 62
    v = torch.full_like(k, 5.0)
    for scaling in (1.0, 0.125, 1e-3):
        got = sspmm_amd.cross_attention(q, k, v, offsets_of([n]), offsets_of([sources]), scaling=scaling)
        assert (got == 5).all(), scaling
