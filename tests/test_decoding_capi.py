"""What the C entries of prefix and cross attention and of the draw refuse, before they touch the device; and the Python ones without a GPU."""
import pytest
import torch

import sspmm_amd

A = 64  # any aligned non-null address: refused calls never look at it


@pytest.fixture
def L(built_library):
    from sspmm_amd import _lib
    return _lib.lib()


def _changed(good, call):
    def run(*changes):
        args = list(good)
        for i, v in changes:
            args[i] = v
        return call(*args)
    return run


def test_cross_attention(L):
    size = L.sspmm_cross_attention_workspace_bytes
    need = size(1, 2, 20000, 4, 2, 64)
    assert need > 0 and size(1, 4000, 20000, 4, 2, 64) == 0 and size(0, 2, 20000, 4, 2, 64) == 0 and size(1, 2, 20000, 4, 3, 64) == 0 and size(1, 2, -1, 4, 2, 64) == 0
    #        type seqs tokens sources heads kv d offsets source_offsets q row head k row head v row head scale out row head workspace bytes stream
    good = [0, 1, 2, 20000, 4, 2, 64, A, A, A, 256, 64, A, 128, 64, A, 128, 64, 0.125, A, 256, 64, A, need, None]
    run = _changed(good, L.sspmm_cross_attention)
    for i, v in ((0, 2), (0, -1), (1, -1), (2, -1), (2, (1 << 30) + 1), (3, -1), (3, (1 << 30) + 1), (4, 3), (4, 0), (5, 0), (6, 48), (6, 256), (7, None), (8, None), (9, None),
                 (9, A + 8), (10, 252), (10, 56), (10, 1 << 23), (11, 4), (11, -8), (12, None), (13, 1 << 23), (15, None), (16, 32), (18, 0.0), (18, -1.0),
                 (18, float("nan")), (18, float("inf")), (18, 3.0e38), (19, None), (19, A + 2), (20, 60), (21, 3), (22, None), (22, A + 8), (23, need - 1)):
        assert run((i, v)) == 1, (i, v)
    assert run((1, 0), (7, None), (8, None)) == 0 and run((2, 0), (9, None)) == 0
    # queries times heads of a group are counted in 31 bits
    assert run((2, 1 << 30)) == 1


def test_plan_and_prefix_attention(L):
    size, room = L.sspmm_prefix_plan_bytes, L.sspmm_prefix_attention_workspace_bytes
    need, states = size(4, 1, 8, 2), room(4, 1, 8, 2, 64)
    assert need > 0 and states > 0 and size(1024, 1, 8, 2) > need
    for sizes in ((0, 1, 8, 2), (1025, 1, 8, 2), (4, 0, 8, 2), (4, 1, 7, 2), (4, 1, 8, 0), (4, 1, 0, 2), (4, 1 << 18, 8, 2), (1024, 512, 16, 2), (-1, 1, 8, 2)):
        assert size(*sizes) == 0 and room(*sizes, 64) == 0, sizes
    assert room(4, 1, 8, 2, 65) == 0
    #        table rows slots lengths page queries heads kv plan bytes stream
    plan = _changed([A, 4, 8, A, 32, 1, 8, 2, A, need, None], L.sspmm_plan_prefixes)
    for i, v in ((0, None), (1, -1), (1, 1025), (2, 0), (2, 1 << 26), (3, None), (4, 16), (4, 0), (5, -1), (6, 7), (7, 3), (7, 0), (8, None), (8, A + 8), (9, need - 1)):
        assert plan((i, v)) == 1, (i, v)
    assert plan((1, 0), (0, None)) == 0 and plan((5, 0), (8, None)) == 0
    #        type form rows queries heads q seq row head table slots plan bytes pages kv page d keys values scales scale out seq row head workspace bytes stream
    good = [0, 0, 4, 1, 8, A, 512, 512, 64, A, 8, A, need, 100, 2, 32, 64, A, A, A, 0.125, A, 512, 512, 64, A, states, None]
    run = _changed(good, L.sspmm_prefix_attention)
    for i, v in ((0, 2), (1, 2), (2, -1), (2, 1025), (3, -1), (4, 7), (4, 0), (5, None), (5, A + 8), (6, 4), (6, -8), (7, 32), (8, 4), (9, None), (10, 0), (10, 1 << 26), (11, None),
                 (11, A + 8), (12, need - 1), (13, 0), (14, 3), (15, 48), (16, 96), (17, None), (18, None), (18, A + 8), (19, None), (20, 0.0), (20, float("inf")), (21, None), (22, 4),
                 (23, 8), (24, 4), (25, None), (25, A + 4), (26, states - 1)):
        assert run((i, v)) == 1, (i, v)
    assert run((2, 0)) == 0 and run((3, 0)) == 0


def test_sample_tokens(L):
    size = L.sspmm_sample_tokens_workspace_bytes
    need = size(2, 100000)
    assert need > 0 and size(2, 1000) == 0 and size(1000, 100000) == 0 and size(0, 100000) == 0 and size(2, 0) == 0
    #        type rows vocab logits stride uniform temperature all top_k all top_p all min_p all tokens probabilities workspace bytes stream
    good = [0, 2, 100000, A, 100000, A, A, 1.0, A, 0, A, 1.0, A, 0.0, A, A, A, need, None]
    run = _changed(good, L.sspmm_sample_tokens)
    for i, v in ((0, 3), (0, -1), (1, -1), (1, 1 << 22), (2, 0), (2, (1 << 24) + 1), (3, None), (3, A + 1), (4, -1), (5, None), (5, A + 2), (6, A + 1), (8, A + 2), (10, A + 2), (12, A + 2),
                 (14, None), (14, A + 2), (15, A + 2), (16, None), (16, A + 8), (17, need - 1)):
        assert run((i, v)) == 1, (i, v)
    assert run((0, 2), (3, A + 2)) == 1 and run((1, 0), (3, None)) == 0


def test_python_entries_want_a_gpu(built_library):
    q, k = torch.zeros(4, 2, 64, dtype=torch.float16), torch.zeros(4, 1, 64, dtype=torch.float16)
    ints = torch.zeros(2, dtype=torch.int32)
    keys, values, scales = sspmm_amd.new_cache(2, 1, 32, 64, device="cpu")
    table = torch.zeros(1, 1, dtype=torch.int32)
    plan = sspmm_amd.PrefixPlan(1, 1, 4, 2, 1, 32, ints)
    for call in (lambda: sspmm_amd.cross_attention(q, k, k, ints, ints), lambda: sspmm_amd.plan_prefixes(table, ints[:1], 1, 2, 1, 32),
                 lambda: sspmm_amd.prefix_attention(q[None], table, plan, keys, values, scales),
                 lambda: sspmm_amd.sample_tokens(torch.zeros(2, 8), torch.zeros(2))):
        with pytest.raises(TypeError):
            call()
