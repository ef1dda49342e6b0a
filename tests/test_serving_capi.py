"""What the C entries of the serving operators refuse, before they touch the device; and the Python ones without a GPU."""
import pytest
import torch

import sspmm_amd

A = 64  # any aligned non-null address: refused calls never look at it


@pytest.fixture
def L(built_library):
    from sspmm_amd import _lib
    return _lib.lib()


def _changed(good, call):
    """call(*good with one argument replaced) for (index, value)."""
    def run(*changes):
        args = list(good)
        for i, v in changes:
            args[i] = v
        return call(*args)
    return run


def test_prompt_attention(L):
    #        type seqs tokens heads kv d offsets q row head k row head v row head causal scale out row head stream
    good = [0, 1, 8, 4, 2, 64, A, A, 256, 64, A, 128, 64, A, 128, 64, 1, 0.125, A, 256, 64, None]
    run = _changed(good, L.sspmm_prompt_attention)
    for i, v in ((0, 2), (0, -1), (1, -1), (2, -1), (2, (1 << 30) + 1), (3, 3), (3, 0), (4, 0), (5, 48), (5, 256), (6, None), (7, None), (7, A + 8), (8, 252), (8, 56),
                 (8, 1 << 23), (9, 4), (9, -8), (10, None), (11, 1 << 23), (13, None), (14, 32), (17, 0.0), (17, -1.0), (17, float("nan")), (17, float("inf")), (17, 3.0e38),
                 (18, None), (18, A + 2), (19, 60), (20, 3)):
        assert run((i, v)) == 1, (i, v)
    assert run((1, 0), (6, None), (7, None)) == 0 and run((2, 0), (18, None)) == 0


def test_cache_write(L):
    #        type form seqs tokens offsets starts k row head v row head table slots pages kv page d keys values scales stream
    good = [0, 0, 1, 8, A, A, A, 128, 64, A, 128, 64, A, 4, 4, 2, 32, 64, A, A, A, None]
    run = _changed(good, L.sspmm_cache_write)
    for i, v in ((0, 2), (1, 2), (1, -1), (2, -1), (3, -1), (4, None), (5, None), (6, None), (6, A + 4), (7, 127), (7, 56), (8, 1), (9, None), (11, -64), (12, None), (13, -1),
                 (14, 0), (14, (1 << 30) + 1), (15, 0), (15, 65536), (16, 16), (16, 96), (17, 80), (18, None), (18, A + 1), (19, None), (20, None), (20, A + 2)):
        assert run((i, v)) == 1, (i, v)
    assert run((2, 0)) == 0 and run((3, 0)) == 0 and run((13, 0)) == 0


def test_cache_attention(L):
    #        type form seqs queries heads q seq row head table slots lengths pages kv page d keys values scales scale out seq row head workspace bytes stream
    good = [0, 0, 2, 1, 4, A, 256, 256, 64, A, 640, A, 100, 2, 32, 64, A, A, A, 0.125, A, 256, 256, 64, A, 1 << 30, None]
    run = _changed(good, L.sspmm_cache_attention)
    for i, v in ((0, 3), (1, 2), (2, -1), (2, 65536), (3, -1), (3, 1 << 19), (4, 3), (4, 0), (5, None), (5, A + 8), (6, 4), (6, -8), (7, 32), (8, 4), (9, None), (10, 0),
                 (10, 1 << 26), (11, None), (12, 0), (13, 3), (14, 48), (15, 96), (16, None), (17, None), (17, A + 8), (18, None), (19, 0.0), (19, float("inf")), (20, None), (21, 4),
                 (22, 8), (23, 4), (24, None), (24, A + 4), (25, 0)):
        assert run((i, v)) == 1, (i, v)
    assert run((2, 0)) == 0 and run((3, 0)) == 0
    size = L.sspmm_cache_attention_workspace_bytes
    need = size(2, 1, 4, 2, 64, 640, 32)
    assert need > 0 and run((25, need - 1)) == 1
    assert size(2, 1, 3, 2, 64, 64, 32) == 0 and size(0, 1, 4, 2, 64, 64, 32) == 0 and size(2, 1, 4, 2, 65, 64, 32) == 0
    assert size(2, 1, 4, 2, 64, 64, 32) == 0 and size(60000, 1, 4, 2, 64, 640, 32) == 0  # short rows; enough rows for the chip: nothing is split


def test_pages(L):
    many, need, lists = L.sspmm_reserve_pages_workspace_bytes(100000, 40, 800), L.sspmm_fork_pages_workspace_bytes(4, 3), L.sspmm_compact_pages_workspace_bytes(100)
    assert L.sspmm_reserve_pages_workspace_bytes(100, 4, 8) == 0 and many == 4 * (40 + 32000) and need > 0 and lists > 1200
    assert L.sspmm_reserve_pages_workspace_bytes(0, 4, 8) == 0 and L.sspmm_fork_pages_workspace_bytes(4, 0) == 0 and L.sspmm_compact_pages_workspace_bytes(-1) == 0
    # refs pages table rows slots ...
    reserve = _changed([A, 100000, A, 40, 800, A, A, 32, A, many, None], L.sspmm_reserve_pages)
    for i, v in ((0, None), (1, 0), (2, None), (3, -1), (4, -1), (4, 1 << 30), (5, None), (6, None), (7, 0), (8, None), (8, A + 2), (9, many - 1)):
        assert reserve((i, v)) == 1, (i, v)
    release = _changed([A, 100, A, 4, 8, A, A, 2, None], L.sspmm_release_pages)
    for i, v in ((0, None), (1, -1), (2, None), (5, None), (6, None), (7, -1)):
        assert release((i, v)) == 1, (i, v)
    fork = _changed([A, 100, A, 4, 8, A, A, A, 3, 2, 32, 64, A, A, A, A, need, None], L.sspmm_fork_pages)
    for i, v in ((0, None), (2, None), (5, None), (6, None), (7, None), (8, -1), (9, 0), (10, 33), (11, 16), (12, None), (13, A + 1), (14, None), (15, None), (15, A + 1), (16, need - 1)):
        assert fork((i, v)) == 1, (i, v)
    compact = _changed([A, 100, A, 4, 8, 2, 32, 64, A, A, A, A, lists, None], L.sspmm_compact_pages)
    for i, v in ((0, None), (1, 0), (2, None), (5, 0), (6, 0), (7, 33), (8, None), (9, None), (10, None), (11, None), (12, lists - 1)):
        assert compact((i, v)) == 1, (i, v)
    assert reserve((3, 0)) == 0 and release((7, 0)) == 0 and fork((8, 0)) == 0 and compact((4, 0)) == 0


def test_python_entries_want_a_gpu(built_library):
    q, k = torch.zeros(4, 2, 64, dtype=torch.float16), torch.zeros(4, 1, 64, dtype=torch.float16)
    ints = torch.zeros(2, dtype=torch.int32)
    keys, values, scales = sspmm_amd.new_cache(2, 1, 32, 64, device="cpu")
    assert keys.shape == (2, 1, 32, 64) and values.shape == (2, 1, 64, 32) and scales.shape == (2, 2, 1) and keys.dtype is torch.int8
    table = torch.zeros(1, 1, dtype=torch.int32)
    for call in (lambda: sspmm_amd.prompt_attention(q, k, k, ints), lambda: sspmm_amd.cache_write(k, k, ints, ints[:1], table, keys, values, scales),
                 lambda: sspmm_amd.cache_attention(q[None], table, ints[:1], keys, values, scales), lambda: sspmm_amd.reserve_pages(ints, table, ints[:1], ints, 32),
                 lambda: sspmm_amd.release_pages(ints, table, ints[:1], ints), lambda: sspmm_amd.fork_pages(ints, table, ints[:1], ints, ints, keys, values, scales),
                 lambda: sspmm_amd.compact_pages(ints, table, keys, values, scales)):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(TypeError):
        sspmm_amd.new_cache(2, 1, 32, 64, torch.uint8, "cpu")


def test_gradients_are_noticed(built_library):
    """Backward and forward, before anything else is asked of an argument."""
    from torch.autograd import forward_ad
    from sspmm_amd import serving
    t = torch.ones(3)
    serving._no_gradients(t)
    with pytest.raises(RuntimeError, match="gradients"):
        serving._no_gradients(t, t.clone().requires_grad_())
    with forward_ad.dual_level():
        serving._no_gradients(t)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            serving._no_gradients(t, forward_ad.make_dual(t, t))
    with torch.no_grad():
        serving._no_gradients(t.clone().requires_grad_())
