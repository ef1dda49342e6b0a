"""Operators of a decoder that answers: attention over whole prompts of different lengths, and a paged cache in 8 bits that the
tokens after them are written to and read from.  They stand beside the attention of the encoders (`attention.py`, and
`attention_fm` in `layers.py`), which knows sequences of one length and no order; the reference has no counterpart.

    keys, values, scales = new_cache(pages, kv_heads, page_size, head_dim, torch.int8, device)
    out = prompt_attention(q, k, v, offsets)                          # tokens of all prompts one behind the other
    reserve_pages(page_refs, page_table, starts, offsets, page_size)  # pages for the new tokens
    cache_write(k, v, offsets, starts, page_table, keys, values, scales)
    out = cache_attention(q, page_table, lengths, keys, values, scales)  # the newest tokens of every row

Lists and tables are int32 tensors on the GPU, read when the kernels run: no call waits for the device, so a step can be captured in a
graph.  What the device alone knows is not checked by the host: entries that name no token, row or page are passed over.
Inference only, as all operators here: inputs that want gradients are refused.
"""
import math

import torch

from . import _lib
from .attention import FUSED_HEAD_WIDTHS as HEAD_WIDTHS

TYPES = {torch.float16: 0, torch.bfloat16: 1}
CACHE_TYPES = {torch.int8: 0, torch.float8_e4m3fn: 1}
PAGE_SIZES = (32, 64, 128)


def new_cache(pages, kv_heads, page_size, head_dim, dtype=torch.int8, device="cuda"):
    """(keys, values, scales) of a cache of zeros: [pages, kv_heads, page_size, head_dim] and [pages, kv_heads, head_dim, page_size] of
    `dtype` (torch.int8 or torch.float8_e4m3fn), float32 [pages, 2, kv_heads].  An element is its code times its block's scale."""
    if dtype not in CACHE_TYPES:
        raise TypeError("a cache holds torch.int8 or torch.float8_e4m3fn, got %s" % (dtype,))
    if page_size not in PAGE_SIZES or head_dim not in HEAD_WIDTHS:
        raise ValueError("pages have 32, 64 or 128 tokens and heads 32, 64 or 128 features")
    return (torch.zeros(pages, kv_heads, page_size, head_dim, dtype=dtype, device=device),
            torch.zeros(pages, kv_heads, head_dim, page_size, dtype=dtype, device=device),
            torch.zeros(pages, 2, kv_heads, dtype=torch.float32, device=device))


def _ints(name, t, dim, device):
    if t.dtype is not torch.int32 or t.get_device() != device or not t.is_contiguous():
        raise TypeError("%s must be a contiguous int32 tensor on the other arguments' GPU" % name)
    if t.dim() != dim:
        raise ValueError("%s must have %d dimension%s" % (name, dim, "s" if dim > 1 else ""))


def _activations(name, t, dim, dtype, device):
    if dtype not in TYPES or t.dtype is not dtype or t.get_device() != device or device < 0:
        raise TypeError("%s must be a float16 or bfloat16 tensor on a GPU, of the same type and on the same GPU as the others" % name)
    if t.dim() != dim:
        raise ValueError("%s must have %d dimensions" % (name, dim))
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("%s wants gradients, and this operator has no backward pass" % name)


def _rows(t, token):
    """t as the kernels read it: features side by side, 16-byte aligned rows; one that lies otherwise is copied.  token: the dimension of the tokens."""
    s = t.stride()
    d = t.size(-1)
    if s[-1] == 1 and t.data_ptr() % 16 == 0 and d <= s[token] < 1 << 23:
        for x in s[:-1]:
            if x % 8:
                break
        else:
            return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _scaling(scaling, d):
    if scaling is None:
        return 1.0 / math.sqrt(d)
    if not 0.0 < scaling <= 2.0e38:
        raise ValueError("scaling must be positive and finite")
    return float(scaling)


def _heads(heads, kv_heads, d):
    if d not in HEAD_WIDTHS:
        raise ValueError("heads have 32, 64 or 128 features, got %d" % d)
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError("the heads of q (%d) must be a multiple of those of keys and values (%d)" % (heads, kv_heads))


def _out(out, q):
    if out is None:
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if out.shape != q.shape or out.dtype is not q.dtype or out.get_device() != q.get_device():
        raise ValueError("out must have q's shape and type and lie on its GPU")
    if out.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("out wants gradients, and this operator has no backward pass")
    if _rows(out, 1 if out.dim() == 4 else 0) is not out:
        raise ValueError("out must have its features side by side in 16-byte aligned rows")
    return out


def _cache(keys, values, scales, device):
    """(format, pages, kv_heads, page_size, head_dim)"""
    form = CACHE_TYPES.get(keys.dtype)
    if form is None or values.dtype is not keys.dtype or scales.dtype is not torch.float32:
        raise TypeError("keys and values must be torch.int8 or torch.float8_e4m3fn, the same, and scales float32")
    if not (keys.get_device() == values.get_device() == scales.get_device() == device):
        raise TypeError("keys, values and scales must be on the other arguments' GPU")
    if keys.dim() != 4:
        raise ValueError("keys must be [pages, kv_heads, page_size, head_dim]")
    pages, kv, page_size, d = keys.shape
    if values.shape != (pages, kv, d, page_size) or scales.shape != (pages, 2, kv):
        raise ValueError("keys %s want values [pages, kv_heads, head_dim, page_size] and scales [pages, 2, kv_heads]" % (tuple(keys.shape),))
    if page_size not in PAGE_SIZES or d not in HEAD_WIDTHS or pages < 1 or kv < 1:
        raise ValueError("a cache has pages of 32, 64 or 128 tokens and heads of 32, 64 or 128 features")
    if not (keys.is_contiguous() and values.is_contiguous() and scales.is_contiguous()) or keys.data_ptr() % 16 or values.data_ptr() % 16:
        raise ValueError("keys, values and scales must be contiguous, and 16-byte aligned")
    return form, pages, kv, page_size, d


def prompt_attention(q, k, v, offsets, scaling=None, causal=True, out=None):
    """softmax(q k^T * scaling) v for every sequence and head on packed tokens: q [tokens, heads, d], k and v [tokens, kv_heads, d], float16 or
    bfloat16, d = 32, 64 or 128, heads a multiple of kv_heads; sequence b is tokens offsets[b] .. offsets[b + 1] - 1 (int32 on the GPU,
    ascending).  causal: a token sees itself and those before it; otherwise all of its sequence.  Returns [tokens, heads, d]; tokens of no
    sequence are not written, in `out` either.  Views of a fused projection are read where they lie; what lies otherwise than the kernel reads
    (features apart, rows not 16-byte aligned) is copied first.  scaling: 1 / sqrt(d) by default."""
    device = q.get_device()
    for name, t in (("q", q), ("k", k), ("v", v)):
        _activations(name, t, 3, q.dtype, device)
    tokens, heads, d = q.shape
    kv = k.size(1)
    if k.shape != v.shape or k.size(0) != tokens or k.size(2) != d:
        raise ValueError("k and v must both be [tokens, kv_heads, d] with q's tokens and d")
    _heads(heads, kv, d)
    _ints("offsets", offsets, 1, device)
    if offsets.numel() < 1:
        raise ValueError("offsets must hold one value more than there are sequences")
    scale = _scaling(scaling, d)
    out = _out(out, q)
    if tokens == 0:
        return out
    q, k, v = _rows(q, 0), _rows(k, 0), _rows(v, 0)
    sq, sk, sv, so = q.stride(), k.stride(), v.stride(), out.stride()
    rc = _lib.call(_lib.lib().sspmm_prompt_attention, q.device, TYPES[q.dtype], offsets.numel() - 1, tokens, heads, kv, d, offsets.data_ptr(),
                   q.data_ptr(), sq[0], sq[1], k.data_ptr(), sk[0], sk[1], v.data_ptr(), sv[0], sv[1], causal, scale, out.data_ptr(), so[0], so[1])
    _lib.check(rc, "sspmm_prompt_attention")
    return out


def cache_write(k, v, offsets, starts, page_table, keys, values, scales):
    """Tokens offsets[b] .. offsets[b + 1] - 1 of k and v [tokens, kv_heads, d] into the cache, at positions starts[b] on of row b of
    page_table [rows, slots].  The tokens of a page have one scale per head for their keys and one for their values: the largest magnitude
    / 127 (int8), or the smallest power of two that brings it to 448 or less (e4m3).  Tokens before starts[b] in its page stay, at the
    larger of their scale and the new tokens'; what lies behind the last new token in its page counts as unwritten.  An infinity or NaN makes
    its block's scale NaN, until the page is written from its first position again.  Tokens for which the row has no page are dropped.  No
    two rows of a call may write to one page (fork_pages gives every row its own last page)."""
    device = k.get_device()
    _activations("k", k, 3, k.dtype, device)
    _activations("v", v, 3, k.dtype, device)
    form, pages, kv, page_size, d = _cache(keys, values, scales, device)
    tokens = k.size(0)
    if k.shape != (tokens, kv, d) or v.shape != k.shape:
        raise ValueError("k and v must be [tokens, %d, %d] for this cache" % (kv, d))
    _ints("offsets", offsets, 1, device)
    _ints("starts", starts, 1, device)
    _ints("page_table", page_table, 2, device)
    n = starts.numel()
    if offsets.numel() != n + 1 or page_table.size(0) != n:
        raise ValueError("offsets must hold one value more than starts, and page_table a row for each of them")
    if tokens == 0 or n == 0 or page_table.size(1) == 0:
        return
    k, v = _rows(k, 0), _rows(v, 0)
    sk, sv = k.stride(), v.stride()
    rc = _lib.call(_lib.lib().sspmm_cache_write, k.device, TYPES[k.dtype], form, n, tokens, offsets.data_ptr(), starts.data_ptr(), k.data_ptr(), sk[0], sk[1],
                   v.data_ptr(), sv[0], sv[1], page_table.data_ptr(), page_table.size(1), pages, kv, page_size, d, keys.data_ptr(), values.data_ptr(),
                   scales.data_ptr())
    _lib.check(rc, "sspmm_cache_write")


def cache_attention(q, page_table, lengths, keys, values, scales, scaling=None, out=None):
    """Attention of the newest tokens of every row over the cache: q [rows, n, heads, d] are the last n of row b's lengths[b] tokens, whose keys
    and values are in the cache already, and query i sees positions 0 .. lengths[b] - n + i.  Returns [rows, n, heads, d]; a query that sees
    nothing (a row shorter than n, or empty) is zeros.  Positions for which the row has no page are masked."""
    device = q.get_device()
    _activations("q", q, 4, q.dtype, device)
    form, pages, kv, page_size, d = _cache(keys, values, scales, device)
    rows, n, heads, dq = q.shape
    if dq != d:
        raise ValueError("q must have the cache's %d features a head" % d)
    _heads(heads, kv, d)
    _ints("page_table", page_table, 2, device)
    _ints("lengths", lengths, 1, device)
    if page_table.size(0) != rows or lengths.numel() != rows:
        raise ValueError("page_table and lengths must have a row for each of q's %d" % rows)
    slots = page_table.size(1)
    if slots < 1:
        raise ValueError("page_table must have a slot")
    scale = _scaling(scaling, d)
    out = _out(out, q)
    if rows == 0 or n == 0:
        return out
    q = _rows(q, 1)
    sq, so = q.stride(), out.stride()
    L = _lib.lib()
    size = L.sspmm_cache_attention_workspace_bytes(rows, n, heads, kv, d, slots, page_size)
    room = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
    rc = _lib.call(L.sspmm_cache_attention, q.device, TYPES[q.dtype], form, rows, n, heads, q.data_ptr(), sq[0], sq[1], sq[2], page_table.data_ptr(), slots,
                   lengths.data_ptr(), pages, kv, page_size, d, keys.data_ptr(), values.data_ptr(), scales.data_ptr(), scale, out.data_ptr(), so[0], so[1],
                   so[2], None if room is None else room.data_ptr(), size)
    _lib.check(rc, "sspmm_cache_attention")
    return out


def _table(page_refs, page_table):
    """(pages, rows, slots, device)"""
    device = page_table.get_device()
    if device < 0:
        raise TypeError("page_table must be on a GPU")
    _ints("page_table", page_table, 2, device)
    _ints("page_refs", page_refs, 1, device)
    if page_refs.numel() < 1:
        raise ValueError("page_refs must have a count for every page")
    return page_refs.numel(), page_table.size(0), page_table.size(1), device


def _workspace(pages, rows, slots, count, like):
    size = _lib.lib().sspmm_page_workspace_bytes(pages, rows, slots, count)
    return torch.empty(size, dtype=torch.uint8, device=like.device), size


def reserve_pages(page_refs, page_table, starts, offsets, page_size):
    """Gives a page to every slot of page_table [rows, slots] that is to hold row b's new tokens, offsets[b + 1] - offsets[b] of them from
    position starts[b] on, and has none (an entry below zero): the lowest free ones, in the order of rows and slots.  page_refs [pages]: how many entries
    name a page, free where that is not positive.  When no page is free the rest stay without."""
    pages, rows, slots, device = _table(page_refs, page_table)
    _ints("starts", starts, 1, device)
    _ints("offsets", offsets, 1, device)
    if starts.numel() != rows or offsets.numel() != rows + 1:
        raise ValueError("page_table must have a row for each of starts, and offsets one value more")
    if page_size not in PAGE_SIZES:
        raise ValueError("pages have 32, 64 or 128 tokens")
    if rows == 0 or slots == 0:
        return
    room, size = _workspace(pages, rows, slots, 0, page_table)
    rc = _lib.call(_lib.lib().sspmm_reserve_pages, page_table.device, page_refs.data_ptr(), pages, page_table.data_ptr(), rows, slots, starts.data_ptr(),
                   offsets.data_ptr(), page_size, room.data_ptr(), size)
    _lib.check(rc, "sspmm_reserve_pages")


def _lengths(lengths, rows, device):
    _ints("lengths", lengths, 1, device)
    if lengths.numel() != rows:
        raise ValueError("lengths must have a value for every row of page_table")


def release_pages(page_refs, page_table, lengths, rows):
    """The pages that the rows named in `rows` hold lose a reference each; the rows become empty (entries -1, lengths 0)."""
    pages, all_rows, slots, device = _table(page_refs, page_table)
    _lengths(lengths, all_rows, device)
    _ints("rows", rows, 1, device)
    if rows.numel() == 0 or slots == 0:
        return
    rc = _lib.call(_lib.lib().sspmm_release_pages, page_table.device, page_refs.data_ptr(), pages, page_table.data_ptr(), all_rows, slots, lengths.data_ptr(),
                   rows.data_ptr(), rows.numel())
    _lib.check(rc, "sspmm_release_pages")


def _pool_of(page_refs, keys, values, scales, device):
    _, pages, kv, page_size, d = _cache(keys, values, scales, device)
    if page_refs.numel() != pages:
        raise ValueError("page_refs must have a count for each of the cache's %d pages" % pages)
    return kv, page_size, d


def fork_pages(page_refs, page_table, lengths, parents, children, keys, values, scales):
    """Row children[i], which holds no pages, becomes a copy of row parents[i]: full pages are shared, a last page that is not full is copied to the
    lowest free one, lengths follow.  A child for which no page is free, or whose parent is itself a child in the call, is left empty
    with length 0.  Named twice as a child, a row becomes its last naming."""
    pages, rows, slots, device = _table(page_refs, page_table)
    _lengths(lengths, rows, device)
    _ints("parents", parents, 1, device)
    _ints("children", children, 1, device)
    if parents.numel() != children.numel():
        raise ValueError("parents and children must be of one length")
    kv, page_size, d = _pool_of(page_refs, keys, values, scales, device)
    count = children.numel()
    if count == 0 or rows == 0 or slots == 0:
        return
    room, size = _workspace(pages, rows, slots, count, page_table)
    rc = _lib.call(_lib.lib().sspmm_fork_pages, page_table.device, page_refs.data_ptr(), pages, page_table.data_ptr(), rows, slots, lengths.data_ptr(),
                   parents.data_ptr(), children.data_ptr(), count, kv, page_size, d, keys.data_ptr(), values.data_ptr(), scales.data_ptr(), room.data_ptr(), size)
    _lib.check(rc, "sspmm_fork_pages")


def compact_pages(page_refs, page_table, keys, values, scales):
    """With n pages in use, moves the contents of those at n and behind to the free ones below n, and page_table's entries and
    page_refs with them: the pages from n on are free afterwards."""
    pages, rows, slots, device = _table(page_refs, page_table)
    kv, page_size, d = _pool_of(page_refs, keys, values, scales, device)
    if rows == 0 or slots == 0:
        return
    room, size = _workspace(pages, rows, slots, 0, page_table)
    rc = _lib.call(_lib.lib().sspmm_compact_pages, page_table.device, page_refs.data_ptr(), pages, page_table.data_ptr(), rows, slots, kv, page_size, d,
                   keys.data_ptr(), values.data_ptr(), scales.data_ptr(), room.data_ptr(), size)
    _lib.check(rc, "sspmm_compact_pages")
