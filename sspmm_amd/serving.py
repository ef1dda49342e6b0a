"""Operators of a decoder that answers: attention over whole prompts of different lengths, and a paged cache in 8 bits that the
tokens after them are written to and read from.  They stand beside the attention of the encoders (`attention.py`, and
`attention_fm` in `layers.py`), which knows sequences of one length and no order; the reference has no counterpart.

    keys, values, scales = new_cache(pages, kv_heads, page_size, head_dim, torch.int8, device)
    out = prompt_attention(q, k, v, offsets)                          # tokens of all prompts one behind the other
    reserve_pages(page_refs, page_table, starts, offsets, page_size)  # pages for the new tokens
    cache_write(k, v, offsets, starts, page_table, keys, values, scales)
    out = cache_attention(q, page_table, lengths, keys, values, scales)  # the newest tokens of every row
    plan = plan_prefixes(page_table, lengths, queries, heads, kv_heads, page_size)  # or, of rows that share pages, once a step
    out = prefix_attention(q, page_table, plan, keys, values, scales)    # and in every layer
    out = cross_attention(q, k, v, offsets, source_offsets)              # on an encoder's states
    tokens = sample_tokens(logits, uniform, temperature, top_k, top_p, min_p)

Lists and tables are int32 tensors on the GPU, read when the kernels run: no call waits for the device, so a step can be captured in a
graph.  What the device alone knows is not checked by the host: entries that name no token, row or page are passed over.
Inference only, as all operators here: inputs that want gradients, backward or forward, are refused.
"""
import functools
import math

import torch

from . import _lib
from .attention import FUSED_HEAD_WIDTHS as HEAD_WIDTHS

_forward_ad = torch.autograd.forward_ad

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


# Calls of a few microseconds: each entry asks for all it wants of its arguments in one expression, and goes through it again, name by name, for the
# error only (prompt_attention 11.3 -> 9.8 us of the host, 4.5 of which are the C call with its launch).

def _ints(name, t, dim, device):
    if t.dtype is not torch.int32 or t.get_device() != device or device < 0 or not t.is_contiguous():
        raise TypeError("%s must be a contiguous int32 tensor on the other arguments' GPU" % name)
    if t.dim() != dim:
        raise ValueError("%s must have %d dimension%s" % (name, dim, "s" if dim > 1 else ""))


def _listed(t, dim, device):
    """Whether t is an int32 list or table as the kernels read it."""
    return t.dtype is torch.int32 and t.get_device() == device and t.dim() == dim and t.is_contiguous()


def _activations(name, t, dim, dtype, device):
    if dtype not in TYPES or t.dtype is not dtype or t.get_device() != device or device < 0:
        raise TypeError("%s must be a float16 or bfloat16 tensor on a GPU, of the same type and on the same GPU as the others" % name)
    if t.dim() != dim:
        raise ValueError("%s must have %d dimensions" % (name, dim))


def _no_gradients(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                raise RuntimeError("an argument wants gradients, and this operator has no backward pass")
    if _forward_ad._current_level >= 0:
        for t in tensors:
            if _forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("an argument carries forward-mode gradients, and this operator has no rule for them")


def _tokens(t):
    """(address, elements from token to token, from head to head, the tensor that has to live as long) of t [tokens, heads, d] as the kernels read it:
    features side by side, 16-byte aligned rows.  What lies otherwise is copied."""
    row, head, one = t.stride()
    at = t.data_ptr()
    if one == 1 and (row | head | at >> 1) & 7 == 0 and t.size(2) <= row < 1 << 23:
        return at, row, head, t
    t = t.contiguous()
    if t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    _, heads, d = t.shape
    return t.data_ptr(), heads * d, d, t


def _queries(t):
    """The same of t [rows, n, heads, d], with the elements from row to row in front."""
    row, token, head, one = t.stride()
    at = t.data_ptr()
    if one == 1 and (row | token | head | at >> 1) & 7 == 0 and t.size(3) <= token < 1 << 23:
        return at, row, token, head, t
    t = t.contiguous()
    if t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    _, n, heads, d = t.shape
    return t.data_ptr(), n * heads * d, heads * d, d, t


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


def _apart(t):
    """Whether t's elements lie at different places."""
    reach = 0
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride <= reach:
            return False
        reach += stride * (size - 1)
    return True


def _out(out, q, places):
    """(out or a new tensor, its places): of q's shape, written where it lies."""
    if out is None:
        out = q.new_empty(q.shape)
        return out, places(out)
    if out.shape != q.shape or out.dtype is not q.dtype or out.get_device() != q.get_device():
        raise ValueError("out must have q's shape and type and lie on its GPU")
    _no_gradients(out)
    at = places(out)
    if at[-1] is not out or not (out.is_contiguous() or _apart(out)):
        raise ValueError("out must have its features side by side in 16-byte aligned rows that do not overlap")
    return out, at


def _cache(keys, values, scales, device):
    """(format, pages, kv_heads, page_size, head_dim)"""
    kind = keys.dtype
    form = CACHE_TYPES.get(kind)
    if (form is not None and values.dtype is kind and scales.dtype is torch.float32 and keys.get_device() == device and values.get_device() == device and
            scales.get_device() == device and keys.dim() == 4 and keys.is_contiguous() and values.is_contiguous() and scales.is_contiguous()):
        pages, kv, page_size, d = keys.shape
        if (page_size in PAGE_SIZES and d in HEAD_WIDTHS and values.shape == (pages, kv, d, page_size) and scales.shape == (pages, 2, kv) and
                (keys.data_ptr() | values.data_ptr()) & 15 == 0 and pages > 0 and kv > 0):
            return form, pages, kv, page_size, d
    if form is None or values.dtype is not kind or scales.dtype is not torch.float32:
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
    raise ValueError("keys, values and scales must be contiguous, and 16-byte aligned")


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(entry, *sizes):
    return getattr(_lib.lib(), entry)(*sizes)


def prompt_attention(q, k, v, offsets, scaling=None, causal=True, out=None):
    """softmax(q k^T * scaling) v for every sequence and head on packed tokens: q [tokens, heads, d], k and v [tokens, kv_heads, d], float16 or
    bfloat16, d = 32, 64 or 128, heads a multiple of kv_heads; sequence b is tokens offsets[b] .. offsets[b + 1] - 1 (int32 on the GPU,
    ascending).  causal: a token sees itself and those before it; otherwise all of its sequence.  Returns [tokens, heads, d]; tokens of no
    sequence are not written, in `out` either.  Views of a fused projection are read where they lie; what lies otherwise than the kernel reads
    (features apart, rows not 16-byte aligned) is copied first.  out may be q, and may not overlap with k and v.  scaling: 1 / sqrt(d) by
    default.  (tokens / 128 + sequences) * heads is below 2^23."""
    dtype, device = q.dtype, q.get_device()
    kind = TYPES.get(dtype)
    if (kind is None or device < 0 or k.dtype is not dtype or v.dtype is not dtype or k.get_device() != device or v.get_device() != device or
            q.dim() != 3 or k.dim() != 3 or v.dim() != 3):
        for name, t in (("q", q), ("k", k), ("v", v)):
            _activations(name, t, 3, dtype, device)
    _no_gradients(q, k, v)
    tokens, heads, d = q.shape
    shape = k.shape
    kv = shape[1]
    if shape != v.shape or shape[0] != tokens or shape[2] != d:
        raise ValueError("k and v must both be [tokens, kv_heads, d] with q's tokens and d")
    _heads(heads, kv, d)
    if not _listed(offsets, 1, device):
        _ints("offsets", offsets, 1, device)
    sequences = offsets.numel() - 1
    if sequences < 0:
        raise ValueError("offsets must hold one value more than there are sequences")
    scale = _scaling(scaling, d)
    out, (to, out_row, out_head, _) = _out(out, q, _tokens)
    if tokens == 0:
        return out
    (q_at, q_row, q_head, q_), (k_at, k_row, k_head, k_), (v_at, v_row, v_head, v_) = _tokens(q), _tokens(k), _tokens(v)
    rc = _lib.call(_lib.lib().sspmm_prompt_attention, q.device, kind, sequences, tokens, heads, kv, d, offsets.data_ptr(), q_at, q_row, q_head, k_at, k_row,
                   k_head, v_at, v_row, v_head, causal, scale, to, out_row, out_head)
    if rc:
        _lib.check(rc, "sspmm_prompt_attention")
    return out


def cross_attention(q, k, v, offsets, source_offsets, scaling=None, out=None):
    """softmax(q k^T * scaling) v of packed queries over packed states of other lengths, a decoder's over its encoder's: q [tokens, heads, d], k and v
    [source_tokens, kv_heads, d]; the queries of sequence b, offsets[b] .. offsets[b + 1] - 1, see all of source_offsets[b] .. source_offsets[b + 1] - 1 and
    nothing else.  Types, head widths, strides, scaling and out as in prompt_attention; single tokens are sequences of one.  A sequence without states is
    zeros; tokens of no sequence are not written.  Work is shared out by the mean length of the sources, which the host knows: one that is many times longer than the mean is faster in a call of its
    own (single tokens, 32 heads on 8 of 128: 65536 states 51 us alone, 798 beside 63 sequences of 100)."""
    dtype, device = q.dtype, q.get_device()
    kind = TYPES.get(dtype)
    if (kind is None or device < 0 or k.dtype is not dtype or v.dtype is not dtype or k.get_device() != device or v.get_device() != device or
            q.dim() != 3 or k.dim() != 3 or v.dim() != 3):
        for name, t in (("q", q), ("k", k), ("v", v)):
            _activations(name, t, 3, dtype, device)
    _no_gradients(q, k, v)
    tokens, heads, d = q.shape
    shape = k.shape
    source_tokens, kv = shape[0], shape[1]
    if shape != v.shape or shape[2] != d:
        raise ValueError("k and v must both be [source_tokens, kv_heads, d] with q's d")
    _heads(heads, kv, d)
    if not (_listed(offsets, 1, device) and _listed(source_offsets, 1, device)):
        _ints("offsets", offsets, 1, device)
        _ints("source_offsets", source_offsets, 1, device)
    sequences = offsets.numel() - 1
    if sequences < 0 or source_offsets.numel() != sequences + 1:
        raise ValueError("offsets and source_offsets must both hold one value more than there are sequences")
    scale = _scaling(scaling, d)
    out, (to, out_row, out_head, _) = _out(out, q, _tokens)
    if tokens == 0:
        return out
    (q_at, q_row, q_head, q_), (k_at, k_row, k_head, k_), (v_at, v_row, v_head, v_) = _tokens(q), _tokens(k), _tokens(v)
    size = _workspace_bytes("sspmm_cross_attention_workspace_bytes", sequences, tokens, source_tokens, heads, kv, d)
    room = offsets.new_empty(size >> 2) if size else None
    rc = _lib.call(_lib.lib().sspmm_cross_attention, q.device, kind, sequences, tokens, source_tokens, heads, kv, d, offsets.data_ptr(), source_offsets.data_ptr(),
                   q_at, q_row, q_head, k_at, k_row, k_head, v_at, v_row, v_head, scale, to, out_row, out_head,
                   None if room is None else room.data_ptr(), size)
    if rc:
        _lib.check(rc, "sspmm_cross_attention")
    return out


def cache_write(k, v, offsets, starts, page_table, keys, values, scales):
    """Tokens offsets[b] .. offsets[b + 1] - 1 of k and v [tokens, kv_heads, d] into the cache, at positions starts[b] on of row b of
    page_table [rows, slots].  The tokens of a page have one scale per head for their keys and one for their values: the largest magnitude
    times 1 / 127 in 32 bits (int8), or the smallest power of two that brings it to 448 or less (e4m3).  Tokens before starts[b] in its page stay, at the
    larger of their scale and the new tokens'; what lies behind the last new token in its page counts as unwritten.  An infinity or NaN makes
    its block's scale NaN, until the page is written from its first position again.  Tokens for which the row has no page are dropped.  No
    two rows of a call may write to one page (fork_pages gives every row its own last page; a row that goes back in front of the position
    where it was forked writes to pages that its relatives read, too)."""
    dtype, device = k.dtype, k.get_device()
    kind = TYPES.get(dtype)
    if kind is None or device < 0 or v.dtype is not dtype or v.get_device() != device or k.dim() != 3 or v.dim() != 3:
        _activations("k", k, 3, dtype, device)
        _activations("v", v, 3, dtype, device)
    _no_gradients(k, v, keys, values, scales)
    form, pages, kv, page_size, d = _cache(keys, values, scales, device)
    tokens = k.size(0)
    if k.shape != (tokens, kv, d) or v.shape != k.shape:
        raise ValueError("k and v must be [tokens, %d, %d] for this cache" % (kv, d))
    if not (_listed(offsets, 1, device) and _listed(starts, 1, device) and _listed(page_table, 2, device)):
        _ints("offsets", offsets, 1, device)
        _ints("starts", starts, 1, device)
        _ints("page_table", page_table, 2, device)
    n = starts.numel()
    rows, slots = page_table.shape
    if offsets.numel() != n + 1 or rows != n:
        raise ValueError("offsets must hold one value more than starts, and page_table a row for each of them")
    if tokens == 0 or n == 0 or slots == 0:
        return
    (k_at, k_row, k_head, k_), (v_at, v_row, v_head, v_) = _tokens(k), _tokens(v)
    rc = _lib.call(_lib.lib().sspmm_cache_write, k.device, kind, form, n, tokens, offsets.data_ptr(), starts.data_ptr(), k_at, k_row, k_head, v_at, v_row,
                   v_head, page_table.data_ptr(), slots, pages, kv, page_size, d, keys.data_ptr(), values.data_ptr(), scales.data_ptr())
    if rc:
        _lib.check(rc, "sspmm_cache_write")


def cache_attention(q, page_table, lengths, keys, values, scales, scaling=None, out=None):
    """Attention of the newest tokens of every row over the cache: q [rows, n, heads, d] are the last n of row b's lengths[b] tokens, whose keys
    and values are in the cache already, and query i sees positions 0 .. lengths[b] - n + i.  Returns [rows, n, heads, d]; a query that sees
    nothing (a row shorter than n, or empty) is zeros.  Positions for which the row has no page are masked.  out may be q.  At most 65535 rows, and
    2^20 of n * heads."""
    dtype, device = q.dtype, q.get_device()
    kind = TYPES.get(dtype)
    if kind is None or device < 0 or q.dim() != 4:
        _activations("q", q, 4, dtype, device)
    _no_gradients(q, keys, values, scales)
    form, pages, kv, page_size, d = _cache(keys, values, scales, device)
    rows, n, heads, dq = q.shape
    if dq != d:
        raise ValueError("q must have the cache's %d features a head" % d)
    _heads(heads, kv, d)
    if not (_listed(page_table, 2, device) and _listed(lengths, 1, device)):
        _ints("page_table", page_table, 2, device)
        _ints("lengths", lengths, 1, device)
    given, slots = page_table.shape
    if given != rows or lengths.numel() != rows:
        raise ValueError("page_table and lengths must have a row for each of q's %d" % rows)
    if slots < 1:
        raise ValueError("page_table must have a slot")
    scale = _scaling(scaling, d)
    out, (to, out_seq, out_row, out_head, _) = _out(out, q, _queries)
    if rows == 0 or n == 0:
        return out
    q_at, q_seq, q_row, q_head, q_ = _queries(q)
    size = _workspace_bytes("sspmm_cache_attention_workspace_bytes", rows, n, heads, kv, d, slots, page_size)
    room = scales.new_empty(size >> 2) if size else None
    rc = _lib.call(_lib.lib().sspmm_cache_attention, q.device, kind, form, rows, n, heads, q_at, q_seq, q_row, q_head, page_table.data_ptr(), slots,
                   lengths.data_ptr(), pages, kv, page_size, d, keys.data_ptr(), values.data_ptr(), scales.data_ptr(), scale, to, out_seq, out_row, out_head,
                   None if room is None else room.data_ptr(), size)
    if rc:
        _lib.check(rc, "sspmm_cache_attention")
    return out


class PrefixPlan:
    """Which rows of a page table share their leading pages, as plan_prefixes found it on the device, for calls of prefix_attention with the sizes it names."""
    __slots__ = ("rows", "slots", "queries", "heads", "kv_heads", "page_size", "data")

    def __init__(self, rows, slots, queries, heads, kv_heads, page_size, data):
        self.rows, self.slots, self.queries, self.heads, self.kv_heads, self.page_size, self.data = rows, slots, queries, heads, kv_heads, page_size, data


def plan_prefixes(page_table, lengths, queries, heads, kv_heads, page_size, plan=None):
    """Which rows of page_table [rows, slots] share leading pages, once a step for the prefix_attention of all layers: a PrefixPlan for `queries` newest tokens of
    every row.  Rows that begin with the same page are compared with the lowest of them; those that share at least the number of pages that saves most
    are a group.  `plan`: one of the same sizes, made anew in place (for a step captured in a graph whose plan is made outside).  At most 1024 rows, 2^20 of
    queries * heads and 2^22 of rows * queries * heads."""
    device = page_table.get_device()
    if device < 0:
        raise TypeError("page_table must be on a GPU")
    if not (_listed(page_table, 2, device) and _listed(lengths, 1, device)):
        _ints("page_table", page_table, 2, device)
        _ints("lengths", lengths, 1, device)
    rows, slots = page_table.shape
    if lengths.numel() != rows:
        raise ValueError("lengths must have a value for every row of page_table")
    if slots < 1 or page_size not in PAGE_SIZES:
        raise ValueError("page_table must have a slot, and pages 32, 64 or 128 tokens")
    size = _workspace_bytes("sspmm_prefix_plan_bytes", rows, queries, heads, kv_heads)
    if size == 0 and rows and queries:
        raise ValueError("a plan is for up to 1024 rows, 2^20 queries * heads and 2^22 rows * queries * heads, heads a multiple of kv_heads")
    if plan is None:
        plan = PrefixPlan(rows, slots, queries, heads, kv_heads, page_size, page_table.new_empty(size >> 2))
    elif ((plan.rows, plan.slots, plan.queries, plan.heads, plan.kv_heads, plan.page_size) != (rows, slots, queries, heads, kv_heads, page_size) or
          not _listed(plan.data, 1, device) or 4 * plan.data.numel() < size):
        raise ValueError("plan is of other sizes, or on another GPU")
    if rows and queries:
        rc = _lib.call(_lib.lib().sspmm_plan_prefixes, page_table.device, page_table.data_ptr(), rows, slots, lengths.data_ptr(), page_size, queries, heads, kv_heads,
                       plan.data.data_ptr(), 4 * plan.data.numel())
        if rc:
            _lib.check(rc, "sspmm_plan_prefixes")
    return plan


def prefix_attention(q, page_table, plan, keys, values, scales, scaling=None, out=None):
    """cache_attention for rows that share leading pages, as fork_pages leaves them: a page that a group of rows shares is read once for all of them.  q
    [rows, n, heads, d], page_table and the cache as there; plan: plan_prefixes of this table and the rows' lengths, which are taken from it."""
    dtype, device = q.dtype, q.get_device()
    kind = TYPES.get(dtype)
    if kind is None or device < 0 or q.dim() != 4:
        _activations("q", q, 4, dtype, device)
    _no_gradients(q, keys, values, scales)
    form, pages, kv, page_size, d = _cache(keys, values, scales, device)
    rows, n, heads, dq = q.shape
    if dq != d:
        raise ValueError("q must have the cache's %d features a head" % d)
    _heads(heads, kv, d)
    if not _listed(page_table, 2, device):
        _ints("page_table", page_table, 2, device)
    if not _listed(plan.data, 1, device):
        _ints("plan's data", plan.data, 1, device)
    slots = page_table.size(1)
    if (plan.rows, plan.slots, plan.queries, plan.heads, plan.kv_heads, plan.page_size) != (rows, slots, n, heads, kv, page_size) or page_table.size(0) != rows:
        raise ValueError("plan is for %d rows of %d slots, %d queries, %d heads on %d, pages of %d" %
                         (plan.rows, plan.slots, plan.queries, plan.heads, plan.kv_heads, plan.page_size))
    scale = _scaling(scaling, d)
    out, (to, out_seq, out_row, out_head, _) = _out(out, q, _queries)
    if rows == 0 or n == 0:
        return out
    q_at, q_seq, q_row, q_head, q_ = _queries(q)
    size = _workspace_bytes("sspmm_prefix_attention_workspace_bytes", rows, n, heads, kv, d)
    room = scales.new_empty(size >> 2)
    rc = _lib.call(_lib.lib().sspmm_prefix_attention, q.device, kind, form, rows, n, heads, q_at, q_seq, q_row, q_head, page_table.data_ptr(), slots,
                   plan.data.data_ptr(), 4 * plan.data.numel(), pages, kv, page_size, d, keys.data_ptr(), values.data_ptr(), scales.data_ptr(), scale, to, out_seq,
                   out_row, out_head, room.data_ptr(), size)
    if rc:
        _lib.check(rc, "sspmm_prefix_attention")
    return out


LOGIT_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
MOST_TOKENS = 1 << 24  # of a vocabulary


def _setting(name, value, dtype, rows, device, fits):
    """(address or None, the value for all rows) of one of sample_tokens' settings."""
    if isinstance(value, torch.Tensor):
        if value.dtype is not dtype or value.get_device() != device or not value.is_contiguous() or value.dim() != 1:
            raise TypeError("%s must be a number, or a contiguous %s tensor of one dimension on the logits' GPU" % (name, str(dtype).split(".")[1]))
        if value.numel() != rows:
            raise ValueError("%s must have a value for each of the %d rows" % (name, rows))
        _no_gradients(value)
        return value.data_ptr(), 0
    if not fits(value):
        raise ValueError("%s cannot be %r" % (name, value))
    return None, value


def sample_tokens(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, probabilities=False):
    """A token of each row of logits [rows, vocab] (float16, bfloat16 or float32), drawn with uniform [rows] (float32, in [0, 1)): int32 [rows].

    With the weights w = exp((l - max l) / temperature), kept are those with w >= min_p; of these the top_k first in the order of falling logits, equal ones by
    rising index; of these the shortest run, at least one, whose weights reach top_p of the sum of all of these.  The token is the first in that order at which
    the running sum of the weights exceeds uniform times their sum.  Each setting is a number or a tensor with one for every row (float32, top_k int32).
    temperature 0: the largest logit, its first index; top_k 0, top_p 1, min_p 0: everything is kept.  What tensors hold, which the host does not look at, is taken to the nearer end:
    temperature, top_k, top_p and min_p below 0 as 0, top_p and min_p above 1 as 1 (a min_p of 1 keeps the largest logits), uniform below 0 as 0, of 1 and above as the last number below; and NaN as
    temperature 0, as what keeps everything, and as uniform 0.  Logits of -infinity, and NaN, are never drawn; of +infinity they share the draw; a row without any other gives -1.
    probabilities: (tokens, float32 [rows] of the probabilities with which they were drawn).

    Weights are whole multiples of 2^-b (vocab * 2^b <= 2^62, b at most 50) of the power of 2^(1/16) nearest to them, so that no order of sums changes a token.  Rows may lie apart, at any element;
    other strides are copied first.  At most 2^24 tokens in a vocabulary, and fewer than 2^22 rows."""
    kind, device = LOGIT_TYPES.get(logits.dtype), logits.get_device()
    if kind is None or device < 0:
        raise TypeError("logits must be a float16, bfloat16 or float32 tensor on a GPU")
    if logits.dim() != 2:
        raise ValueError("logits must be [rows, vocab]")
    _no_gradients(logits, uniform)
    rows, vocab = logits.shape
    if not 1 <= vocab <= MOST_TOKENS:
        raise ValueError("a vocabulary has 1 to 2^24 tokens, got %d" % vocab)
    if uniform.dtype is not torch.float32 or uniform.get_device() != device or not uniform.is_contiguous():
        raise TypeError("uniform must be a contiguous float32 tensor on the logits' GPU")
    if uniform.shape != (rows,):
        raise ValueError("uniform must have a number for each of the %d rows" % rows)
    t_at, t_all = _setting("temperature", temperature, torch.float32, rows, device, lambda x: 0.0 <= x < math.inf)
    k_at, k_all = _setting("top_k", top_k, torch.int32, rows, device, lambda x: 0 <= x < 1 << 31)
    p_at, p_all = _setting("top_p", top_p, torch.float32, rows, device, lambda x: 0.0 <= x <= 1.0)
    m_at, m_all = _setting("min_p", min_p, torch.float32, rows, device, lambda x: 0.0 <= x <= 1.0)
    tokens = torch.empty(rows, dtype=torch.int32, device=logits.device)
    chances = torch.empty(rows, dtype=torch.float32, device=logits.device) if probabilities else None
    if rows:
        if logits.stride(1) != 1 and vocab > 1:
            logits = logits.contiguous()
        size = _workspace_bytes("sspmm_sample_tokens_workspace_bytes", rows, vocab)
        room = uniform.new_empty(size >> 2) if size else None
        rc = _lib.call(_lib.lib().sspmm_sample_tokens, logits.device, kind, rows, vocab, logits.data_ptr(), logits.stride(0), uniform.data_ptr(), t_at, t_all, k_at, k_all,
                       p_at, p_all, m_at, m_all, tokens.data_ptr(), chances.data_ptr() if probabilities else None,
                       None if room is None else room.data_ptr(), size)
        if rc:
            _lib.check(rc, "sspmm_sample_tokens")
    return (tokens, chances) if probabilities else tokens


def _table(page_refs, page_table):
    """(pages, rows, slots, device)"""
    device = page_table.get_device()
    if device < 0 or not (_listed(page_table, 2, device) and _listed(page_refs, 1, device)):
        if device < 0:
            raise TypeError("page_table must be on a GPU")
        _ints("page_table", page_table, 2, device)
        _ints("page_refs", page_refs, 1, device)
    pages = page_refs.numel()
    if pages < 1:
        raise ValueError("page_refs must have a count for every page")
    rows, slots = page_table.shape
    return pages, rows, slots, device


def _room(page_refs, entry, *sizes):
    """(address, bytes, tensor) of a workspace"""
    size = _workspace_bytes(entry, *sizes)
    if size == 0:
        return None, 0, None
    room = page_refs.new_empty(size >> 2)
    return room.data_ptr(), size, room


def reserve_pages(page_refs, page_table, starts, offsets, page_size):
    """Gives a page to every slot of page_table [rows, slots] that begins with one of row b's new tokens, offsets[b + 1] - offsets[b] of them from
    position starts[b] on, and has none (an entry below zero): the lowest free ones, in the order of rows and slots.  page_refs [pages]: how many entries
    name a page, free where that is not positive.  When no page is free the rest stay without, and a slot whose first position was given none stays
    without until the row is released: its tokens are dropped, and masked."""
    pages, rows, slots, device = _table(page_refs, page_table)
    if not (_listed(starts, 1, device) and _listed(offsets, 1, device)):
        _ints("starts", starts, 1, device)
        _ints("offsets", offsets, 1, device)
    if starts.numel() != rows or offsets.numel() != rows + 1:
        raise ValueError("page_table must have a row for each of starts, and offsets one value more")
    if page_size not in PAGE_SIZES:
        raise ValueError("pages have 32, 64 or 128 tokens")
    if rows == 0 or slots == 0:
        return
    room, size, room_ = _room(page_refs, "sspmm_reserve_pages_workspace_bytes", pages, rows, slots)
    rc = _lib.call(_lib.lib().sspmm_reserve_pages, page_table.device, page_refs.data_ptr(), pages, page_table.data_ptr(), rows, slots, starts.data_ptr(),
                   offsets.data_ptr(), page_size, room, size)
    if rc:
        _lib.check(rc, "sspmm_reserve_pages")


def _lengths(lengths, rows, device):
    if not _listed(lengths, 1, device):
        _ints("lengths", lengths, 1, device)
    if lengths.numel() != rows:
        raise ValueError("lengths must have a value for every row of page_table")


def release_pages(page_refs, page_table, lengths, rows):
    """The pages that the rows named in `rows` hold lose a reference each; the rows become empty (entries -1, lengths 0)."""
    pages, all_rows, slots, device = _table(page_refs, page_table)
    _lengths(lengths, all_rows, device)
    if not _listed(rows, 1, device):
        _ints("rows", rows, 1, device)
    count = rows.numel()
    if count == 0 or slots == 0:
        return
    rc = _lib.call(_lib.lib().sspmm_release_pages, page_table.device, page_refs.data_ptr(), pages, page_table.data_ptr(), all_rows, slots, lengths.data_ptr(),
                   rows.data_ptr(), count)
    if rc:
        _lib.check(rc, "sspmm_release_pages")


def _pool_of(pages, keys, values, scales, device):
    _no_gradients(keys, values, scales)
    _, held, kv, page_size, d = _cache(keys, values, scales, device)
    if pages != held:
        raise ValueError("page_refs must have a count for each of the cache's %d pages" % held)
    return kv, page_size, d


def fork_pages(page_refs, page_table, lengths, parents, children, keys, values, scales):
    """Row children[i] becomes a copy of row parents[i]: full pages are shared, a last page that is not full is copied to the lowest one that was free
    before the call, lengths follow, and the pages that the child held lose a reference each.  A child for which no page is free, or
    whose parent is no row, has no page for its last tokens or becomes another's copy in the call, is left empty with length 0: rows do not change
    places in one call, they are copied to rows that are not parents.  A row that is its own parent stays as it is, and may be another's
    parent.  Named twice as a child, a row becomes its last naming."""
    pages, rows, slots, device = _table(page_refs, page_table)
    _lengths(lengths, rows, device)
    if not (_listed(parents, 1, device) and _listed(children, 1, device)):
        _ints("parents", parents, 1, device)
        _ints("children", children, 1, device)
    count = children.numel()
    if parents.numel() != count:
        raise ValueError("parents and children must be of one length")
    kv, page_size, d = _pool_of(pages, keys, values, scales, device)
    if count == 0 or rows == 0 or slots == 0:
        return
    room, size, room_ = _room(page_refs, "sspmm_fork_pages_workspace_bytes", rows, count)
    rc = _lib.call(_lib.lib().sspmm_fork_pages, page_table.device, page_refs.data_ptr(), pages, page_table.data_ptr(), rows, slots, lengths.data_ptr(),
                   parents.data_ptr(), children.data_ptr(), count, kv, page_size, d, keys.data_ptr(), values.data_ptr(), scales.data_ptr(), room, size)
    if rc:
        _lib.check(rc, "sspmm_fork_pages")


def compact_pages(page_refs, page_table, keys, values, scales):
    """With n pages in use, moves the contents of those at n and behind to the free ones below n, and page_table's entries and
    page_refs with them: the pages from n on are free afterwards."""
    pages, rows, slots, device = _table(page_refs, page_table)
    kv, page_size, d = _pool_of(pages, keys, values, scales, device)
    if rows == 0 or slots == 0:
        return
    room, size, room_ = _room(page_refs, "sspmm_compact_pages_workspace_bytes", pages)
    rc = _lib.call(_lib.lib().sspmm_compact_pages, page_table.device, page_refs.data_ptr(), pages, page_table.data_ptr(), rows, slots, kv, page_size, d,
                   keys.data_ptr(), values.data_ptr(), scales.data_ptr(), room, size)
    if rc:
        _lib.check(rc, "sspmm_compact_pages")
