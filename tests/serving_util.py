"""Plain implementations in 64 bits of the serving operators, and how far a right one may be from them."""
import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}  # half a step of the subnormal numbers (bf16's are far below anything here)


def attention(q, k, v, visible, scale, p_type, out_type):
    """One head: (softmax over the first visible[i] keys of q k^T * scale, times v; the largest error of a right kernel), both in 64 bits.

    p rounded to p_type: half a step of each, relative to sum p |v|; scores: products summed in 32 bits, (d + 4) 2^-24 of sum |q| |k|, and
    the exponential's argument and value some 2^-22 and 2^-23 of the largest; the result rounded to out_type; below the normal numbers of fp16 half a
    step of the subnormal ones a key, of values up to max |v| (the largest p is at least one)."""
    q, k, v = q.double(), k.double(), v.double()
    n, d = k.shape
    s = (q @ k.t().contiguous()) * scale
    hidden = torch.arange(n, device=q.device)[None, :] >= visible[:, None]
    s = s.masked_fill(hidden, float("-inf"))
    p = torch.softmax(s, -1).masked_fill(hidden, 0.0)  # (rows without keys: NaN to zeros)
    # (zero times what is masked is zero, whatever it is: sums over the visible part alone)
    finite = torch.isfinite(v)
    out = p @ torch.where(finite, v, 0.0)
    sees = (~hidden).double()
    for what in (float("inf"), float("-inf")):
        out = torch.where(sees @ (v == what).double() > 0, out + what, out)
    out = torch.where(sees @ torch.isnan(v).double() > 0, float("nan"), out)
    a = p @ torch.where(finite, v, 0.0).abs()
    size = (q.abs() @ k.abs().t().contiguous()).masked_fill(hidden, 0.0).amax(-1, keepdim=True) * scale
    e = size * ((d + 4) * 2.0 ** -24 + 2.0 ** -22) + 2.0 ** -21
    most = torch.where(finite, v, 0.0).abs().amax() if n else 0.0
    off = a * (HALF_STEP[p_type] + 2 * e + 2.0 ** -18) + out.abs() * HALF_STEP[out_type] + n * SMALLEST[p_type] * most + SMALLEST[out_type]
    return out, off * 1.01


def check(got, want, off, what=""):
    got = got.double()
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "%s: NaN elsewhere" % (what,)
    rest = ~finite & ~torch.isnan(want)
    assert torch.equal(got[rest], want[rest]), "%s: infinities differ" % (what,)
    far = ((got - want).abs() - off)[finite]
    assert far.numel() == 0 or far.max().item() <= 0, "%s: off by %.3g more than %.3g" % (what, far.max().item(), off[finite].max().item())


def offsets_of(lengths):
    return torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32, device="cuda")


def check_prompt(got, q, k, v, lengths, causal, scale, what=""):
    group, at = q.size(1) // k.size(1), 0
    for n in lengths:
        part = slice(at, at + n)
        visible = torch.arange(1, n + 1, device="cuda") if causal else torch.full((n,), n, device="cuda")
        for h in range(q.size(1) if n else 0):
            want, off = attention(q[part, h], k[part, h // group], v[part, h // group], visible, scale, q.dtype, q.dtype)
            check(got[part, h], want, off, "%s sequence at %d of %d, head %d" % (what, at, n, h))
        at += n


def row_of_cache(table_row, keys, values, scales, n):
    """(k, v) of a row's first n positions in 64 bits, [n, kv_heads, d]."""
    page = keys.size(2)
    held = table_row[:-(-n // page)].long()
    k = keys.view(torch.int8)[held].view(keys.dtype).double() * scales[held, 0].double()[:, :, None, None]
    v = values.view(torch.int8)[held].view(values.dtype).double() * scales[held, 1].double()[:, :, None, None]
    kv, d = keys.size(1), keys.size(3)
    return k.transpose(1, 2).reshape(-1, kv, d)[:n], v.permute(0, 3, 1, 2).reshape(-1, kv, d)[:n]


def check_step(got, q, table, lengths, keys, values, scales, scale, what=""):
    rows, n, heads, d = q.shape
    group = heads // keys.size(1)
    for b in range(rows):
        length = int(lengths[b])
        if length == 0:
            assert not got[b].any(), "%s: row %d is empty" % (what, b)
            continue
        k, v = row_of_cache(table[b], keys, values, scales, length)
        visible = torch.arange(length - n + 1, length + 1, device="cuda")
        for h in range(heads):
            want, off = attention(q[b, :, h], k[:, h // group], v[:, h // group], visible, scale, torch.float16, q.dtype)
            check(got[b, :, h], want, off, "%s row %d of %d, head %d" % (what, b, length, h))


def scale_for(most, dtype):
    """The scale of a block whose largest magnitude is `most` (float32)."""
    if dtype is torch.int8:
        s = most * torch.tensor(1.0 / 127.0, dtype=torch.float32, device=most.device)
    else:
        mantissa, exponent = torch.frexp(most)
        e = (exponent - 9 + (mantissa > 0.875).int()).clamp(min=-126)
        s = torch.where(most == 0, torch.zeros_like(most), torch.ldexp(torch.ones_like(most, dtype=torch.float64), e.double()).float())
    return torch.where(torch.isfinite(most), s, float("nan"))


def codes_for(x, scale, dtype):
    """x / scale in 8 bits, as bytes; scale broadcasts.  Zeros where the scale is zero or NaN."""
    y = torch.where(scale > 0, x.float() / torch.where(scale > 0, scale, 1.0), 0.0)
    return y.round().clamp(-127, 127).to(torch.int8) if dtype is torch.int8 else y.to(torch.float8_e4m3fn).view(torch.int8)


def write(k, v, offsets, starts, table, keys, values, scales):
    """The cache write on host copies, block by block, in place."""
    page, kind = keys.size(2), keys.dtype
    kb, vb = keys.view(torch.int8), values.view(torch.int8)
    for b in range(len(starts)):
        s, n, at = int(starts[b]), int(offsets[b + 1]) - int(offsets[b]), int(offsets[b])
        if n <= 0 or s < 0:
            continue
        for slot in range(s // page, -(-(s + n) // page)):
            if slot >= table.size(1):
                break
            p = int(table[b, slot])
            if not 0 <= p < keys.size(0):
                continue
            low, high = max(s, slot * page), min(s + n, (slot + 1) * page)
            kept, end = low - slot * page, high - slot * page
            for i, (x, pool) in enumerate(((k, kb), (v, vb))):
                new = x[at + low - s:at + high - s].float().transpose(0, 1)  # [kv, tokens, d]
                most = new.abs().amax((1, 2))
                needed = scale_for(most, kind)
                old = scales[p, i].clone()
                now = needed if kept == 0 else torch.where(torch.isnan(old) | torch.isnan(needed), float("nan"), torch.maximum(old, needed))
                block = pool[p] if i == 0 else pool[p].transpose(1, 2)  # [kv, page, d], a view
                if kept:
                    held = block[:, :kept].contiguous().view(kind).float()
                    moved = codes_for(held * old[:, None, None], now[:, None, None], kind)
                    block[:, :kept] = torch.where((now > old)[:, None, None], moved, block[:, :kept])
                block[:, kept:end] = codes_for(new, now[:, None, None], kind)
                scales[p, i] = now
