"""Serving with attention: prompts, and the paged cache in 8 bits that single tokens read, as timing cases.

    own                 False: the plain forms, elementary torch operations; True: the package's operators
    listed()            the named cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what a program holds before the call
    run(state)          one pass
    work(case)          bytes and operations the pass cannot do without
    exact(case, seed)   what run returns, from the definitions in 64 bits

Five kinds of work:

    prompt   attention over whole prompts, packed one behind the other, on views of a fused projection
    write    pages for new tokens, and their keys and values into the cache
    step     attention of the newest tokens of every sequence over the cache
    fork     the children of a step given up, and sequences forked anew
    compact  the pages in use moved to the front of the pool

The cache: keys [pages, kv_heads, page_size, d] and values [pages, kv_heads, d, page_size] in 8 bits (int8 or e4m3), scales
[pages, 2, kv_heads] (keys, values), page_table [rows, slots] (-1: no page), page_refs [pages], how many rows hold a page.
A block (the tokens of a page, one head, keys or values) has one scale: its largest magnitude / 127 for int8, the smallest power of
two that brings it to 448 or less for e4m3.
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
CACHE_TYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def _text(lengths):
    return ",".join(str(n) for n in lengths)


def _lengths(case):
    return [int(n) for n in case["lengths"].split(",")]


def listed():
    return [
        # prompts of a chat service that arrived together: ragged, one of them a single token
        {"name": "prompt_mixed", "kind": "prompt", "lengths": "1811,1,97,2048,640,333,1400,18,1025", "heads": 32, "kv_heads": 8, "d": 128, "type": "bf16",
         "causal": True},
        # one long document
        {"name": "prompt_long", "kind": "prompt", "lengths": "16001", "heads": 8, "kv_heads": 1, "d": 128, "type": "bf16", "causal": True},
        # the encoder layer's attention (12 heads of 64 features, 8 x 512 tokens), both directions
        {"name": "prompt_encoder", "kind": "prompt", "lengths": _text([512] * 8), "heads": 12, "kv_heads": 12, "d": 64, "type": "f16", "causal": False},
        # the smallest call: a few words
        {"name": "prompt_words", "kind": "prompt", "lengths": "5,1,17", "heads": 4, "kv_heads": 2, "d": 64, "type": "f16", "causal": True},
        # keys and values of prompts into the cache, some behind earlier turns
        {"name": "write_prompts", "kind": "write", "lengths": "2048,777,4096,63,1100", "starts": "0,100,0,4095,0", "kv_heads": 8, "d": 128, "page_size": 64,
         "type": "bf16", "cache": "e4m3"},
        # one new token for each of 48 sequences
        {"name": "write_step", "kind": "write", "lengths": _text([1] * 48), "starts": _text([(37 * i * i + 11 * i) % 2000 for i in range(48)]), "kv_heads": 8,
         "d": 64, "page_size": 32, "type": "f16", "cache": "int8"},
        # a decoding step of a full batch, sequences of all ages
        {"name": "step_batch", "kind": "step", "lengths": _text([64 + (797 * i * i + 331 * i) % 4000 for i in range(64)]), "queries": 1, "heads": 32,
         "kv_heads": 8, "d": 128, "page_size": 64, "type": "bf16", "cache": "int8"},
        # one long conversation
        {"name": "step_long", "kind": "step", "lengths": "131009", "queries": 1, "heads": 16, "kv_heads": 4, "d": 128, "page_size": 128, "type": "bf16",
         "cache": "e4m3"},
        # five drafted tokens a sequence, every head with keys of its own, one sequence shorter than the draft
        {"name": "step_drafted", "kind": "step", "lengths": "900,3,257,1500,64,65,1023,311", "queries": 5, "heads": 12, "kv_heads": 12, "d": 64,
         "page_size": 32, "type": "f16", "cache": "int8"},
        # four continuations each of eight sequences
        {"name": "fork_branches", "kind": "fork", "lengths": "1000,77,2047,513,64,900,1,1601", "children": 4, "kv_heads": 8, "d": 128, "page_size": 64,
         "cache": "int8"},
        # a pool of which a quarter lies scattered
        {"name": "compact_pool", "kind": "compact", "pages": 4096, "used": 2500, "moves": 1000, "rows": 64, "kv_heads": 8, "d": 128, "page_size": 64,
         "cache": "int8"},
        # a small pool, a few pages to move
        {"name": "compact_few", "kind": "compact", "pages": 331, "used": 200, "moves": 17, "rows": 9, "kv_heads": 2, "d": 64, "page_size": 32,
         "cache": "e4m3"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _heads(rng):
    kv = rng.choice((1, 2, 3, 4, 8))
    return kv * rng.choice((1, 2, 3, 4, 6, 8)), kv


def draw(rng):
    kind = rng.choice(("prompt", "prompt", "write", "step", "step", "fork", "compact"))
    if kind == "prompt":
        heads, kv = _heads(rng)
        heads, d = min(heads, 32), rng.choice((32, 64, 128))
        heads -= heads % kv
        causal = rng.random() < 0.75
        lengths, left = [], 8.0e11 / (4 * d * heads)
        for _ in range(_log(rng, 1, 24)):
            n = _log(rng, 1, 12000)
            n = max(1, min(n, int(math.sqrt(max(1.0, left / 2)))))
            lengths.append(n)
            left -= n * n
        while len(lengths) * heads * max(lengths) ** 2 > 2.5e9:  # (the plain form holds this many scores)
            lengths[lengths.index(max(lengths))] = max(lengths) // 2 + 1
        return {"kind": kind, "lengths": _text(lengths), "heads": heads, "kv_heads": kv, "d": d, "type": rng.choice(sorted(TYPES)), "causal": causal}
    kv, d, page, cache, kind_of = rng.choice((1, 2, 4, 8)), rng.choice((32, 64, 128)), rng.choice((32, 64, 128)), rng.choice(sorted(CACHE_TYPES)), rng.choice(sorted(TYPES))
    if kind == "write":
        lengths = [_log(rng, 1, rng.choice((1, 4, 2000))) for _ in range(_log(rng, 1, 64))]
        return {"kind": kind, "lengths": _text(lengths), "starts": _text([rng.choice((0, _log(rng, 1, 5000))) for _ in lengths]), "kv_heads": kv, "d": d,
                "page_size": page, "type": kind_of, "cache": cache}
    if kind == "step":
        lengths = [_log(rng, 1, 4096) for _ in range(_log(rng, 2, 64))] if rng.random() < 0.75 else [_log(rng, 4096, 120000)]
        return {"kind": kind, "lengths": _text(lengths), "queries": rng.choice((1, 1, 1, 2, 3, 4, 6, 8)), "heads": kv * rng.choice((1, 2, 3, 4, 8)),
                "kv_heads": kv, "d": d, "page_size": page, "type": kind_of, "cache": cache}
    if kind == "fork":
        return {"kind": kind, "lengths": _text([_log(rng, 1, 3000) for _ in range(_log(rng, 1, 16))]), "children": rng.choice((1, 2, 3, 5)), "kv_heads": kv,
                "d": d, "page_size": page, "cache": cache}
    pages = _log(rng, 40, 4000)
    used = rng.randint(pages // 4, 3 * pages // 4)
    return {"kind": kind, "pages": pages, "used": used, "moves": rng.randint(1, min(used, pages - used) // 2), "rows": _log(rng, 1, 64), "kv_heads": kv,
            "d": d, "page_size": page, "cache": cache}


def work(case):
    kind, d = case["kind"], case["d"]
    if kind == "prompt":
        n = _lengths(case)
        pairs = sum(x * (x + 1) // 2 if case["causal"] else x * x for x in n)
        return {"bytes": 2 * sum(n) * d * 2 * (case["heads"] + case["kv_heads"]), "flops": 4 * d * case["heads"] * pairs}
    kv, page = case["kv_heads"], case["page_size"]
    block = 2 * kv * (page * d + 4)  # bytes of a page with its scales
    if kind == "write":
        n = sum(_lengths(case))
        return {"bytes": n * kv * d * 2 * (2 + 1), "flops": 8 * n * kv * d}
    if kind == "step":
        n, q = _lengths(case), case["queries"]
        seen = sum(max(0, x - i) for x in n for i in range(q))
        return {"bytes": sum(n) * kv * 2 * d + sum(-(-x // page) for x in n) * kv * 8 + 4 * len(n) * q * case["heads"] * d,
                "flops": 4 * d * case["heads"] * seen}
    if kind == "fork":
        n = _lengths(case)
        parts, held = sum(x % page > 0 for x in n), sum(-(-x // page) for x in n)
        return {"bytes": case["children"] * (2 * parts * block + 4 * 5 * held), "flops": case["children"] * 2 * held}
    return {"bytes": case["moves"] * 2 * block + 4 * (case["pages"] + 2 * case["used"]), "flops": case["pages"]}


# ---- what a program has in hand


def _values(g, shape, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda") * scale


def _offsets(lengths):
    return torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32, device="cuda")


def _pool(case, g, pages):
    """(keys, values, scales) of a pool whose tokens have been quantised block by block."""
    kv, d, page = case["kv_heads"], case["d"], case["page_size"]
    parts, scales = [], []
    for shape in ((pages, kv, page, d), (pages, kv, d, page)):
        # (features of different size, as projections leave them)
        by = torch.exp(0.5 * torch.randn((kv, 1, d) if shape[2] == page else (kv, d, 1), generator=g, device="cuda"))
        x = torch.randn(shape, generator=g, device="cuda") * by
        s = _scale_of(x.abs().amax((2, 3)), case["cache"])
        parts.append(_codes(x / s[:, :, None, None], case["cache"]))
        scales.append(s)
    return parts[0], parts[1], torch.stack(scales, 1).contiguous()


def _tables(case, g, held, rows, spare):
    """(page_table, page_refs): row i holds held[i] pages of its own, anywhere in a pool with `spare` pages more."""
    total, slots = sum(held), max(held) + 1
    at = torch.randperm(total + spare, generator=g, device="cuda")[:total].to(torch.int32)
    table = torch.full((rows, slots), -1, dtype=torch.int32, device="cuda")
    first = 0
    for i, n in enumerate(held):
        table[i, :n] = at[first:first + n]
        first += n
    refs = torch.zeros(total + spare, dtype=torch.int32, device="cuda")
    refs[at.long()] = 1
    return table, refs


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind, d = case["kind"], case["d"]
    state = {"case": case}
    if kind == "prompt":
        lengths, heads, kv = _lengths(case), case["heads"], case["kv_heads"]
        qkv = _values(g, (sum(lengths), (heads + 2 * kv) * d))
        qkv[:, :heads * d] *= 1.5
        state |= {"qkv": qkv.to(TYPES[case["type"]]), "offsets": _offsets(lengths), "longest": max(lengths)}
        return state
    page, kv = case["page_size"], case["kv_heads"]
    if kind == "write":
        lengths, starts = _lengths(case), [int(n) for n in case["starts"].split(",")]
        held = [-(-s // page) for s in starts]
        need = sum(-(-(s + n) // page) for s, n in zip(starts, lengths)) - sum(held)
        table, refs = _tables(case, g, held, len(held), need + 9)
        wide = max(-(-(s + n) // page) for s, n in zip(starts, lengths))
        table = torch.nn.functional.pad(table, (0, max(0, wide - table.size(1))), value=-1).contiguous()
        kv_new = _values(g, (sum(lengths), 2 * kv * d)).to(TYPES[case["type"]])
        state |= {"kv": kv_new, "offsets": _offsets(lengths), "starts": torch.tensor(starts, dtype=torch.int32, device="cuda")}
    elif kind == "step":
        lengths, heads = _lengths(case), case["heads"]
        table, refs = _tables(case, g, [-(-n // page) for n in lengths], len(lengths), 5)
        state |= {"q": _values(g, (len(lengths), case["queries"], heads, d), 1.5).to(TYPES[case["type"]]),
                  "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda")}
    elif kind == "fork":
        lengths, times = _lengths(case), case["children"]
        n = len(lengths)
        table, refs = _tables(case, g, [-(-x // page) for x in lengths], n * (1 + times), n * times + 3)
        free = (refs == 0).nonzero().flatten()
        free = free[torch.randperm(free.numel(), generator=g, device="cuda")].to(torch.int32)
        given = torch.tensor(lengths + [0] * (n * times), dtype=torch.int32, device="cuda")
        taken = 0
        for i, x in enumerate(lengths):  # (the children of the step before)
            rows = [n + i * times + j for j in range(times)]
            full, part = x // page, x % page > 0
            for row in rows:
                table[row, :full] = table[i, :full]
                if part:
                    table[row, full] = free[taken]
                    refs[free[taken].long()] = 1
                    taken += 1
                given[row] = x
            refs[table[i, :full].long()] += times
        state |= {"lengths": given, "parents": torch.arange(n, device="cuda", dtype=torch.int32).repeat_interleave(times).contiguous(),
                  "children": torch.arange(n, n * (1 + times), device="cuda", dtype=torch.int32)}
    else:
        pages, used, moves, rows = case["pages"], case["used"], case["moves"], case["rows"]
        low, high = torch.randperm(used, generator=g, device="cuda"), torch.randperm(pages - used, generator=g, device="cuda") + used
        at = torch.cat([low[moves:], high[:moves]])
        at = at[torch.randperm(used, generator=g, device="cuda")].to(torch.int32)
        slots = -(-used // rows) + 1
        flat = torch.full((rows * (slots - 1),), -1, dtype=torch.int32, device="cuda")
        flat[:used] = at
        table = torch.full((rows, slots), -1, dtype=torch.int32, device="cuda")
        table[:, :slots - 1] = flat.view(rows, slots - 1)
        table[rows - 1, slots - 1] = at[0]  # a page that two rows share
        refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        refs.scatter_add_(0, table.flatten().clamp(min=0).long(), (table.flatten() >= 0).int())
        state |= {"handed_table": table.clone(), "handed_refs": refs.clone()}
    keys, values, scales = _pool(case, g, refs.numel())
    return state | {"table": table, "refs": refs, "keys": keys, "values": values, "scales": scales}


# ---- the operators in their plain form


def _scale_of(amax, cache):
    if cache == "int8":
        return amax / 127.0
    mantissa, exponent = torch.frexp(amax)  # mantissa in [0.5, 1): amax = 2 mantissa * 2^(exponent - 1), and 448 = 1.75 * 2^8
    exponent = (exponent - 9 + (mantissa > 0.875).int()).clamp(min=-126)
    return torch.where(amax == 0, torch.zeros_like(amax), ((exponent + 127) << 23).view(torch.float32))


def _codes(x, cache):
    """x, over its scale, in 8 bits."""
    x = torch.nan_to_num(x, nan=0.0)  # 0 / 0, a block of zeros
    return x.round().clamp(-127, 127).to(torch.int8) if cache == "int8" else x.to(torch.float8_e4m3fn)


def _bits(t):
    return t if t.dtype == torch.int8 else t.view(torch.int8)


def _split(state):
    case = state["case"]
    heads, kv, d, qkv = case["heads"], case["kv_heads"], case["d"], state["qkv"]
    n = qkv.size(0)
    return (qkv[:, :heads * d].view(n, heads, d), qkv[:, heads * d:(heads + kv) * d].view(n, kv, d), qkv[:, (heads + kv) * d:].view(n, kv, d))


def _plain_prompt(q, k, v, offsets, longest, causal):
    tokens, heads, d = q.shape
    kv, n = k.size(1), offsets.numel() - 1
    off = offsets.long()
    pos = torch.arange(longest, device=q.device)
    rows = (off[:-1, None] + pos).clamp(max=tokens - 1)  # [n, longest]
    inside = pos < (off[1:] - off[:-1])[:, None]
    Q = q.float()[rows].view(n, longest, kv, heads // kv, d).permute(0, 2, 3, 1, 4).reshape(n, kv, heads // kv * longest, d)
    K = k.float()[rows].permute(0, 2, 3, 1).contiguous()  # [n, kv, d, longest]
    V = v.float()[rows].permute(0, 2, 1, 3).contiguous()
    s = (Q @ K).view(n, kv, heads // kv, longest, longest) * (1.0 / math.sqrt(d))
    mask = inside[:, None, None, None, :]
    if causal:
        mask = mask & (pos[None, :] <= pos[:, None])
    s = s.masked_fill_(~mask, float("-inf"))
    p = s.sub_(s.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(n, kv, heads // kv * longest, longest) @ V).view(n, kv, heads // kv, longest, d) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(n, longest, heads, d)
    token = torch.arange(tokens, device=q.device)
    of = torch.searchsorted(off[1:].contiguous(), token, right=True)
    return out[of, token - off[of]].to(q.dtype)


def _plain_reserve(refs, table, starts, offsets, page):
    first, count = starts.long() // page, (starts + offsets[1:] - offsets[:-1] + page - 1).long() // page
    slot = torch.arange(table.size(1), device=table.device)
    missing = (slot >= first[:, None]) & (slot < count[:, None]) & (table < 0)
    rank = missing.flatten().long().cumsum(0).view_as(table) - 1
    free = refs == 0
    order = torch.argsort((~free).int(), stable=True)
    fits = missing & (rank < free.sum())
    page_of = order[rank.clamp(0, refs.numel() - 1)]
    table.copy_(torch.where(fits, page_of.int(), table))
    refs.scatter_add_(0, torch.where(fits, page_of, 0).flatten(), fits.flatten().int())


def _plain_write(k, v, offsets, starts, table, keys, values, scales, cache):
    page, off = keys.size(2), offsets.long()
    token = torch.arange(k.size(0), device=k.device)
    row = torch.searchsorted(off[1:].contiguous(), token, right=True)
    pos = starts.long()[row] + token - off[row]
    at, slot = table.long()[row, pos // page], pos % page
    # scales: of the new tokens alone where a page begins with them, else no smaller than before
    old_row = starts.long()
    first = table.long().gather(1, (old_row // page).clamp(max=table.size(1) - 1)[:, None])[:, 0]  # the page a row goes on in
    kept = old_row % page
    amax = torch.zeros_like(scales)
    both = torch.stack([k.float().abs().amax(-1), v.float().abs().amax(-1)], 1)  # [tokens, 2, kv]
    amax.scatter_reduce_(0, at[:, None, None].expand_as(both), both, "amax")
    touched = torch.zeros(scales.size(0), dtype=torch.bool, device=k.device).index_fill_(0, at, True)
    goes_on = torch.zeros_like(touched).scatter_(0, first.clamp(min=0), (kept > 0) & (first >= 0) & (off[1:] > off[:-1]))
    before = scales.clone()
    needed = _scale_of(amax, cache)
    scales.copy_(torch.where(touched[:, None, None], torch.where(goes_on[:, None, None], torch.maximum(before, needed), needed), before))
    # the tokens that were there, to the new scale (rows without any: their page as it is)
    f = first.clamp(min=0)
    ratio_old, ratio_new = before[f], scales[f]
    grown = (goes_on[f][:, None] & (ratio_new[:, 0] > ratio_old[:, 0]), goes_on[f][:, None] & (ratio_new[:, 1] > ratio_old[:, 1]))
    s = torch.arange(page, device=k.device)
    old_k, old_v = keys[f], values[f]
    new_k = _codes(old_k.float() * ratio_old[:, 0, :, None, None] / ratio_new[:, 0, :, None, None], cache)
    new_v = _codes(old_v.float() * ratio_old[:, 1, :, None, None] / ratio_new[:, 1, :, None, None], cache)
    mask = s[None, :] < kept[:, None]
    mask_k, mask_v = mask[:, None, :, None] & grown[0][:, :, None, None], mask[:, None, None, :] & grown[1][:, :, None, None]
    _bits(keys)[f] = torch.where(mask_k, _bits(new_k), _bits(old_k))
    _bits(values)[f] = torch.where(mask_v, _bits(new_v), _bits(old_v))
    _bits(keys)[at, :, slot] = _bits(_codes(k.float() / scales[at, 0][:, :, None], cache))
    _bits(values)[at, :, :, slot] = _bits(_codes(v.float() / scales[at, 1][:, :, None], cache))


def _plain_step(q, table, lengths, keys, values, scales):
    n, queries, heads, d = q.shape
    kv, page = keys.size(1), keys.size(2)
    at = table.long().clamp(min=0)
    m = at.size(1) * page
    K = keys.view(torch.int8)[at].view(keys.dtype).float() * scales[at][:, :, 0, :, None, None]  # [n, slots, kv, page, d]
    K = K.permute(0, 2, 4, 1, 3).reshape(n, kv, d, m)
    V = values.view(torch.int8)[at].view(values.dtype).float() * scales[at][:, :, 1, :, None, None]  # [n, slots, kv, d, page]
    V = V.permute(0, 2, 1, 4, 3).reshape(n, kv, m, d)
    g = heads // kv
    Q = q.float().view(n, queries, kv, g, d).permute(0, 2, 1, 3, 4).reshape(n, kv, queries * g, d)
    s = (Q @ K).view(n, kv, queries, g, m) * (1.0 / math.sqrt(d))
    last = lengths.long()[:, None] - queries + torch.arange(queries, device=q.device)  # the newest key that a query sees
    mask = (torch.arange(m, device=q.device) <= last[:, :, None])[:, None, :, None, :]
    s = s.masked_fill(~mask, float("-inf"))
    most = s.amax(-1, keepdim=True)
    p = (s - torch.where(most == float("-inf"), 0.0, most)).exp()
    total = p.sum(-1, keepdim=True)
    out = (p.view(n, kv, queries * g, m) @ V).view(n, kv, queries, g, d)
    out = torch.where(total > 0, out / total, 0.0)
    return out.permute(0, 2, 1, 3, 4).reshape(n, queries, heads, d).to(q.dtype)


def _plain_release(refs, table, lengths, rows):
    rows = rows.long()
    held = table[rows].flatten()
    refs.scatter_add_(0, held.clamp(min=0).long(), -(held >= 0).int())
    table[rows] = -1
    lengths[rows] = 0


def _plain_fork(refs, table, lengths, parents, children, keys, values, scales):
    page = keys.size(2)
    parents, children = parents.long(), children.long()
    length, rows = lengths[parents], table[parents]
    full, part = length.long() // page, length % page > 0
    free = refs == 0
    order = torch.argsort((~free).int(), stable=True)
    rank = part.long().cumsum(0) - 1
    fits = ~part | (rank < free.sum())
    copied = part & fits
    page_of = order[rank.clamp(0, refs.numel() - 1)]
    slot = torch.arange(table.size(1), device=table.device)
    shared = (slot < full[:, None]) & fits[:, None] & (rows >= 0)
    own_page = copied[:, None] & (slot == full[:, None])
    table[children] = torch.where(shared, rows, torch.where(own_page, page_of[:, None].int(), -1))
    lengths[children] = torch.where(fits, length, 0)
    refs.scatter_add_(0, torch.where(shared, rows, 0).flatten().long(), shared.flatten().int())
    refs.scatter_add_(0, torch.where(copied, page_of, 0), copied.int())
    source = rows.long().gather(1, full.clamp(max=table.size(1) - 1)[:, None])[:, 0]
    anything = rows[:, 0].clamp(min=0).long()  # (where nothing is copied, a page onto itself)
    source, target = torch.where(copied, source, anything), torch.where(copied, page_of, anything)
    for pool in (_bits(keys), _bits(values), scales):
        pool[target] = pool[source]


def _plain_compact(refs, table, keys, values, scales):
    used = refs > 0
    index = torch.arange(refs.numel(), device=refs.device)
    boundary = used.sum()
    source, target = (used & (index >= boundary)).nonzero()[:, 0], (~used & (index < boundary)).nonzero()[:, 0]
    for pool in (_bits(keys), _bits(values), scales):
        pool[target] = pool[source]
    refs[target] = refs[source]
    refs[source] = 0
    index[source] = target
    table.copy_(torch.where(table >= 0, index[table.clamp(min=0).long()].int(), table))


def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if kind == "prompt":
        q, k, v = _split(state)
        if own:
            import sspmm_amd
            return sspmm_amd.prompt_attention(q, k, v, state["offsets"], causal=case["causal"])
        return _plain_prompt(q, k, v, state["offsets"], state["longest"], case["causal"])
    table, refs, keys, values, scales = (state[x] for x in ("table", "refs", "keys", "values", "scales"))
    if kind == "step":
        if own:
            import sspmm_amd
            return sspmm_amd.cache_attention(state["q"], table, state["lengths"], keys, values, scales)
        return _plain_step(state["q"], table, state["lengths"], keys, values, scales)
    if kind == "write":
        kv, d, page = case["kv_heads"], case["d"], case["page_size"]
        k, v = state["kv"].view(-1, 2, kv, d).unbind(1)
        if own:
            import sspmm_amd
            sspmm_amd.reserve_pages(refs, table, state["starts"], state["offsets"], page)
            sspmm_amd.cache_write(k, v, state["offsets"], state["starts"], table, keys, values, scales)
        else:
            _plain_reserve(refs, table, state["starts"], state["offsets"], page)
            _plain_write(k, v, state["offsets"], state["starts"], table, keys, values, scales, case["cache"])
        return table, refs, keys, values, scales
    if kind == "fork":
        if own:
            import sspmm_amd
            sspmm_amd.release_pages(refs, table, state["lengths"], state["children"])
            sspmm_amd.fork_pages(refs, table, state["lengths"], state["parents"], state["children"], keys, values, scales)
        else:
            _plain_release(refs, table, state["lengths"], state["children"])
            _plain_fork(refs, table, state["lengths"], state["parents"], state["children"], keys, values, scales)
        return table, refs, state["lengths"], keys, values, scales
    # (tables that the host keeps, handed over)
    table.copy_(state["handed_table"])
    refs.copy_(state["handed_refs"])
    if own:
        import sspmm_amd
        sspmm_amd.compact_pages(refs, table, keys, values, scales)
    else:
        _plain_compact(refs, table, keys, values, scales)
    return table, refs, keys, values, scales


# ---- from the definitions, in 64 bits


def _exact_head(q, k, v, scale, visible):
    """softmax(q k^T scale) v over the first visible[i] keys of each query, in 64 bits."""
    s = torch.mm(q, k.t().contiguous()) * scale
    s[torch.arange(k.size(0), device=q.device)[None, :] >= visible[:, None]] = float("-inf")
    out = torch.mm(torch.softmax(s, -1), v)
    out[visible <= 0] = 0.0
    return out


def exact(case, seed):
    state, kind, d = prepare(case, seed), case["kind"], case["d"]
    if kind == "prompt":
        q, k, v = (t.double() for t in _split(state))
        out, at = torch.empty_like(q), 0
        group = case["heads"] // case["kv_heads"]
        for n in _lengths(case):
            ends = torch.arange(1, n + 1, device=q.device) if case["causal"] else torch.full((n,), n, device=q.device)
            for h in range(case["heads"]):
                part = slice(at, at + n)
                out[part, h] = _exact_head(q[part, h], k[part, h // group], v[part, h // group], d ** -0.5, ends)
            at += n
        return out
    keys, values, scales, table = state["keys"], state["values"], state["scales"], state["table"]
    page, kv = case["page_size"], case["kv_heads"]
    if kind == "step":
        lengths, queries, heads = _lengths(case), case["queries"], case["heads"]
        q, group = state["q"].double(), heads // kv
        out = torch.zeros_like(q)
        for b, n in enumerate(lengths):
            held = table[b, :-(-n // page)].long()
            for h in range(kv):
                K = (keys.view(torch.int8)[held, h].view(keys.dtype).double() * scales[held, 0, h].double()[:, None, None]).reshape(-1, d)[:n]
                V = (values.view(torch.int8)[held, h].view(values.dtype).double() * scales[held, 1, h].double()[:, None, None]).transpose(1, 2).reshape(-1, d)[:n]
                ends = torch.arange(n - queries + 1, n + 1, device=q.device).repeat_interleave(group)
                rows = q[b, :, h * group:(h + 1) * group].reshape(queries * group, d)
                out[b, :, h * group:(h + 1) * group] = _exact_head(rows, K, V, d ** -0.5, ends).view(queries, group, d)
        return out
    if kind != "write":
        return None  # pages are moved as they are
    # (int8: the codes are whole numbers of steps, which the scales' own rounding may move by one)
    lengths, starts, kind_of = _lengths(case), [int(n) for n in case["starts"].split(",")], case["cache"]
    free = [i for i, r in enumerate(state["refs"].tolist()) if r == 0]
    rows, at = table.tolist(), 0
    scale, codes = scales.double(), [keys.double(), values.double().transpose(2, 3).contiguous()]  # [pages, kv, page, d]
    new = state["kv"].double().view(-1, 2, kv, d)
    for b, (s, n) in enumerate(zip(starts, lengths)):
        for slot in range(s // page, -(-(s + n) // page)):
            if rows[b][slot] < 0:
                rows[b][slot] = free.pop(0)
            p, low, high = rows[b][slot], max(s, slot * page), min(s + n, (slot + 1) * page)
            x, kept, end = new[at + low - s:at + high - s], low - slot * page, high - slot * page
            most = x.abs().amax((0, 3))  # [2, kv]
            needed = most / 127 if kind_of == "int8" else torch.where(most > 0, torch.exp2(torch.ceil(torch.log2(most / 448))), most)
            now = torch.maximum(scale[p], needed) if kept else needed
            for i in range(2):
                over = torch.where(now[i] > 0, now[i], 1.0)[:, None, None]
                if kind_of == "e4m3":  # (quotients by powers of two: exact, in 32 bits too)
                    codes[i][p, :, :kept] = (codes[i][p, :, :kept] * scale[p, i][:, None, None] / over).float().to(torch.float8_e4m3fn).double()
                    codes[i][p, :, kept:end] = (x[:, i].transpose(0, 1) / over).float().to(torch.float8_e4m3fn).double()
            scale[p] = now
        at += n
    if kind_of == "int8":
        return None, None, None, None, scale
    return None, None, codes[0], codes[1].transpose(2, 3).contiguous(), scale
