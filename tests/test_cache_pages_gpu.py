"""Pages of the cache against a model of them in Python, and the serving operators together as a decoder runs them."""
import random

import pytest
import torch

import sspmm_amd
from serving_util import attention, check, check_prompt, check_step, offsets_of, row_of_cache

pytestmark = pytest.mark.gpu


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Model:
    """What the operators should do, with the pool's contents as one number a page."""

    def __init__(self, pages, rows, slots, page):
        self.refs, self.table, self.lengths, self.page = [0] * pages, [[-1] * slots for _ in range(rows)], [0] * rows, page
        self.pool = list(range(pages))

    def _take(self):
        for p, r in enumerate(self.refs):
            if r <= 0:
                self.refs[p] = 1
                return p
        return -1

    def reserve(self, starts, counts):
        for b, (s, n) in enumerate(zip(starts, counts)):
            if n <= 0 or s < 0:
                continue
            for slot in range(s // self.page, min(len(self.table[b]), -(-(s + n) // self.page))):
                if self.table[b][slot] < 0:
                    self.table[b][slot] = self._take()

    def release(self, rows):
        for b in rows:
            if 0 <= b < len(self.table):
                for p in self.table[b]:
                    if 0 <= p < len(self.refs):
                        self.refs[p] -= 1
                self.table[b] = [-1] * len(self.table[b])
                self.lengths[b] = 0

    def fork(self, parents, children):
        last = {c: i for i, c in enumerate(children) if 0 <= c < len(self.table)}
        plans = []
        for i, (p, c) in enumerate(zip(parents, children)):
            if last.get(c) != i:
                continue
            plan = None
            if 0 <= p < len(self.table) and p not in last:
                n = max(0, min(self.lengths[p], len(self.table[p]) * self.page))
                full, part = n // self.page, n % self.page > 0
                source = self.table[p][full] if part else None
                if not part or 0 <= source < len(self.refs):
                    target = self._take() if part else None
                    if target != -1:
                        plan = (p, n, full, source, target)
            plans.append((c, plan))
        for c, plan in plans:
            self.table[c], self.lengths[c] = [-1] * len(self.table[c]), 0
            if plan is not None:
                p, n, full, source, target = plan
                self.lengths[c] = n
                for s in range(full):
                    page = self.table[p][s]
                    if 0 <= page < len(self.refs):
                        self.table[c][s] = page
                        self.refs[page] += 1
                if source is not None:
                    self.table[c][full] = target
                    self.pool[target] = self.pool[source]

    def compact(self):
        n = sum(r > 0 for r in self.refs)
        holes = [p for p in range(n) if self.refs[p] <= 0]
        movers = [p for p in range(n, len(self.refs)) if self.refs[p] > 0]
        to = dict(zip(movers, holes))
        for a, b in to.items():
            self.pool[b], self.refs[b], self.refs[a] = self.pool[a], self.refs[a], 0
        self.table = [[to.get(p, p) for p in row] for row in self.table]


class Device:
    def __init__(self, pages, rows, slots, page, kv=2, d=32):
        self.page = page
        self.refs, self.lengths = _ints([0] * pages), _ints([0] * rows)
        self.table = torch.full((rows, slots), -1, dtype=torch.int32, device="cuda")
        self.cache = sspmm_amd.new_cache(pages, kv, page, d)
        self.marks = torch.arange(pages, device="cuda")
        for pool in self.cache[:2]:  # every byte of page p: p, by two of its digits in turn
            flat = pool.view(pages, -1)
            flat[:, 0::2] = (self.marks % 127).to(torch.int8)[:, None]
            flat[:, 1::2] = (self.marks // 127 % 127).to(torch.int8)[:, None]
        self.cache[2][:] = self.marks[:, None, None].float()

    def contents(self, pages):
        """Which page's contents each page has; all parts of it have to say so."""
        got = self.cache[2][pages, 0, 0].long()
        assert (self.cache[2][pages] == got[:, None, None]).all()
        for pool in self.cache[:2]:
            flat = pool.view(pool.size(0), -1)[pages]
            assert (flat[:, 0::2].long() == (got % 127)[:, None]).all() and (flat[:, 1::2].long() == (got // 127 % 127)[:, None]).all()
        return got.tolist()

    def same(self, model, what):
        assert self.refs.tolist() == model.refs, what
        assert self.table.tolist() == model.table, what
        assert self.lengths.tolist() == model.lengths, what
        used = [p for p, r in enumerate(model.refs) if r > 0]
        if used:
            assert self.contents(torch.tensor(used, device="cuda")) == [model.pool[p] for p in used], what


@pytest.mark.parametrize("pages,rows,slots,page", [(60, 6, 9, 32), (300, 40, 12, 64), (9000, 30, 400, 32), (5, 3, 4, 128), (4097, 70, 70, 32)])
@pytest.mark.parametrize("seed", [1, 2, 3])
def test_runs_of_calls(built_library, pages, rows, slots, page, seed):
    r = random.Random(100 * seed + pages)
    model, dev = Model(pages, rows, slots, page), Device(pages, rows, slots, page)
    for step in range(25):
        kind = r.choice(("grow", "grow", "grow", "release", "fork", "compact"))
        print(pages, seed, step, kind, flush=True)
        if kind == "grow":
            counts = [r.choice((0, 1, 1, r.randint(1, 3 * page))) if r.random() < 0.7 else 0 for _ in range(rows)]
            counts = [min(n, slots * page - l) for n, l in zip(counts, model.lengths)]
            model.reserve(model.lengths, counts)
            sspmm_amd.reserve_pages(dev.refs, dev.table, dev.lengths, offsets_of(counts), page)
            model.lengths = [l + n for l, n in zip(model.lengths, counts)]
            dev.lengths += _ints(counts)
        elif kind == "release":
            named = [r.randrange(-2, rows + 2) for _ in range(r.randint(0, 4))]
            model.release(named)
            sspmm_amd.release_pages(dev.refs, dev.table, dev.lengths, _ints(named))
        elif kind == "fork":
            empty = [b for b in range(rows) if model.lengths[b] == 0 and max(model.table[b]) < 0]
            children = [r.choice(empty + [-1, rows]) for _ in range(r.randint(0, 6))] if empty else []
            parents = [r.randrange(-1, rows + 1) for _ in children]
            model.fork(parents, children)
            sspmm_amd.fork_pages(dev.refs, dev.table, dev.lengths, _ints(parents), _ints(children), *dev.cache)
        else:
            model.compact()
            sspmm_amd.compact_pages(dev.refs, dev.table, *dev.cache)
        dev.same(model, "step %d, %s" % (step, kind))


def test_running_out_of_pages(built_library):
    model, dev = Model(5, 4, 6, 32), Device(5, 4, 6, 32)
    for starts, counts in (([0, 0, 0, 0], [40, 0, 33, 0]), ([40, 0, 33, 0], [60, 70, 0, 1])):
        model.reserve(starts, counts)
        sspmm_amd.reserve_pages(dev.refs, dev.table, _ints(starts), offsets_of(counts), 32)
        dev.same(model, counts)
    assert (dev.refs == 1).all() and (dev.table[1] < 0).all()  # what row 1 and 3 wanted was not there
    model.lengths = [100, 0, 33, 0]
    dev.lengths.copy_(_ints(model.lengths))
    model.fork([2, 0], [1, 3])
    sspmm_amd.fork_pages(dev.refs, dev.table, dev.lengths, _ints([2, 0]), _ints([1, 3]), *dev.cache)
    dev.same(model, "fork")
    assert dev.lengths.tolist() == [100, 0, 33, 0]


def test_every_page_of_a_large_pool_and_none(built_library):
    for pages in (1, 4096, 8192, 12289, 16385, 20480):
        model, dev = Model(pages, 3, pages + 1, 32), Device(pages, 3, pages + 1, 32, kv=1)
        model.compact()
        sspmm_amd.compact_pages(dev.refs, dev.table, *dev.cache)
        dev.same(model, "empty")
        counts = [0, 32 * (pages // 2), 32 * (pages - pages // 2)]
        model.reserve([0, 0, 0], counts)
        sspmm_amd.reserve_pages(dev.refs, dev.table, _ints([0, 0, 0]), offsets_of(counts), 32)
        model.compact()
        sspmm_amd.compact_pages(dev.refs, dev.table, *dev.cache)
        dev.same(model, "full")
        model.release([1])
        sspmm_amd.release_pages(dev.refs, dev.table, dev.lengths, _ints([1, 1]))
        model.compact()
        sspmm_amd.compact_pages(dev.refs, dev.table, *dev.cache)
        dev.same(model, "half")


def test_captured_and_replayed(built_library):
    """A step's calls in one graph: children given up, forked anew, pages for the next tokens, the pool compacted."""
    page, rows, slots, pages = 32, 8, 6, 64
    dev = Device(pages, rows, slots, page)
    counts = [70, 33, 64, 1, 0, 0, 0, 0]
    sspmm_amd.reserve_pages(dev.refs, dev.table, dev.lengths, offsets_of(counts), page)
    dev.lengths += _ints(counts)
    parents, children, more = _ints([0, 1, 3, 0]), _ints([4, 5, 6, 7]), offsets_of([40, 1, 1, 1, 1, 1, 31, 2])

    def step():
        sspmm_amd.release_pages(dev.refs, dev.table, dev.lengths, children)
        sspmm_amd.fork_pages(dev.refs, dev.table, dev.lengths, parents, children, *dev.cache)
        sspmm_amd.reserve_pages(dev.refs, dev.table, dev.lengths, more, page)
        sspmm_amd.compact_pages(dev.refs, dev.table, *dev.cache)

    state = [dev.refs, dev.table, dev.lengths, *dev.cache]
    start = [t.clone() for t in state]
    step()
    torch.cuda.synchronize()
    for t, s in zip(state, start):
        t.copy_(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for turn in range(4):
        for t, s in zip(state, start):
            t.copy_(s)
        parents.copy_(_ints([turn % 4, 1, 3, 0]))
        step()
        torch.cuda.synchronize()
        want = [t.clone() for t in state]
        for t, s in zip(state, start):
            t.copy_(s)
        g.replay()
        torch.cuda.synchronize()
        for name, t, w in zip(("refs", "table", "lengths", "keys", "values", "scales"), state, want):
            assert torch.equal(t, w), (turn, name)


@pytest.mark.parametrize("form", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_together_as_a_decoder_runs_them(built_library, dtype, form):
    """Prompts, their keys and values into the cache, drafted and single tokens on forks of them, a compaction in between; every attention against the
    formula on what the cache holds, and what it holds against what went in."""
    heads, kv, d, page, pages, rows = 8, 2, 64, 32, 60, 6
    g = torch.Generator(device="cuda")
    g.manual_seed(21)
    cache = sspmm_amd.new_cache(pages, kv, page, d, form)
    refs, table = _ints([0] * pages), torch.full((rows, 8), -1, dtype=torch.int32, device="cuda")
    lengths, held = _ints([0] * rows), [torch.zeros(0, 2, kv, d, device="cuda", dtype=dtype) for _ in range(rows)]

    def tokens(counts):
        x = torch.randn(sum(counts), (heads + 2 * kv) * d, generator=g, device="cuda").to(dtype)
        q, k, v = x[:, :heads * d].view(-1, heads, d), x[:, heads * d:(heads + kv) * d].view(-1, kv, d), x[:, (heads + kv) * d:].view(-1, kv, d)
        at = 0
        for b, n in enumerate(counts):
            held[b] = torch.cat([held[b], torch.stack([k[at:at + n], v[at:at + n]], 1)])
            at += n
        return q, k, v

    def put(k, v, counts):
        sspmm_amd.reserve_pages(refs, table, lengths, offsets_of(counts), page)
        sspmm_amd.cache_write(k, v, offsets_of(counts), lengths, table, *cache)
        lengths.add_(_ints(counts))

    counts = [70, 33, 1, 0, 0, 0]
    q, k, v = tokens(counts)
    check_prompt(sspmm_amd.prompt_attention(q, k, v, offsets_of(counts)), q, k, v, counts, True, d ** -0.5)
    put(k, v, counts)
    sspmm_amd.fork_pages(refs, table, lengths, _ints([0, 0, 1]), _ints([3, 4, 5]), *cache)
    for child, parent in ((3, 0), (4, 0), (5, 1)):
        held[child] = held[parent]
    for step, n in enumerate((1, 3, 1, 1, 5, 1)):
        counts = [n] * rows
        q, k, v = tokens(counts)
        put(k, v, counts)
        got = sspmm_amd.cache_attention(q.view(rows, n, heads, d), table, lengths, *cache)
        check_step(got, q.view(rows, n, heads, d), table, lengths.tolist(), *cache, d ** -0.5, "step %d" % step)
        if step == 2:
            sspmm_amd.release_pages(refs, table, lengths, _ints([0]))
            held[0] = held[0][:0]
            sspmm_amd.compact_pages(refs, table, *cache)
            used = int((refs > 0).sum())
            assert (refs[:used] > 0).all() and int(table.max()) < used
    assert lengths.tolist() == [len(h) for h in held]
    for b in range(rows):
        n = int(lengths[b])
        for i, got in enumerate(row_of_cache(table[b], *cache, n)):
            s = cache[2][table[b, :-(-n // page)].long(), i].double().repeat_interleave(page, 0)[:n, :, None]
            x = held[b][:, i].double()
            # int8: half a step, and half a step for each time the page's scale grew (at most once a call); e4m3: 2^-4, or half the smallest
            # steps of all the scales it had, each at most half of the next
            near = s * 0.5 * 8 if form is torch.int8 else x.abs() * 2.0 ** -4 + s * 2.0 ** -9
            assert ((got - x).abs() <= near).all(), (b, i)


def test_refusals(built_library):
    dev = Device(10, 3, 4, 32)
    t, refs, n, cache = dev.table, dev.refs, dev.lengths, dev.cache
    one, off = _ints([0]), offsets_of([1, 1, 1])
    for call, kind in ((lambda: sspmm_amd.reserve_pages(refs.long(), t, n, off, 32), TypeError), (lambda: sspmm_amd.reserve_pages(refs, t.cpu(), n, off, 32), TypeError),
                       (lambda: sspmm_amd.reserve_pages(refs, t, n, off, 48), ValueError), (lambda: sspmm_amd.reserve_pages(refs, t, n[:2], off, 32), ValueError),
                       (lambda: sspmm_amd.reserve_pages(refs, t, n, off[:3], 32), ValueError), (lambda: sspmm_amd.reserve_pages(refs, t.t(), n, off, 32), TypeError),
                       (lambda: sspmm_amd.reserve_pages(refs[:0], t, n, off, 32), ValueError), (lambda: sspmm_amd.release_pages(refs, t, n[:1], one), ValueError),
                       (lambda: sspmm_amd.release_pages(refs, t, n, one.cpu()), TypeError), (lambda: sspmm_amd.fork_pages(refs, t, n, one, _ints([1, 2]), *cache), ValueError),
                       (lambda: sspmm_amd.fork_pages(refs[:9].clone(), t, n, one, one, *cache), ValueError),
                       (lambda: sspmm_amd.compact_pages(refs[:9].clone(), t, *cache), ValueError), (lambda: sspmm_amd.compact_pages(refs, t[0], *cache), ValueError),
                       (lambda: sspmm_amd.compact_pages(refs, t, cache[0].float(), *cache[1:]), TypeError)):
        with pytest.raises(kind):
            call()
    before = [x.clone() for x in (t, refs, n)]
    none = _ints([])
    sspmm_amd.release_pages(refs, t, n, none)
    sspmm_amd.fork_pages(refs, t, n, none, none, *cache)
    sspmm_amd.reserve_pages(refs, t[:0], none, offsets_of([]), 32)
    assert all(torch.equal(a, b) for a, b in zip((t, refs, n), before))


@pytest.mark.parametrize("seed", [1, 2, 3, 4])
def test_beams_that_take_the_places_of_others(built_library, seed):
    """Children that hold pages give them back, whatever becomes of them; rows that are their own parents stay, and are parents of others."""
    r = random.Random(seed)
    pages, rows, slots, page = 160, 12, 8, 32
    model, dev = Model(pages, rows, slots, page), Device(pages, rows, slots, page)
    counts = [r.randint(0, slots * page) for _ in range(rows)]
    model.reserve([0] * rows, counts)
    sspmm_amd.reserve_pages(dev.refs, dev.table, dev.lengths, offsets_of(counts), page)
    model.lengths = counts
    dev.lengths.copy_(_ints(counts))
    for step in range(12):
        children = [r.randrange(-1, rows) for _ in range(r.randint(1, rows))]
        parents = [c if r.random() < 0.3 else r.randrange(-1, rows) for c in children]
        last = {c: i for i, c in enumerate(children) if c >= 0}
        moved = [c for c, i in last.items() if parents[i] != c]
        before = [list(model.table[c]) for c in moved]
        pairs = sorted((last[c], c) for c in moved)
        model.fork([parents[i] for i, _ in pairs], [c for _, c in pairs])
        for row in before:
            for p in row:
                if p >= 0:
                    model.refs[p] -= 1
        sspmm_amd.fork_pages(dev.refs, dev.table, dev.lengths, _ints(parents), _ints(children), *dev.cache)
        dev.same(model, "seed %d, step %d: %s of %s" % (seed, step, children, parents))
        held = [p for row in model.table for p in row if p >= 0]
        assert model.refs == [held.count(p) for p in range(pages)]



@pytest.mark.parametrize("form", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("old", [100.0, float("nan")])
def test_a_page_that_was_missing_is_not_entered_in_the_middle(built_library, form, old):
    """A row whose tokens found no free page goes on when another row's pages are free again: the positions that were dropped stay masked, nothing of the other row's
    keys, values and scales is read or kept."""
    page, kv, heads, d, pages = 32, 2, 4, 64, 3
    g = torch.Generator(device="cuda")
    g.manual_seed(41)
    cache = sspmm_amd.new_cache(pages, kv, page, d, form)
    refs, table, lengths = _ints([0] * pages), torch.full((3, 4), -1, dtype=torch.int32, device="cuda"), _ints([0, 0, 0])

    def put(counts, size=1.0):
        x = (torch.randn(sum(counts), 2, kv, d, generator=g, device="cuda") * size).half()
        sspmm_amd.reserve_pages(refs, table, lengths, offsets_of(counts), page)
        sspmm_amd.cache_write(x[:, 0], x[:, 1], offsets_of(counts), lengths, table, *cache)
        lengths.add_(_ints(counts))
        return x

    def step(n):
        q = torch.randn(3, n, heads, d, generator=g, device="cuda").half()
        return q, sspmm_amd.cache_attention(q, table, lengths, *cache)

    put([40, 20, 0], old if old == old else 1.0)
    if old != old:
        cache[2][table[0, :2].long()] = old
    put([0, 0, 10])  # there is no page for these
    assert refs.tolist() == [1, 1, 1] and (table[2] < 0).all()
    sspmm_amd.release_pages(refs, table, lengths, _ints([0]))
    put([0, 0, 5])  # positions 10 .. 14: their page has lost its front
    assert (table[2] < 0).all() and refs.tolist() == [0, 0, 1]
    assert not step(1)[1][2].any()
    x = put([0, 0, 30])  # 15 .. 44: of these, 32 .. 44 lie in a page that begins with them
    assert table[2].tolist() == [-1, 0, -1, -1] and refs.tolist() == [1, 0, 1]
    k, v = row_of_cache(table[2, 1:], *cache, 13)
    for i, got in enumerate((k, v)):
        s = cache[2][0, i].double()[None, :, None]
        want = x[17:, i].double()
        assert ((got - want).abs() <= (s * 0.5 if form is torch.int8 else want.abs() * 2.0 ** -4 + s * 2.0 ** -10) * 1.001).all()
    q, got = step(2)
    for h in range(heads):
        visible = torch.tensor([12, 13], device="cuda")
        check(got[2, :, h], *attention(q[2, :, h], k[:, h // 2], v[:, h // 2], visible, 0.125, torch.float16, torch.float16))


def test_a_fork_of_a_row_longer_than_its_table(built_library):
    """The child's tokens behind the table count as the parent's do: the newest queries of either see the same positions."""
    page, d, n = 32, 64, 4
    cache = sspmm_amd.new_cache(4, 1, page, d)
    refs, table, lengths = _ints([0] * 4), torch.full((3, 2), -1, dtype=torch.int32, device="cuda"), _ints([0, 0, -7])
    g = torch.Generator(device="cuda")
    g.manual_seed(43)
    x = torch.randn(66, 2, 1, d, generator=g, device="cuda").half()
    off = offsets_of([66, 0, 0])
    sspmm_amd.reserve_pages(refs, table, lengths.clamp(min=0), off, page)
    sspmm_amd.cache_write(x[:, 0], x[:, 1], off, lengths, table, *cache)
    lengths += off.diff()
    sspmm_amd.fork_pages(refs, table, lengths, _ints([0, 2]), _ints([1, 2]), *cache)
    assert lengths.tolist() == [66, 66, -7] and refs.tolist() == [2, 2, 0, 0] and table[1].tolist() == table[0].tolist()
    q = torch.randn(1, n, 2, d, generator=g, device="cuda").half().expand(3, n, 2, d)
    got = sspmm_amd.cache_attention(q, table, lengths, *cache)
    assert torch.equal(got[0], got[1]) and not got[2].any()
    k, v = row_of_cache(table[0], *cache, 64)
    for h in range(2):
        visible = torch.tensor([63, 64, 64, 64], device="cuda")
        check(got[1, :, h], *attention(q[1, :, h], k[:, 0], v[:, 0], visible, 0.125, torch.float16, torch.float16))
