"""A decoder's steps on an encoder's states, from the prompt to forked rows and drawn tokens: the operators together, as a program uses them."""
import pytest
import torch

import sspmm_amd
from serving_util import attention, check, check_step, offsets_of
from test_sample_gpu import _draw

pytestmark = pytest.mark.gpu

HEADS, KV, D, PAGE, VOCAB, LAYERS = 8, 2, 64, 32, 1009, 2


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Decoder:
    """Two layers of attention to what was said and to the source, and a head; weights small enough that activations keep their size."""

    def __init__(self, seed):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        width = HEADS * D
        make = lambda *shape: torch.randn(shape, generator=g, device="cuda").half() * shape[0] ** -0.5  # noqa: E731
        self.embedding = torch.randn(VOCAB, width, generator=g, device="cuda").half()
        self.qkv = [make(width, width + 2 * KV * D) for _ in range(LAYERS)]
        self.cross_q, self.cross_kv = [make(width, width) for _ in range(LAYERS)], [make(width, 2 * KV * D) for _ in range(LAYERS)]
        self.head = make(width, VOCAB) * 3

    def source(self, states):
        return [(states @ w).view(-1, 2, KV, D).unbind(1) for w in self.cross_kv]

    def split(self, x, layer):
        y = x @ self.qkv[layer]
        n = y.size(0)
        return y[:, :HEADS * D].view(n, HEADS, D), y[:, HEADS * D:(HEADS + KV) * D].view(n, KV, D), y[:, (HEADS + KV) * D:].view(n, KV, D)

    def step(self, tokens, refs, table, lengths, offsets, source, source_offsets, caches, uniform, settings, seen=None):
        """One new token a row: drawn tokens and their probabilities; lengths go on by one."""
        x = self.embedding[tokens.long()]
        sspmm_amd.reserve_pages(refs, table, lengths, offsets, PAGE)
        behind = lengths + 1
        plan = sspmm_amd.plan_prefixes(table, behind, 1, HEADS, KV, PAGE)
        for layer, cache in enumerate(caches):
            q, k, v = self.split(x, layer)
            sspmm_amd.cache_write(k, v, offsets, lengths, table, *cache)
            y = sspmm_amd.prefix_attention(q[:, None], table, plan, *cache)[:, 0]
            if seen is not None:
                check_step(y[:, None], q[:, None], table, behind, *cache, D ** -0.5, "layer %d" % layer)
            x = x + y.reshape(x.shape)
            cq = (x @ self.cross_q[layer]).view(-1, HEADS, D)
            y = sspmm_amd.cross_attention(cq, *source[layer], offsets, source_offsets)
            if seen is not None:
                seen(cq, source[layer], y)
            x = x + y.reshape(x.shape)
        logits = x @ self.head
        drawn, chances = sspmm_amd.sample_tokens(logits, uniform, *settings, probabilities=True)
        lengths.copy_(behind)
        return logits, drawn, chances


@pytest.mark.parametrize("form", [torch.int8, torch.float8_e4m3fn])
def test_prompts_forks_steps_and_draws(built_library, form):
    model, sources, prompts, rows = Decoder(1), [50, 131], [70, 33], 6
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    states = torch.randn(sum(sources), HEADS * D, generator=g, device="cuda").half()
    whole = model.source(states)
    caches = [sspmm_amd.new_cache(64, KV, PAGE, D, form) for _ in range(LAYERS)]
    refs, table = torch.zeros(64, dtype=torch.int32, device="cuda"), torch.full((rows, 8), -1, dtype=torch.int32, device="cuda")
    # ---- the prompts, at rows 0 and 1
    tokens = torch.randint(0, VOCAB, (sum(prompts),), generator=g, device="cuda")
    x, offsets, starts = model.embedding[tokens], offsets_of(prompts + [0] * 4), _ints([0] * rows)
    sspmm_amd.reserve_pages(refs, table, starts, offsets, PAGE)
    for layer, cache in enumerate(caches):
        q, k, v = model.split(x, layer)
        sspmm_amd.cache_write(k, v, offsets, starts, table, *cache)
        x = x + sspmm_amd.prompt_attention(q, k, v, offsets).reshape(x.shape)
        cq = (x @ model.cross_q[layer]).view(-1, HEADS, D)
        y = sspmm_amd.cross_attention(cq, *whole[layer], offsets_of(prompts), offsets_of(sources))
        for h in range(HEADS):
            want, off = attention(cq[70:, h], whole[layer][0][50:, h * KV // HEADS], whole[layer][1][50:, h * KV // HEADS], torch.full((33,), 131, device="cuda"), D ** -0.5, q.dtype, q.dtype)
            check(y[70:, h], want, off, "prompt, layer %d head %d" % (layer, h))
        x = x + y.reshape(x.shape)
    # ---- three continuations of the first, one more of the second; each row draws its own first token from the prompt's last logits
    lengths = _ints(prompts + [0] * 4)
    parents = [0, 1, 0, 0, 1, 0]
    for cache in caches[:1]:
        sspmm_amd.fork_pages(refs, table, lengths, _ints([0, 0, 1, 0]), _ints([2, 3, 4, 5]), *cache)
    # (one table for all layers: the copied last pages of the others)
    for cache in caches[1:]:
        for child in range(2, rows):
            parent, slot = parents[child], prompts[parents[child]] // PAGE
            for pool in cache:
                pool[int(table[child, slot])] = pool[int(table[parent, slot])]
    last = x[torch.tensor([69, 102], device="cuda")] @ model.head
    uniform = torch.rand(rows, generator=g, device="cuda")
    settings = (torch.tensor([0.0, 0.7, 1.0, 1.0, 0.9, 1.3], device="cuda"), _ints([0, 50, 0, 20, 0, 0]), torch.tensor([1.0, 0.9, 0.95, 1.0, 1.0, 0.8], device="cuda"), 0.01)
    tokens = sspmm_amd.sample_tokens(last[parents], uniform, *settings)
    # ---- steps; every row's source is its parent's, copied behind one another
    at = [0, 50, 181]
    order = torch.cat([torch.arange(at[p], at[p + 1]) for p in parents]).cuda()
    source = [(k[order], v[order]) for k, v in whole]
    one, source_offsets = offsets_of([1] * rows), offsets_of([sources[p] for p in parents])

    def seen(cq, kv, y):
        first = 0
        for b, p in enumerate(parents):
            for h in range(HEADS):
                k, v = (t[first:first + sources[p], h * KV // HEADS] for t in kv)
                want, off = attention(cq[b:b + 1, h], k, v, torch.tensor([sources[p]], device="cuda"), D ** -0.5, cq.dtype, cq.dtype)
                check(y[b:b + 1, h], want, off, "row %d head %d" % (b, h))
            first += sources[p]

    for step in range(3):
        uniform = torch.rand(rows, generator=g, device="cuda")
        logits, tokens, chances = model.step(tokens, refs, table, lengths, one, source, source_offsets, caches, uniform, settings, seen)
        host = logits.double().cpu().numpy()
        for i in range(rows):
            t, k, p = (float(s[i]) for s in settings[:3])
            want = _draw(host[i], float(uniform[i]), t, int(k), p, float(torch.tensor(settings[3], dtype=torch.float32)))
            assert (int(tokens[i]), float(chances[i])) == (want[0], pytest.approx(want[1], rel=2e-7)), (step, i)
    assert lengths.tolist() == [prompts[p] + 3 for p in parents]
    # ---- the same captured: a copy of everything goes the eager way beside it
    torch.cuda.synchronize()
    mine = [tokens.clone(), refs.clone(), table.clone(), lengths.clone(), [tuple(t.clone() for t in c) for c in caches], uniform.clone()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = model.step(mine[0], mine[1], mine[2], mine[3], one, source, source_offsets, mine[4], mine[5], settings)
        mine[0].copy_(out[1])
    for step in range(40):
        uniform = torch.rand(rows, generator=g, device="cuda")
        mine[5].copy_(uniform)
        graph.replay()
        logits, tokens, chances = model.step(tokens, refs, table, lengths, one, source, source_offsets, caches, uniform, settings)
        torch.cuda.synchronize()
        assert torch.equal(mine[0], tokens) and torch.equal(out[2], chances), step
        assert torch.equal(mine[2], table) and torch.equal(mine[3], lengths), step
