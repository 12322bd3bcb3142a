"""Generating with the library's serving operators together: a small decoder with 4-bit layers over a paged 8-bit cache, three
beams for each of two prompts. Every step is plan, layers (norm, 4-bit products, append, attention), log probabilities
with alternatives, the choice, fork and the pages' copies.

The oracle keeps no shared pages: at each choice it gives every beam pages of its own and copies all of its parent's
with torch. Everything else is the same calls on the same shapes, so that the results have to be equal bit for bit.
"""
import pytest
import torch

import dfattn
from dfattn import ops, w4

pytestmark = pytest.mark.gpu

D, HEADS, D_HEAD, VOCAB, PAGE, N_PAGES, WIDTH, BEAMS, TOP = 128, 4, 32, 601, 16, 160, 8, 3, 4
PROMPTS = [21, 33]


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Model:
    def __init__(self, layers=2):
        g = torch.Generator(device="cuda").manual_seed(11)
        r = lambda *s: torch.randn(*s, generator=g, device="cuda")
        q = lambda n, k, fmt: w4.quantize(r(n, k) * k ** -0.5, 32, fmt)
        self.embedding, self.ones, self.zeros = r(VOCAB, D), torch.ones(D, device="cuda"), torch.zeros(D, device="cuda")
        self.layers = [dict(qkv=q(3 * D, D, "i4"), out=q(D, D, "u4"), up=q(4 * D, D, "e2m1"), down=q(D, 4 * D, "i4"), bias=0.1 * r(4 * D))
                       for _ in range(layers)]
        self.head = q(VOCAB, D, "i4")

    def caches(self):
        return [dfattn.kv8_cache(N_PAGES, HEADS, D_HEAD, PAGE) for _ in self.layers]

    def norm(self, x):
        return ops.layer_norm_forward(x, self.ones, self.zeros)[0]

    def __call__(self, tokens, caches, slots, table, query_start, seq_lens, most):
        x = self.embedding[tokens.long()]
        for w, cache in zip(self.layers, caches):
            qkv = w4.linear(self.norm(x), w["qkv"])
            dfattn.kv8_append(cache, qkv[:, D:2 * D], qkv[:, 2 * D:], slots)
            a, _ = dfattn.kv8_attention(cache, qkv[:, :D], table, query_start, seq_lens, HEADS, most, WIDTH * PAGE)
            x = w4.linear(a, w["out"], residual=x, out=x)
            h = w4.linear(self.norm(x), w["up"], bias=w["bias"], gelu=True)
            x = w4.linear(h, w["down"], residual=x, out=x)
        return self.norm(x)

    def alternatives(self, x):
        logits = w4.linear(x, self.head)
        _, _, _, ids, top = ops.token_logprobs_forward(logits, torch.zeros(x.shape[0], dtype=torch.int32, device="cuda"), TOP)
        return ids, top


class Shared:
    """The library's fork, copies, free and compaction."""

    def __init__(self, model):
        self.caches = model.caches()
        self.pools = dfattn.page_pools(self.caches)
        self.table = torch.full((2, WIDTH), -1, dtype=torch.int32, device="cuda")
        self.cached = torch.zeros(2, dtype=torch.int32, device="cuda")
        self.clear()

    def clear(self, ended=None):
        _, self.free_pages, self.free_start = dfattn.paged_free(self.table, self.cached, PAGE, N_PAGES, ended)

    def fork(self, parents):
        f = dfattn.paged_fork(self.table, self.cached, parents, PAGE, N_PAGES)
        dfattn.paged_copy(self.pools, f.copy_src, f.copy_dst, f.counts)
        self.table, self.cached, self.free_pages, self.free_start = f.block_table, f.seq_lens, f.free_pages, f.free_start

    def compact(self):
        f = dfattn.paged_compact(self.table, self.cached, PAGE, N_PAGES)
        dfattn.paged_copy(self.pools, f.copy_src, f.copy_dst, f.counts)
        self.free_pages, self.free_start = f.free_pages, f.free_start


class Apart(Shared):
    """Pages of its own for every row, all copied."""

    def fork(self, parents):
        order = torch.randperm(N_PAGES, generator=torch.Generator().manual_seed(int(self.cached.sum()))).tolist()
        table, lens = self.table.tolist(), self.cached.tolist()
        taken = {p for row, n in zip(table, lens) for p in row[:-(-n // PAGE)]}
        order = [p for p in order if p not in taken]
        new, old = [], [t.clone() for c in self.caches for t in c]
        for r in parents.tolist():
            row = [order.pop() for _ in range(-(-lens[r] // PAGE))]
            for a, b in zip(table[r], row):
                for t, u in zip((t for c in self.caches for t in c), old):
                    t.view(torch.int8 if t.dtype != torch.float32 else t.dtype)[b] = u[a]
            new.append(row + [-1] * (WIDTH - len(row)))
        self.table, self.cached = i32(new), i32([lens[r] for r in parents.tolist()])
        self.clear()

    def compact(self):
        pass


def prefill(model, pages):
    tokens = torch.randint(0, VOCAB, (sum(PROMPTS),), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    seq_lens, start, slots, counts = dfattn.paged_plan(pages.cached, i32(PROMPTS), pages.table, pages.free_pages,
                                                       pages.free_start, PAGE, N_PAGES, sum(PROMPTS))
    assert counts.tolist()[:2] == [2, sum(PROMPTS)]
    x = model(tokens, pages.caches, slots, pages.table, start, seq_lens, max(PROMPTS))
    pages.cached = seq_lens
    pages.free_start = counts[2:].clone()
    ids, top = model.alternatives(x[start[1:].long() - 1].contiguous())
    pages.fork(i32([0] * BEAMS + [1] * BEAMS))
    return ids[:, :BEAMS].reshape(-1).contiguous(), top[:, :BEAMS].reshape(-1).clone()  # a beam for each of the first alternatives


def step(model, pages, tokens, scores, one):
    """One token for all beams; (new tokens, scores, parents, the alternatives' log probabilities)."""
    seq_lens, start, slots, counts = dfattn.paged_plan(pages.cached, one, pages.table, pages.free_pages, pages.free_start, PAGE,
                                                       N_PAGES, 2 * BEAMS)
    x = model(tokens, pages.caches, slots, pages.table, start, seq_lens, 1)
    pages.cached = seq_lens
    ids, top = model.alternatives(x)
    total = (scores[:, None] + top).view(2, BEAMS * TOP)
    best, at = torch.sort(total, dim=1, descending=True, stable=True)
    best, at = best[:, :BEAMS], at[:, :BEAMS]
    parents = (at // TOP + BEAMS * torch.arange(2, device="cuda")[:, None]).reshape(-1)
    tokens = ids[parents, (at % TOP).reshape(-1)]
    pages.fork(parents.int())
    return tokens.contiguous(), best.reshape(-1).contiguous(), parents, top


def test_beams(device):
    model = Model()
    a, b = Shared(model), Apart(model)
    one = torch.ones(2 * BEAMS, dtype=torch.int32, device="cuda")
    state = []
    for pages in (a, b):
        state.append(prefill(model, pages))
    assert torch.equal(state[0][0], state[1][0]) and torch.equal(state[0][1], state[1][1])
    shared, unlike = 0, set()
    for n in range(40):
        out = [step(model, pages, *s, one) for pages, s in zip((a, b), state)]
        for x, y in zip(*out):
            assert torch.equal(x, y), n
        state = [o[:2] for o in out]
        unlike.add(tuple(out[0][2].tolist()))
        assert torch.equal(a.cached, b.cached)
        lens = a.cached.tolist()
        held = {p for row, m in zip(a.table.tolist(), lens) for p in row[:-(-m // PAGE)]}
        assert len(held) <= int(a.free_start) <= N_PAGES
        shared = max(shared, sum(-(-m // PAGE) for m in lens) - len(held))
        if n % 13 == 5:
            a.compact()
            assert int(a.free_start) == len(held)
    assert shared >= 4 and len(unlike) > 3  # (pages were shared, and the beams did go on in different ways)
    a.clear(i32([0, 1, 0, 0, 1, 1]))
    assert a.cached.tolist()[1] == 0 and int(a.free_start) < N_PAGES
    a.clear(i32([1] * 6))
    assert int(a.free_start) == 0 and sorted(a.free_pages.tolist()) == list(range(N_PAGES))


def test_step_captured(device):
    """A whole step in a graph, replayed, against the same steps run eagerly."""
    model = Model(1)
    pages = Shared(model)
    one = torch.ones(2 * BEAMS, dtype=torch.int32, device="cuda")
    tokens, scores = prefill(model, pages)
    names = ("table", "cached", "free_pages", "free_start")
    hold = {n: getattr(pages, n).clone() for n in names}
    first = {n: t.clone() for n, t in hold.items()}
    caches = [t.clone() for t in pages.pools.tensors]
    tok, sco = tokens.clone(), scores.clone()

    def once():
        for n in names:
            setattr(pages, n, hold[n])
        t, s, parents, top = step(model, pages, tok, sco, one)
        for n in names:
            hold[n].copy_(getattr(pages, n))
        tok.copy_(t)
        sco.copy_(s)
        return parents, top

    def start_again():
        for n in names:
            hold[n].copy_(first[n])
        for t, c in zip(pages.pools.tensors, caches):
            t.copy_(c)
        tok.copy_(tokens)
        sco.copy_(scores)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        want = []
        for _ in range(20):
            parents, top = once()
            want.append((parents.clone(), top.clone(), tok.clone(), sco.clone(), hold["table"].clone(), hold["free_start"].clone()))
        start_again()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        parents, top = once()
    start_again()
    for n, w in enumerate(want):
        graph.replay()
        torch.cuda.synchronize()
        used = -(-hold["cached"] // PAGE)
        seen = torch.arange(WIDTH, device="cuda")[None, :] < used[:, None]
        got = (parents, top, tok, sco, torch.where(seen, hold["table"], -1), hold["free_start"])
        for x, y in zip(got, w[:4] + (torch.where(seen, w[4], -1), w[5])):
            assert torch.equal(x, y), n
        torch.zeros(1000, device="cuda").sum().item()  # (work of its own between the replays)
