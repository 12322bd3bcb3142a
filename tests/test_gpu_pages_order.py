"""The lists of a fork: what stands where in free_pages, which pages are given out; and calls on large pools."""
import random

import pytest
import torch

import dfattn
import paged_reference as ref

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("requests,children,width,n_pages", [(2, 5, 4, 40), (20, 60, 12, 900), (20, 60, 12, 250), (60, 480, 9, 9000), (60, 480, 9, 500)])
def test_free_pages_after_a_fork(device, requests, children, width, n_pages):
    """Held of the parents, then new as copy_dst has them, then free; each part rising. In one workgroup and in several, with
    pages left and without."""
    page, rng = 16, random.Random(children)
    ids = list(range(n_pages))
    rng.shuffle(ids)
    lens = [rng.randint(1, min(width, n_pages // requests) * page) for _ in range(requests)]
    table = [[ids.pop() if j < -(-n // page) else -1 for j in range(width)] for n in lens]
    parents = [rng.randrange(requests) for _ in range(children)]
    f = dfattn.paged_fork(i32(table), i32(lens), i32(parents), page, n_pages)
    refs, order, start, pairs = f.refs.tolist(), f.free_pages.tolist(), int(f.free_start), int(f.counts[0])
    new = f.copy_dst.tolist()[:pairs]
    assert pairs > 0 and new == sorted(new)
    held = {p for r in parents for p in table[r][:-(-lens[r] // page)]}
    assert order == sorted(held) + new + sorted(set(range(n_pages)) - held - set(new))
    assert start == len(held) + pairs and all(refs[p] > 0 for p in order[:start]) and not any(refs[p] for p in order[start:])
    rows = [row[:-(-n // page)] for row, n in zip(f.block_table.tolist(), f.seq_lens.tolist())]
    assert refs == [sum(p in row for row in rows) for p in range(n_pages)]


def test_large_pools_captured(device):
    """More pages than a call's one allocation takes the workspace for: fork, free and compact, eager and as a graph, on changed
    parents, with the allocator's other tensors written between the replays."""
    page, n_pages, requests, children, width = 16, 140000, 12, 30, 20
    rng = random.Random(3)
    lens = [rng.randint(1, width * page) for _ in range(requests)]
    table = [[rng.randrange(r * 10000, (r + 1) * 10000) for _ in range(width)] for r in range(requests)]
    t, n, parents, ended = i32(table), i32(lens), i32([0] * children), i32([0] * children)

    def step():
        f = dfattn.paged_fork(t, n, parents, page, n_pages)
        c = dfattn.paged_compact(f.block_table, f.seq_lens, page, n_pages, torch.full_like(f.block_table, -1))
        after = f.seq_lens.clone()
        return f, c, after, dfattn.paged_free(f.block_table, after, page, n_pages, ended)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = step()
    for seed in range(3):
        rng = random.Random(seed)
        now, gone = [rng.randrange(-1, requests) for _ in range(children)], [rng.randrange(2) for _ in range(children)]
        parents.copy_(i32(now))
        ended.copy_(i32(gone))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = ref.fork(table, lens, now, page, n_pages)
        for f, c, after, freed in (got, step()):
            torch.full((1 << 20,), -1, dtype=torch.int32, device="cuda")
            rows = [row[:len(w)] for row, w in zip(f.block_table.tolist(), want["rows"])]
            assert rows == want["rows"] and f.seq_lens.tolist() == want["lens"] and f.refs.tolist() == want["refs"]
            assert f.free_pages.tolist() == want["free_pages"] and f.free_start.tolist() == [want["free_start"]]
            dense = ref.compact(rows, want["lens"], page, n_pages)
            assert [row[:len(w)] for row, w in zip(c.block_table.tolist(), dense["rows"])] == dense["rows"]
            assert c.refs.tolist() == dense["refs"] and c.free_start.tolist() == [dense["free_start"]]
            assert list(zip(c.copy_src.tolist(), c.copy_dst.tolist()))[:len(dense["copies"])] == dense["copies"]
            last = ref.free(rows, want["lens"], page, n_pages, gone)
            assert after.tolist() == last["lens"] and [x.tolist() for x in freed] == [last["refs"], last["free_pages"], [last["free_start"]]]


@pytest.mark.parametrize("n_pages,page_bytes", [(70000, 65536), ((1 << 24) - 5, 272), ((1 << 24) - 5, 260), ((1 << 24) - 5, 257)])
def test_copies_past_32_bits(device, n_pages, page_bytes):
    """Pools of more than 2^32 bytes, in pieces of 16 (long and short pages), 4 and 1 bytes: what is copied, and what stays."""
    pool = torch.zeros(n_pages, page_bytes, dtype=torch.int8, device="cuda")
    assert pool.nbytes > 1 << 32
    far = n_pages - 1
    border = (1 << 32) // page_bytes  # the page across 2^32 bytes
    src, dst = [far, 3, border, 7], [0, border + 1, 5, far - 1]
    g = torch.Generator(device="cuda").manual_seed(page_bytes)
    for p in src:
        pool[p] = torch.randint(-128, 128, (page_bytes,), generator=g, device="cuda", dtype=torch.int8)
    want = {p: pool[p].clone() for p in src}
    want.update({d: pool[s].clone() for s, d in zip(src, dst)})
    dfattn.paged_copy([pool], i32(src), i32(dst))
    for p, w in want.items():
        assert torch.equal(pool[p], w), p
        pool[p] = 0
    assert not pool.view(torch.int8).any()
