"""Pages of a paged cache between steps (dfattn_paged_fork, _free, _compact, _copy) against plain Python (paged_reference)."""
import random

import pytest
import torch

import dfattn
import paged_reference as ref

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def batch(seed, requests, width, page, n_pages, share=1, odd_ids=False, longer=False):
    """(table, lens) as lists: random lengths (0 and whole pages among them), ids of which groups of `share` rows have some
    in common; all ids may stand behind a row's pages."""
    rng = random.Random(seed)
    ids = list(range(n_pages))
    rng.shuffle(ids)
    lens, table = [], []
    for r in range(requests):
        n = rng.choice((0, 1, page, rng.randint(0, width) * page, rng.randint(0, width * page), rng.randint(0, width * page)))
        lens.append(n + (5 * page if longer and rng.random() < 0.2 else 0))
        row = []
        for j in range(width):
            if r % share and j < min(lens[r - r % share], n) // page // 2:
                row.append(table[r - r % share][j])  # (whole in both)
            elif j < -(-n // page) and ids:
                row.append(ids.pop())
            else:
                row.append(rng.choice((-1, rng.randrange(n_pages), n_pages, 2 ** 31 - 1)))
        if odd_ids and rng.random() < 0.5 and n:
            row[rng.randrange(-(-n // page))] = rng.choice((-1, n_pages, n_pages + 7))
        table.append(row)
    return table, lens


def same_lists(f, want, n_pages):
    assert f.refs.tolist() == want["refs"]
    assert f.free_pages.tolist() == want["free_pages"]
    assert f.free_start.tolist() == [want["free_start"]]
    pairs = want["copies"]
    assert list(zip(f.copy_src.tolist(), f.copy_dst.tolist())) == pairs + [(-1, -1)] * (f.copy_src.numel() - len(pairs))
    assert f.counts.tolist()[0] == len(pairs)


def check_fork(table, lens, parents, page, n_pages, keep=None):
    width = len(table[0])
    want = ref.fork(table, lens, parents, page, n_pages, keep)
    new_table = torch.full((len(parents), width), -7, dtype=torch.int32, device="cuda")
    t, n = i32(table), i32(lens)
    f = dfattn.paged_fork(t, n, i32(parents), page, n_pages, None if keep is None else i32(keep), new_table)
    assert f.seq_lens.tolist() == want["lens"]
    got = f.block_table.tolist()
    assert [row[:len(w)] for row, w in zip(got, want["rows"])] == want["rows"]
    assert all(set(row[len(w):]) <= {-7} for row, w in zip(got, want["rows"]))
    same_lists(f, want, n_pages)
    assert f.counts.tolist()[1] == want["cut"]
    assert t.tolist() == table and n.tolist() == lens
    return f


SIZES = [(1, 1, 1, 1, 1), (3, 2, 16, 9, 4), (8, 12, 16, 120, 8), (20, 40, 20, 900, 60), (5, 300, 32, 1600, 33), (300, 9, 16, 4000, 700),
         (64, 70, 1, 5000, 64), (40, 500, 16, 30000, 90)]


@pytest.mark.parametrize("requests,width,page,n_pages,children", SIZES)
@pytest.mark.parametrize("keep", [False, True])
def test_fork(device, requests, width, page, n_pages, children, keep):
    for seed in range(3):
        rng = random.Random(seed)
        table, lens = batch(seed, requests, width, page, n_pages, share=(1, 3, 4)[seed], odd_ids=seed == 1, longer=seed == 2)
        parents = [rng.choice((rng.randrange(requests), rng.randrange(requests), rng.randrange(min(3, requests)), -1, requests,
                               2 ** 31 - 1)) for _ in range(children)]
        kept = [rng.choice((0, page, rng.randint(0, width * page), 2 ** 31 - 1)) for _ in range(children)]
        check_fork(table, lens, parents, page, n_pages, kept if keep else None)


def test_fork_rules(device):
    """Who keeps a page, who gets a new one: rows 5 5 7 long with pages of 4."""
    table, lens = [[0, 1], [2, 3], [4, 5]], [5, 5, 7]
    f = check_fork(table, lens, [0, 0, 1, 2, 2, 2], 4, 10)
    assert f.block_table.tolist() == [[0, 1], [0, 6], [2, 3], [4, 5], [4, 7], [4, 8]]
    # One child that keeps only part of a page that another has whole must not write into that.
    f = check_fork(table, lens, [2, 2], 4, 10, [3, 7])
    assert f.block_table.tolist()[0][0] == 0 and f.block_table.tolist()[1] == [4, 5]
    # Both keep a part of it: the first one may.
    f = check_fork(table, lens, [2, 2], 4, 10, [3, 2])
    assert [r[0] for r in f.block_table.tolist()] == [4, 0]
    # Two rows of the table have the same page, both cut inside of it.
    check_fork([[0, 1], [0, 2]], [8, 8], [1, 0, 1], 4, 10, [2, 3, 1])
    # No page left for the last two: their lengths fall to whole pages.
    f = check_fork([[0, 1, 2]], [10], [0, 0, 0, 0], 4, 4)
    assert f.seq_lens.tolist() == [10, 10, 8, 8] and f.counts.tolist() == [1, 2] and f.refs.tolist() == [4, 4, 1, 1]
    # The same page twice in a row.
    check_fork([[3, 3]], [6], [0, 0], 4, 5)


def test_fork_many_rows(device):
    """The largest batch, all of one parent, and more pages than one pass of a workgroup."""
    lens = [1000 if r == 77 else 0 for r in range(8192)]
    table = [[3 * j + 1 for j in range(63)] if r == 77 else [-1] * 63 for r in range(8192)]
    check_fork(table, lens, [77] * 8192, 16, 20000)
    check_fork(table, lens, [77] * 8192, 16, 4000)  # (not enough for all)


@pytest.mark.parametrize("requests,width,page,n_pages,_", SIZES)
def test_free(device, requests, width, page, n_pages, _):
    for seed in range(3):
        rng = random.Random(seed)
        table, lens = batch(seed, requests, width, page, n_pages, share=(1, 3, 4)[seed], odd_ids=seed == 1, longer=seed == 2)
        ended = None if seed == 0 else [rng.choice((0, 0, 1, -5)) for _ in range(requests)]
        want = ref.free(table, lens, page, n_pages, ended)
        t, n = i32(table), i32(lens)
        refs, free_pages, free_start = dfattn.paged_free(t, n, page, n_pages, None if ended is None else i32(ended))
        assert n.tolist() == want["lens"] and refs.tolist() == want["refs"]
        assert free_pages.tolist() == want["free_pages"] and free_start.tolist() == [want["free_start"]]
        assert t.tolist() == table


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("requests,width,page,n_pages,_", SIZES)
def test_compact(device, requests, width, page, n_pages, _, in_place):
    for seed in range(3):
        table, lens = batch(seed, requests, width, page, n_pages, share=(1, 3, 4)[seed], odd_ids=seed == 1, longer=seed == 2)
        want = ref.compact(table, lens, page, n_pages)
        t = i32(table)
        new = t if in_place else torch.full_like(t, -7)
        f = dfattn.paged_compact(t, i32(lens), page, n_pages, new)
        for row, w, old in zip(f.block_table.tolist(), want["rows"], table):
            assert row[:len(w)] == w and row[len(w):] == (old[len(w):] if in_place else [-7] * (width - len(w)))
        same_lists(f, want, n_pages)


@pytest.mark.parametrize("n_pages,held", [(1024, 0), (1024, 1024), (1, 0), (1, 1), (2, 1), (1025, 1), (5000, 5000), (200000, 1500)])
def test_all_or_nothing(device, n_pages, held):
    """No page held, all of them, the last one only."""
    table = [list(range(n_pages - held, n_pages)) or [0]]
    lens = [held * 2]
    f = dfattn.paged_compact(i32(table), i32(lens), 2, n_pages, torch.zeros_like(i32(table)))
    want = ref.compact(table, lens, 2, n_pages)
    assert f.block_table.tolist()[0][:held] == want["rows"][0]
    same_lists(f, want, n_pages)
    refs, free_pages, free_start = dfattn.paged_free(i32(table), i32(lens), 2, n_pages)
    want = ref.free(table, lens, 2, n_pages)
    assert (refs.tolist(), free_pages.tolist(), free_start.tolist()) == (want["refs"], want["free_pages"], [held])


def pools_of(seed, n_pages, *shapes):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randint(-128, 128, (n_pages,) + s[:-1], generator=g, device="cuda", dtype=torch.int8) if s[-1] is torch.int8 else
            torch.randn((n_pages,) + s[:-1], generator=g, device="cuda").to(s[-1]) for s in shapes]


@pytest.mark.parametrize("shapes", [
    [(16, 768, torch.int8), (12, torch.float32)], [(20, 7, torch.float32)], [(3, torch.int8), (1, torch.bfloat16), (5, 3, torch.bfloat16)],
    [(16, 64, torch.bfloat16)] * 130, [(1, torch.int8)], [(128, 1024, torch.float32)], [(1500, torch.int8), (4, torch.int8)]])
@pytest.mark.parametrize("count", [None, 0, 1, 13, 40])
def test_copy(device, shapes, count):
    n_pages = 64
    pools = pools_of(3, n_pages, *shapes)
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(7)).tolist()
    src, dst = order[:20], order[20:40]
    src[3] = src[5]              # one page to two
    src[7], dst[11] = -1, n_pages  # left out
    want = [p.clone() for p in pools]
    for m in range(20 if count is None else min(count, 20)):
        if 0 <= src[m] < n_pages and 0 <= dst[m] < n_pages:
            for p in want:
                p[dst[m]] = p[src[m]]
    n = None if count is None else i32([count, 99])
    handle = dfattn.page_pools(pools)
    dfattn.paged_copy(handle if count == 13 else pools, i32(src), i32(dst), n)
    for a, b in zip(pools, want):
        assert torch.equal(a.view(torch.int8), b.view(torch.int8))


def test_copy_unaligned(device):
    """Pools that start between 16 and 4 bytes: their pages move in smaller pieces."""
    for shift, size in ((4, 32), (1, 32), (2, 7), (8, 64)):
        whole = torch.arange(40 * size + 16, device="cuda").to(torch.int8)
        pool = whole[shift:shift + 40 * size].view(40, size)
        want = whole.clone()
        want[shift:shift + 40 * size].view(40, size)[5:7] = want[shift:shift + 40 * size].view(40, size)[30:32]
        dfattn.paged_copy([pool], i32([30, 31]), i32([5, 6]))
        assert torch.equal(whole, want)


def test_copy_caches(device):
    """A fork's children of one prompt read what their parent's cache holds."""
    page, n_pages, heads, d = 16, 40, 3, 40
    caches = [dfattn.kv8_cache(n_pages, heads, d, page, torch.float8_e4m3fn), dfattn.kv8_cache(n_pages, heads, d, page)]
    g = torch.Generator(device="cuda").manual_seed(1)
    lens = [37, 20]
    table, slots = [[3, 8, 1, -1], [5, 0, -1, -1]], []
    for row, n in zip(table, lens):
        slots += [row[t // page] * page + t % page for t in range(n)]
    for c in caches:
        dfattn.kv8_append(c, *(torch.randn(sum(lens), heads * d, generator=g, device="cuda") for _ in "kv"), i32(slots))
    f = dfattn.paged_fork(i32(table), i32(lens), i32([1, 0, 0, 1, 0]), page, n_pages)
    dfattn.paged_copy(caches, f.copy_src, f.copy_dst, f.counts)
    assert f.counts.tolist() == [3, 0]
    rows = f.block_table.tolist()
    for c in caches:
        for row, r in zip(rows, [1, 0, 0, 1, 0]):
            mine = [row[t // page] * page + t % page for t in range(lens[r])]
            theirs = [table[r][t // page] * page + t % page for t in range(lens[r])]
            for a, b in zip(dfattn.kv8_read(c, i32(mine), d), dfattn.kv8_read(c, i32(theirs), d)):
                assert torch.equal(a, b)


def test_captured(device):
    """A fork with its copies and a free, replayed on changed parents."""
    page, n_pages, width = 16, 200, 12
    table, lens = batch(4, 6, width, page, n_pages)
    t, n, parents, new = i32(table), i32(lens), i32([0] * 9), torch.zeros(9, width, dtype=torch.int32, device="cuda")
    pools = pools_of(5, n_pages, (16, 64, torch.bfloat16), (3, torch.float32))
    first = [p.clone() for p in pools]
    handle = dfattn.page_pools(pools)
    stream = torch.cuda.Stream()
    ended = torch.zeros(9, dtype=torch.int32, device="cuda")

    def step():
        f = dfattn.paged_fork(t, n, parents, page, n_pages, new_table=new)
        dfattn.paged_copy(handle, f.copy_src, f.copy_dst, f.counts)
        lens_after = f.seq_lens.clone()
        return f, lens_after, dfattn.paged_free(f.block_table, lens_after, page, n_pages, ended)

    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        f, after, freed = step()
    for seed in range(4):
        rng = random.Random(seed)
        now = [rng.randrange(-1, 6) for _ in range(9)]
        gone = [rng.randrange(2) for _ in range(9)]
        parents.copy_(i32(now))
        ended.copy_(i32(gone))
        for p, q in zip(pools, first):
            p.copy_(q)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = ref.fork(table, lens, now, page, n_pages)
        assert f.seq_lens.tolist() == want["lens"]
        rows = [row[:len(w)] for row, w in zip(f.block_table.tolist(), want["rows"])]
        assert rows == want["rows"]
        same_lists(f, want, n_pages)
        for p, q in zip(pools, first):
            q = q.clone()
            for a, b in want["copies"]:
                q[b] = q[a]
            assert torch.equal(p, q)
        last = ref.free(f.block_table.tolist(), want["lens"], page, n_pages, gone)
        assert after.tolist() == last["lens"] and freed[1].tolist() == last["free_pages"]
        assert freed[2].tolist() == [last["free_start"]]


def test_plan_goes_on(device):
    """paged_plan takes what free and fork leave, on another stream: no page is given out twice."""
    page, n_pages, width = 4, 60, 10
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        table = torch.full((4, width), -1, dtype=torch.int32, device="cuda")
        lens = torch.zeros(4, dtype=torch.int32, device="cuda")
        _, free_pages, free_start = dfattn.paged_free(table, lens, page, n_pages)
        for step, (new, parents) in enumerate([([9, 5, 0, 3], [0, 0, 1, 3]), ([1, 1, 1, 1], [2, 2, 0, 1]), ([1, 4, 2, 1], [0, 1, 2, 2])]):
            lens, _, _, counts = dfattn.paged_plan(lens, i32(new), table, free_pages, free_start, page, n_pages, 40)
            assert counts.tolist()[0] == 4
            held = ref.count([row[:-(-n // page)] for row, n in zip(table.tolist(), lens.tolist())], n_pages)
            f = dfattn.paged_fork(table, lens, i32(parents), page, n_pages)
            table, lens, free_pages, free_start = f.block_table, f.seq_lens, f.free_pages, f.free_start
            # Pages that two rows hold are whole in both.
            rows = [row[:n // page] for row, n in zip(table.tolist(), lens.tolist())]
            open_ = [row[n // page] for row, n in zip(table.tolist(), lens.tolist()) if n % page]
            assert len(set(open_)) == len(open_) and not set(open_) & {p for row in rows for p in row}
            assert sum(held) >= len({p for row in rows for p in row})
    stream.synchronize()


@pytest.mark.parametrize("requests,width,n_pages", [(20, 40, 900), (300, 9, 4000)])
def test_compact_captured(device, requests, width, n_pages):
    """Both forms of the tables' kernels, replayed on other lengths, in place and with the copies."""
    page = 16
    table, _ = batch(11, requests, width, page, n_pages)
    table = [[p if 0 <= p < n_pages else j % n_pages for j, p in enumerate(row)] for row in table]
    t, n = i32(table), torch.zeros(requests, dtype=torch.int32, device="cuda")
    pools = pools_of(6, n_pages, (16, 64, torch.bfloat16))
    first = pools[0].clone()
    stream = torch.cuda.Stream()

    def step():
        c = dfattn.paged_compact(t, n, page, n_pages)
        dfattn.paged_copy(pools, c.copy_src, c.copy_dst, c.counts)
        return c

    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        c = step()
    for seed in range(4):
        rng = random.Random(seed)
        lens = [rng.choice((0, rng.randint(0, width * page))) for _ in range(requests)]
        t.copy_(i32(table))
        n.copy_(i32(lens))
        pools[0].copy_(first)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = ref.compact(table, lens, page, n_pages)
        same_lists(c, want, n_pages)
        assert [row[:len(w)] for row, w in zip(t.tolist(), want["rows"])] == want["rows"]
        moved = first.clone()
        if want["copies"]:
            src, dst = zip(*want["copies"])
            moved[list(dst)] = first[list(src)]
        assert torch.equal(pools[0], moved)


def test_two_streams(device):
    """Calls on two streams at once, of both forms, by the stream argument: each has its own lists."""
    sides = []
    for seed, (requests, width, n_pages) in enumerate([(20, 40, 900), (300, 9, 4000)]):
        table, lens = batch(seed, requests, width, 16, n_pages)
        parents = [random.Random(seed + i).randrange(requests) for i in range(requests)]
        sides.append((torch.cuda.Stream(), table, lens, parents, i32(table), i32(lens), i32(parents), n_pages))
    torch.cuda.synchronize()
    got = [[dfattn.paged_fork(t, n, p, 16, pages, stream=s) for s, _, _, _, t, n, p, pages in sides] for _ in range(20)]
    torch.cuda.synchronize()
    for each in got:
        for f, (_, table, lens, parents, _, _, _, pages) in zip(each, sides):
            want = ref.fork(table, lens, parents, 16, pages)
            assert f.seq_lens.tolist() == want["lens"]
            same_lists(f, want, pages)
