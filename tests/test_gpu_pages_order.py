"""The lists of a fork: what stands where in free_pages, which pages are given out."""
import random

import pytest
import torch

import dfattn

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
