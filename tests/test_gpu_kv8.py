"""The paged 8-bit cache on the GPU: tables and slot maps, append, read-back and attention against their float64
definitions (kv8_reference.py), and a run of them together."""
import ctypes
import math

import numpy as np
import pytest
import torch

import dfattn
import kv8_reference as ref
from dfattn import ops

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


def i32(x, device):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=device)


# ---------------------------------------------------------------- plan
PLANS = [
    # cached, new, page, max_pages, free pages, first free, capacity
    ([0], [1], 16, 1, 1, 0, 1),
    ([16], [1], 16, 2, 1, 0, 4),
    ([15], [1], 16, 1, 0, 0, 1),
    ([0, 0, 0], [0, 0, 0], 16, 2, 4, 1, 0),
    ([5, 0, 31, 64, 7], [11, 40, 1, 0, 200], 16, 20, 60, 3, 300),
    ([5, 0, 31, 64, 7], [11, 40, 1, 5, 200], 16, 20, 12, 3, 300),   # the pages run out at the last request
    ([5, 0, 31, 64, 7], [11, 40, 1, 5, 200], 16, 20, 5, 3, 300),    # ... at the second
    ([5, 0, 31, 64, 7], [11, 40, 1, 5, 200], 16, 20, 60, 3, 100),   # the tokens do
    ([5, 0, 31, 64, 7], [11, 400, 1, 5, 20], 16, 20, 60, 3, 500),   # one is longer than its table row
    ([3, 9], [4, 5], 7, 3, 9, 0, 16),                               # a page size of no power of two
    (list(range(700)), [1] * 700, 16, 50, 100, 0, 1000),
    ([i % 37 for i in range(8192)], [(i * 7) % 5 for i in range(8192)], 32, 2, 9000, 11, 20000),
]


@pytest.mark.parametrize("case", range(len(PLANS)))
def test_plan(device, case):
    cached, new, page, width, n_free, first, capacity = PLANS[case]
    say("plan", case)
    r = len(cached)
    had = [-(-c // page) for c in cached]
    n_pages = sum(had) + n_free
    rng = np.random.RandomState(case)
    order = rng.permutation(n_pages)
    table = np.full((r, width), 12345678)
    at = 0
    for i in range(r):
        table[i, :had[i]] = order[at:at + had[i]]
        at += had[i]
    free = order[at:]
    want = ref.plan(cached, new, table, free, first, page, n_pages, capacity)
    got_table = i32(table, device)
    got = dfattn.paged_plan(i32(cached, device), i32(new, device), got_table, i32(free, device), i32([first], device),
                            page, n_pages, capacity)
    for name, t in zip(("seq_lens", "query_start", "slots", "counts"), got):
        assert np.array_equal(t.cpu().numpy(), want[name]), name
    assert np.array_equal(got_table.cpu().numpy(), want["table"])


def test_plan_with_bad_pages_and_free_start(device):
    """A page id outside the pool gives no slot; a free_start past the list leaves nothing free."""
    table = i32([[7, -1, 0]], device)
    seq, start, slots, counts = dfattn.paged_plan(i32([17], device), i32([20], device), table, i32([3], device),
                                                  i32([0], device), 16, 4, 24)
    # positions 17..31 lie in page -1, 32..36 in the new page 3.
    assert slots.tolist() == [-1] * 15 + [48 + i for i in range(5)] + [-1] * 4
    assert seq.tolist() == [37] and counts.tolist() == [1, 20, 1] and table.tolist() == [[7, -1, 3]]
    table = i32([[7, -1, 0]], device)
    seq, start, slots, counts = dfattn.paged_plan(i32([17], device), i32([20], device), table, i32([3], device),
                                                  i32([5], device), 16, 4, 24)
    assert counts.tolist() == [0, 0, 1] and seq.tolist() == [17] and start.tolist() == [0, 0]
    assert slots.tolist() == [-1] * 24 and table.tolist() == [[7, -1, 0]]


# ---------------------------------------------------------------- append and read
def random_rows(rng, n, heads, d, spread=3.0):
    x = rng.randn(n, heads, d) * np.exp(rng.randn(n, heads, 1) * spread)
    return x.astype(np.float32)


def as_act(x, act, device):
    return torch.tensor(x, device=device).to(ref.ACT[act])


SHAPES = [(1, 1, 16), (2, 3, 16), (12, 64, 16), (3, 80, 32), (2, 100, 48), (8, 128, 16), (1, 128, 256), (4, 33, 64)]


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("heads,d,page", SHAPES)
def test_append_and_read(device, heads, d, page, fmt, act):
    """Several appends into the same pages (one row, a few, across pages, over rows written before), every value
    and scale bit for bit; the slots nobody wrote keep their bytes."""
    say("append", heads, d, page, fmt, act)
    rng = np.random.RandomState(heads * 1000 + d)
    pages = 6
    cache = dfattn.kv8_cache(pages, heads, d, page, ref.DTYPE[fmt], device)
    k_ref, v_ref = (ref.Cache(pages, heads, page, d, fmt) for _ in range(2))
    calls = [
        [2 * page],                                              # one row at a page's start
        [2 * page + 1, 2 * page + 2, 2 * page + 3],              # three after it
        [5 * page + i for i in range(page)],                     # a whole page
        [2 * page + 4 + i for i in range(page - 4)] + [i for i in range(page)] + [4 * page, 4 * page + 1],
        [2 * page + 2],                                          # written again: rows 0, 1 are kept
        [4 * page + 2, -1, -1, pages * page, 2 ** 31 - 1],       # slots that are none
        [4 * page + 3 + i for i in range(7)] + [5 * page],       # another page begins anew
    ]
    valid = {}
    for n, slots in enumerate(calls):
        spread = (0.5, 3.0, 1.0)[n % 3]
        k, v = (as_act(random_rows(rng, len(slots), heads, d, spread), act, device) for _ in range(2))
        k_ref.append(k.double().cpu().numpy(), slots)
        v_ref.append(v.double().cpu().numpy(), slots)
        dfattn.kv8_append(cache, k.view(len(slots), -1), v.view(len(slots), -1), i32(slots, device))
        for s in slots:
            if 0 <= s < pages * page:
                valid = {x for x in valid if x // page != s // page or x < s} | {s}
        at = sorted(valid)
        got = dfattn.kv8_read(cache, i32(at, device), d)
        for name, g, w in zip("kv", got, (k_ref, v_ref)):
            assert np.array_equal(g.double().cpu().numpy(), w.read(at)), (name, n)
        for t, w in ((cache.k_scale, k_ref), (cache.v_scale, v_ref)):
            assert np.array_equal(t.double().cpu().numpy(), w.scale), n
    # Any order, repeats, no slots, bf16 out (rounded once).
    at = [at[-1], -1, at[0], at[0], pages * page + 3] + at[::-1]
    for dtype in (torch.float32, torch.bfloat16):
        got = dfattn.kv8_read(cache, i32(at, device), d, dtype)
        for g, w in zip(got, (k_ref, v_ref)):
            assert torch.equal(g.cpu(), torch.tensor(w.read(at)).to(dtype))
    untouched = [3]  # no call wrote page 3
    assert not cache.k.view(torch.int8)[untouched].any() and not cache.v.view(torch.int8)[untouched].any()


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_append_extremes(device, fmt):
    """Zeros, the smallest and largest numbers, and values on every rounding tie."""
    heads, d, page = 2, 64, 16
    cache = dfattn.kv8_cache(4, heads, d, page, ref.DTYPE[fmt], device)
    k_ref = ref.Cache(4, heads, page, d, fmt)
    x = np.zeros((page * 3, heads, d), np.float32)
    top = ref.LIMIT[fmt]
    x[page:2 * page, 0] = np.linspace(-top, top, page * d).reshape(page, d).astype(np.float32)
    x[page:2 * page, 1] = (np.arange(page * d).reshape(page, d) % 255 - 127) + 0.5  # ties
    x[page:2 * page, 1, 0] = 127.0
    x[2 * page, 0, :4] = [3.4028235e38, -3.4028235e38, 1e-45, -1.2e-38]
    x[2 * page, 1, :4] = [1e-45, -1e-42, 1.2e-38, -1.1e-38]
    slots = np.arange(page * 3)
    k = torch.tensor(x, device=device)
    k_ref.append(x.astype(np.float64), slots)
    dfattn.kv8_append(cache, k.view(len(slots), -1), k.view(len(slots), -1), i32(slots, device))
    got, got_v = dfattn.kv8_read(cache, i32(slots, device), d)
    # fp32's largest number rounds to the code 64 times 2^122 (int8) or 256 times 2^120 (e4m3): 2^128 either way,
    # which is infinity in fp32, the type the values are read in.
    with np.errstate(over="ignore"):
        assert np.array_equal(got.cpu().numpy(), k_ref.read(slots).astype(np.float32))
    assert torch.equal(got, got_v)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_append_of_infinities_and_nan(device, fmt, bad):
    """The page and head that got one is NaN as a whole, later rows too, until its first row is written again;
    the other heads and pages are not touched."""
    heads, d, page = 3, 20, 16
    rng = np.random.RandomState(1)
    cache = dfattn.kv8_cache(3, heads, d, page, ref.DTYPE[fmt], device)
    x = random_rows(rng, 2 * page, heads, d)
    put = lambda rows, slots: dfattn.kv8_append(cache, rows.reshape(len(slots), -1), rows.reshape(len(slots), -1),
                                                i32(slots, device))
    put(torch.tensor(x[:20], device=device), list(range(20)))
    clean = dfattn.kv8_read(cache, i32(range(20), device), d)
    y = torch.tensor(x[20:22], device=device)
    y[1, 1, 7] = bad
    put(y, [20, 21])
    put(torch.tensor(x[22:24], device=device), [22, 23])
    for g, w in zip(dfattn.kv8_read(cache, i32(range(24), device), d), clean):
        g, w = g.view(24, heads, d), w.view(20, heads, d)
        assert torch.isnan(g[16:24, 1]).all()
        assert torch.equal(g[:16], w[:16]) and not torch.isnan(g[:, [0, 2]]).any()
    put(torch.tensor(x[:2], device=device), [16, 17])
    for g in dfattn.kv8_read(cache, i32([16, 17], device), d):
        assert torch.isfinite(g).all()


def test_append_from_a_fused_projection(device):
    """Column blocks of one [n, 3 H d] tensor, at an offset that is not 16-byte aligned too."""
    heads, d, page, n = 3, 20, 16, 21
    for act in ("f32", "bf16"):
        wide = as_act(np.random.RandomState(3).randn(n, 3 * heads * d + 1), act, device)
        for shift in (0, 1):
            k, v = (wide[:, shift + i * heads * d:shift + (i + 1) * heads * d] for i in (1, 2 if shift else 2))
            a = dfattn.kv8_cache(2, heads, d, page, device=device)
            b = dfattn.kv8_cache(2, heads, d, page, device=device)
            slots = i32(range(n), device)
            dfattn.kv8_append(a, k, v, slots)
            dfattn.kv8_append(b, k.contiguous(), v.contiguous(), slots)
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def check_calls(device, heads, d, page, pages, fmt, act, calls, shift=0, extra=0, spreads=(0.5, 3.0)):
    """Appends `calls` (lists of slots) and compares every written value and scale bit for bit; rows of k and v
    start heads * d + extra elements apart, the first at element `shift`."""
    rng = np.random.RandomState(heads * 1000 + d + page)
    cache = dfattn.kv8_cache(pages, heads, d, page, ref.DTYPE[fmt], device)
    refs = [ref.Cache(pages, heads, page, d, fmt) for _ in range(2)]
    top = {}
    for n, slots in enumerate(calls):
        wide = [as_act(random_rows(rng, len(slots), 1, heads * d + extra, spreads[n % len(spreads)])[:, 0], act, device)
                for _ in range(2)]
        kv = [w[:, shift:shift + heads * d] for w in wide]
        for r, x in zip(refs, kv):
            r.append(x.double().cpu().numpy().reshape(len(slots), heads, d), slots)
        dfattn.kv8_append(cache, *kv, i32(slots, device))
        for s_ in slots:
            if 0 <= s_ < pages * page:
                top[s_ // page] = s_ % page
        at = [p_ * page + o for p_ in sorted(top) for o in range(top[p_] + 1)]
        for name, g, w in zip("kv", dfattn.kv8_read(cache, i32(at, device), d), refs):
            assert np.array_equal(g.double().cpu().numpy(), w.read(at)), (name, n)
        for t, w in zip(cache[2:], refs):
            assert np.array_equal(t.double().cpu().numpy(), w.scale), n


@pytest.mark.parametrize("fmt,act", [("i8", "f32"), ("e4m3", "bf16")])
@pytest.mark.parametrize("heads,d,page,extra,shift", [
    (2, 64, 16, 0, 0), (3, 128, 16, 4, 0), (1, 20, 48, 1, 1), (2, 64, 64, 0, 0), (1, 100, 64, 8, 4), (2, 33, 128, 0, 0),
    (1, 128, 256, 3, 2), (9, 16, 256, 0, 0)])
def test_append_long_runs(device, heads, d, page, extra, shift, fmt, act):
    """Prompts of many pages with partial first and last ones, rows behind kept rows whose scale grows, runs that
    begin and end anywhere among the tokens, and a thousand requests of one token between them."""
    say("long runs", heads, d, page, fmt, act)
    pages = 1700 if page == 16 else 400 if page <= 64 else 130
    order = np.random.RandomState(page).permutation(pages)
    pos = lambda first, a, b: [int(order[first + t // page]) * page + t % page for t in range(a, b)]
    few = 5 + page // 3
    calls = [
        pos(0, 0, 5) + pos(20, 0, few),                                     # small values
        pos(0, 5, 5 * page + 3) + [-1, -1] + pos(20, few, 3 * page),        # larger ones behind them
        pos(0, 5 * page + 3, 5 * page + 4) + pos(20, 3 * page, 3 * page + 2) +
        [s for i in range(30, pages) for s in pos(i, 0, 1)] + pos(10, 0, 6 * page + 1),
        [s for i in range(30, pages) for s in pos(i, 1, 2 + i % 2)] + pos(10, 6 * page + 1, 6 * page + 2),
    ]
    check_calls(device, heads, d, page, pages, fmt, act, calls, shift, extra)


# ---------------------------------------------------------------- attention
def build(device, lens, heads, d, page, fmt, seed, junk=True):
    """A cache holding lens[r] tokens of each request through the append, in scattered pages, the rest of the
    pool and of the table filled with junk; (cache, table, seq_lens, values of K and V per request)."""
    rng = np.random.RandomState(seed)
    width = max(1, max(-(-n // page) for n in lens) + 1)
    pages = [-(-n // page) for n in lens]
    n_pages = sum(pages) + 2
    order = rng.permutation(n_pages)
    cache = dfattn.kv8_cache(n_pages, heads, d, page, ref.DTYPE[fmt], device)
    if junk:
        for t in cache[:2]:
            t.view(torch.uint8).fill_(0xff)  # e4m3: NaN; int8: -1
        for t in cache[2:]:
            t.fill_(math.nan)
    table = np.full((len(lens), width), 2 ** 31 - 1)
    at, vals = 0, []
    for r, n in enumerate(lens):
        table[r, :pages[r]] = order[at:at + pages[r]]
        at += pages[r]
        if not n:
            vals.append((np.zeros((0, heads, d)),) * 2)
            continue
        pos = np.arange(n)
        slots = i32(table[r, pos // page] * page + pos % page, device)
        k = rng.randn(n, heads, d) * np.where(np.arange(d) % 16 == 0, 3.0, 1.0)
        v = rng.randn(n, heads, d)
        dfattn.kv8_append(cache, *(torch.tensor(x.reshape(n, -1), dtype=torch.float32, device=device) for x in (k, v)),
                          slots)
        vals.append(tuple(x.double().cpu().numpy().reshape(n, heads, d) for x in dfattn.kv8_read(cache, slots, d)))
    return cache, i32(table, device), i32(lens, device), vals


def check_attention(device, lens, qlens, heads, kv_heads, d, page, fmt, act, causal=True, scale=None, seed=0, qstd=1.5,
                    workspace="auto", bad=(), pad=3):
    cache, table, seq, vals = build(device, lens, kv_heads, d, page, fmt, seed)
    rng = np.random.RandomState(seed + 1)
    start = np.concatenate([[0], np.cumsum(qlens)])
    n = int(start[-1]) + pad
    q = as_act(rng.randn(n, heads * d) * qstd, act, device)
    scale = d ** -0.5 if scale is None else scale
    oks = [np.ones(len(vals[r][0]), bool) for r in range(len(lens))]
    for r, page_index, value in bad:
        table[r, page_index] = value
        oks[r][page_index * page:(page_index + 1) * page] = False
    out = torch.full((n, heads * d), 7.0, dtype=q.dtype, device=device)
    lse = torch.full((heads, n), 7.0, device=device)
    max_q, max_len = max(qlens), max(max(lens), 1)
    dfattn.kv8_attention(cache, q, table, i32(start, device), seq, heads, max_q, max_len, scale, causal, out, lse,
                         workspace)
    want, wlse, tol, ltol = ref.attention(
        q.double().cpu().numpy(), lambda r: (vals[r][0], oks[r]), lambda r: (vals[r][1], oks[r]), start, lens, heads,
        kv_heads, d, scale, causal, n, 2.0 ** -22 if act == "f32" else 2.0 ** -11, 0.0 if act == "f32" else 2.0 ** -8,
        page)
    m = int(start[-1])
    got, glse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    assert (got[m:] == 7.0).all() and (glse[:, m:] == 7.0).all(), "rows behind the last sequence"
    assert np.array_equal(np.isneginf(glse[:, :m]), np.isneginf(wlse[:, :m]))
    fin = ~np.isneginf(wlse[:, :m])
    assert not np.isnan(got).any()
    over = np.abs(got - want)[:m] / np.maximum(tol[:m], 1e-300)
    lover = (np.abs(glse - np.where(np.isneginf(wlse), 0, wlse))[:, :m] / np.maximum(ltol[:, :m], 1e-300))[fin]
    say("  out %.3f of its bound, lse %.3f" % (over[tol[:m] > 0].max() if (tol[:m] > 0).any() else 0.0,
                                               lover.max() if lover.size else 0.0))
    assert (np.abs(got - want)[:m] <= tol[:m]).all()
    assert not lover.size or lover.max() <= 1
    return cache, table, seq, q, start, out, lse


ATTENTION = [
    # lens, query lens, heads, kv heads, d, page
    ([1], [1], 1, 1, 64, 16),
    ([2], [1], 12, 12, 64, 16),
    ([16], [1], 2, 2, 16, 16),
    ([17], [1], 2, 2, 1, 16),
    ([63, 64, 65], [1, 1, 1], 12, 12, 64, 16),
    ([300, 0, 1, 1000], [1, 1, 1, 1], 4, 4, 64, 16),             # an empty cache: zeros and -inf
    ([257, 511], [1, 1], 6, 2, 128, 32),
    ([700, 33], [1, 1], 8, 1, 80, 64),
    ([129], [1], 16, 1, 100, 16),
    ([90, 200], [1, 1], 24, 1, 64, 16),                          # more heads on one kv head than a tile's columns
    ([90], [1], 71, 1, 32, 16),                                  # ... than the widest
    ([5, 70, 128], [5, 3, 17], 4, 4, 64, 16),                    # prompts: whole, part, more rows than a tile
    ([200, 40], [33, 40], 2, 1, 112, 48),
    ([300], [65], 3, 3, 64, 256),
    ([150, 0, 90], [0, 0, 90], 2, 2, 33, 16),                    # requests without tokens
    ([3, 10], [7, 10], 2, 2, 64, 16),                            # more queries than positions: rows that see nothing
    ([1500, 20], [1, 4], 4, 2, 64, 16),                          # generating beside a short prompt
    ([1100], [130], 2, 1, 128, 32),
]


@pytest.mark.parametrize("fmt,act", [("i8", "f32"), ("e4m3", "bf16"), ("e4m3", "f32"), ("i8", "bf16")])
@pytest.mark.parametrize("case", range(len(ATTENTION)))
def test_attention(device, case, fmt, act):
    say("attention", case, ATTENTION[case], fmt, act)
    lens, qlens, heads, kv_heads, d, page = ATTENTION[case]
    check_attention(device, lens, qlens, heads, kv_heads, d, page, fmt, act, seed=case)


# Tiles cut between workgroups into two to seventy pieces, of one query to more than a tile's.
CUT = [
    ([2300], [1], 2, 2, 64, 16),
    ([7000, 1], [1, 1], 4, 2, 32, 16),
    ([20000], [1], 1, 1, 64, 32),
    ([36000, 300], [1, 1], 1, 1, 16, 16),
    ([5000, 2300, 130], [9, 1, 100], 4, 2, 128, 64),
    ([9000], [20], 2, 1, 64, 16),
    ([20000], [20], 2, 1, 32, 16),
    ([1300], [1], 600, 600, 16, 16),
    ([2100], [1], 600, 600, 16, 16),                             # more heads than workgroups run at a time
    ([2048, 100], [1, 3], 4, 2, 64, 16),                         # the longest few queries that one workgroup walks
    ([2049, 100], [1, 3], 4, 2, 64, 16),
    ([1025, 1024, 0, 513], [3, 0, 2, 513], 1, 1, 80, 48),
    ([1500, 300, 64], [200, 1, 64], 1, 1, 64, 16),               # many queries of small heads
    ([2200, 1100], [97, 30], 6, 2, 32, 48),
    ([4100, 700], [191, 260], 2, 2, 33, 64),
    ([900, 230], [230, 193], 2, 2, 64, 16),                      # ... of sequences that are not shared out
    ([260] * 40, [200] + [1] * 38 + [195], 4, 4, 16, 16),        # ... in more tiles than run at once
]


@pytest.mark.parametrize("fmt,act", [("i8", "f32"), ("e4m3", "bf16")])
@pytest.mark.parametrize("case", range(len(CUT)))
def test_attention_cut_between_workgroups(device, case, fmt, act):
    say("cut", case, CUT[case], fmt, act)
    lens, qlens, heads, kv_heads, d, page = CUT[case]
    check_attention(device, lens, qlens, heads, kv_heads, d, page, fmt, act, seed=100 + case)


@pytest.mark.parametrize("longest", [1500, 2100])
@pytest.mark.parametrize("r", [4096, 4097])
def test_attention_of_many_requests(device, r, longest):
    """The most requests whose work is shared out, and one more, with one long sequence among them."""
    say("requests", r)
    lens, qlens = [1 + i % 3 for i in range(r)], [1 - (i % 7 == 3) for i in range(r)]
    lens[r // 2] = longest
    check_attention(device, lens, qlens, 1, 1, 16, 16, "i8", "f32", seed=r)


def test_attention_of_many_requests_with_long_bounds(device):
    """Bounds that allow every request many queries, nearly as many (request, tile) pairs as are shared out."""
    r = 815
    lens, qlens = [1 + i % 3 for i in range(r)], [i % 2 for i in range(r)]
    lens[400], qlens[400] = 1500, 200
    say("requests", r)
    check_attention(device, lens, qlens, 1, 1, 16, 16, "i8", "f32", seed=r)


@pytest.mark.parametrize("d", [64, 128])
def test_chunks_replayed_from_a_graph(device, d):
    """Captured before any call of the kind, replayed with other queries."""
    heads, lens, qlens = 2, [2100, 300], [230, 41]
    cache, table, seq, _ = build(device, lens, heads, d, 16, "i8", 50 + d)
    start = i32([0, 230, 271], device)
    q = torch.zeros(271, heads * d, device=device)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = dfattn.kv8_attention(cache, q, table, start, seq, heads, 230, 2100)
    for seed in range(3):
        q.copy_(torch.randn(271, heads * d, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        want = dfattn.kv8_attention(cache, q, table, start, seq, heads, 230, 2100)
        assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_requests_that_share_pages(device):
    """Two requests with a common prefix in the same pages, each with a last page of its own."""
    heads, d, page, n = 2, 64, 16, 200
    cache, table, seq, vals = build(device, [n, n], heads, d, page, "i8", 31)
    common = table.clone()
    common[1, :n // page] = table[0, :n // page]
    q = torch.randn(1, heads * d, device=device)
    out, _ = dfattn.kv8_attention(cache, q.repeat(2, 1), common, i32([0, 1, 2], device), seq, heads, 1, n)
    ok = np.ones(n, bool)
    k, v = (np.concatenate([vals[0][i][:n // page * page], vals[1][i][n // page * page:]]) for i in range(2))
    for r, (kr, vr) in enumerate((vals[0], (k, v))):
        want, _, tol, _ = ref.attention(q.double().cpu().numpy(), lambda _: (kr, ok), lambda _: (vr, ok), [0, 1], [n], heads,
                                        heads, d, d ** -0.5, True, 1, 2.0 ** -22, 0.0, page)
        assert (np.abs(out[r].double().cpu().numpy() - want[0]) <= tol[0]).all()


def test_two_streams_at_once(device):
    """Calls that overlap, each with its own cache and workspace."""
    sets = []
    for i in range(2):
        cache, table, seq, _ = build(device, [3000 + 100 * i, 700], 4, 64, 16, "i8", 40 + i)
        q = torch.randn(2, 4 * 64, device=device)
        start = i32([0, 1, 2], device)
        sets.append((cache, q, table, start, seq, dfattn.kv8_attention(cache, q, table, start, seq, 4, 1, 3100)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(10):
        for s, (cache, q, table, start, seq, want) in zip(streams, sets):
            got.append((dfattn.kv8_attention(cache, q, table, start, seq, 4, 1, 3100, stream=s), want))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for g, w in got for x, y in zip(g, w))


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("case", [1, 5, 6, 11, 12, 15])
def test_attention_without_mask(device, case, act):
    lens, qlens, heads, kv_heads, d, page = ATTENTION[case]
    say("no mask", case)
    check_attention(device, lens, qlens, heads, kv_heads, d, page, "i8", act, causal=False, seed=case)


@pytest.mark.parametrize("case", [5, 7, 12, 16])
def test_attention_without_workspace(device, case):
    lens, qlens, heads, kv_heads, d, page = ATTENTION[case]
    say("no workspace", case)
    check_attention(device, lens, qlens, heads, kv_heads, d, page, "e4m3", "f32", seed=case, workspace=None)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_attention_large_and_small_scores(device, fmt):
    """Scores far beyond exp's range, a scale of zero, and a negative one."""
    for scale, std in ((1.0, 30.0), (0.0, 1.0), (-0.2, 2.0), (1e-3, 1e-3)):
        say("scale", scale, std)
        check_attention(device, [200, 37], [1, 5], 4, 2, 64, 16, fmt, "f32", scale=scale, qstd=std, seed=9)


def test_attention_leaves_bad_pages_out(device):
    """Keys in pages outside the pool are left out, a request of nothing else gets zeros."""
    check_attention(device, [100, 30, 16], [1, 3, 1], 4, 2, 64, 16, "e4m3", "f32", seed=4,
                    bad=[(0, 1, -1), (0, 6, 2 ** 30), (1, 0, -5), (2, 0, 9999)])


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_attention_value_magnitudes(device, fmt):
    """Pages whose scales lie many powers of two apart, up to values near fp32's limits."""
    heads, d, page, n = 2, 64, 16, 160
    rng = np.random.RandomState(5)
    for shift in (0, 100, -100):
        say("magnitudes", fmt, shift)
        cache = dfattn.kv8_cache(10, heads, d, page, ref.DTYPE[fmt], device)
        k = rng.randn(n, heads, d)
        v = rng.randn(n, heads, d) * 2.0 ** (rng.randint(-20, 20, (n // page, 1, 1, 1)).repeat(page, 1).reshape(n, 1, 1) + shift)
        slots = i32(range(n), device)
        dfattn.kv8_append(cache, *(torch.tensor(x.reshape(n, -1), dtype=torch.float32, device=device) for x in (k, v)), slots)
        kr, vr = (x.double().cpu().numpy().reshape(n, heads, d) for x in dfattn.kv8_read(cache, slots, d))
        q = torch.tensor(rng.randn(1, heads * d), dtype=torch.float32, device=device)
        out, lse = dfattn.kv8_attention(cache, q, i32([list(range(10))], device), i32([0, 1], device), i32([n], device),
                                        heads, 1, n)
        ok = np.ones(n, bool)
        want, wlse, tol, ltol = ref.attention(q.double().cpu().numpy(), lambda r: (kr, ok), lambda r: (vr, ok), [0, 1],
                                              [n], heads, heads, d, d ** -0.5, True, 1, 2.0 ** -22, 0.0, page)
        assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()
        assert (np.abs(lse.double().cpu().numpy() - wlse) <= ltol).all()


def test_attention_nan_stays_in_its_page_and_head(device):
    """A NaN value poisons its head's rows that see the page, and no others."""
    heads, d, page = 2, 64, 16
    rng = np.random.RandomState(6)
    cache = dfattn.kv8_cache(6, heads, d, page, torch.float8_e4m3fn, device)
    x = torch.tensor(rng.randn(70, heads * d), dtype=torch.float32, device=device)
    x[40, d + 3] = math.nan  # head 1, the page of positions 32..47
    dfattn.kv8_append(cache, x, x, i32(range(70), device))
    q = torch.tensor(rng.randn(70, heads * d), dtype=torch.float32, device=device)
    out, lse = dfattn.kv8_attention(cache, q, i32([range(6)], device), i32([0, 70], device), i32([70], device), heads, 70,
                                    70)
    bad = torch.isnan(out).view(70, heads, d)
    assert not bad[:, 0].any() and not bad[:32, 1].any() and bad[32:, 1].all()
    assert torch.isnan(lse[1, 32:]).all() and torch.isfinite(lse[0]).all() and torch.isfinite(lse[1, :32]).all()


def test_attention_layouts(device):
    """Queries in a column block of a wider tensor, at odd offsets; no lse (through the C entry)."""
    lens, heads, d = [77, 200], 4, 64
    cache, table, seq, _ = build(device, lens, heads, d, 16, "i8", 2)
    start = i32([0, 2, 5], device)
    for act in (torch.float32, torch.bfloat16):
        wide = torch.randn(5, 3 * heads * d + 5, device=device).to(act)
        for shift in (0, 1, 3):
            q = wide[:, shift:shift + heads * d]
            a, la = dfattn.kv8_attention(cache, q, table, start, seq, heads, 3, 200)
            b, lb = dfattn.kv8_attention(cache, q.contiguous(), table, start, seq, heads, 3, 200)
            assert torch.equal(a, b) and torch.equal(la, lb)
        c = torch.empty_like(b)
        p = lambda t: ctypes.c_void_p(t.data_ptr())
        st = dfattn.lib().dfattn_kv8_attention(
            p(q), *map(p, cache), p(table), p(start), p(seq), p(c), None, 0 if act == torch.float32 else 1, 2, 2, 5, 3,
            200, heads, heads, d, 16, cache.k.shape[0], table.shape[1], q.stride(0), d ** -0.5, 1, None, 0,
            torch.cuda.current_stream().cuda_stream)
        assert st == 0
        d_, _ = dfattn.kv8_attention(cache, q, table, start, seq, heads, 3, 200, workspace=None)
        assert torch.equal(c, d_)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_offsets_past_32_bits(device, fmt):
    """A pool of more than 2^32 bytes: a request's pages at its very end and at its start, through append, read
    and attention, against the same request in a small pool."""
    heads, d, page, n = 16, 128, 256, 600
    pages = (1 << 32) // (heads * d * page) + 40
    say("pages", pages)
    shape = (pages, heads, page, d)
    big = dfattn.KV8Cache(torch.empty(shape, dtype=torch.int8, device=device).view(ref.DTYPE[fmt]),
                          torch.empty((pages, heads, d, page), dtype=torch.int8, device=device).view(ref.DTYPE[fmt]),
                          *(torch.empty((pages, heads), device=device) for _ in range(2)))
    small = dfattn.kv8_cache(3, heads, d, page, ref.DTYPE[fmt], device)
    g = torch.Generator(device=device).manual_seed(3)
    k, v = (torch.randn(n, heads * d, generator=g, device=device) for _ in range(2))
    q = torch.randn(2, heads * d, generator=g, device=device)
    where = np.array([pages - 1, 0, pages - 2])
    pos = np.arange(n)
    got = []
    for cache, table in ((big, where), (small, np.arange(3))):
        slots = i32(table[pos // page] * page + pos % page, device)
        dfattn.kv8_append(cache, k, v, slots)
        got.append(dfattn.kv8_read(cache, slots, d) + dfattn.kv8_attention(
            cache, q, i32([table], device), i32([0, 2], device), i32([n], device), heads, 2, n))
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_bounds_that_are_not_met(device):
    """A longer sequence than max_seq_len is walked whole, queries past max_query_len are left as they were."""
    lens, heads, d = [700], 2, 64
    cache, table, seq, _ = build(device, lens, heads, d, 16, "i8", 8)
    q = torch.randn(5, heads * d, device=device)
    start = i32([0, 5], device)
    want, _ = dfattn.kv8_attention(cache, q, table, start, seq, heads, 5, 700)
    got, _ = dfattn.kv8_attention(cache, q, table, start, seq, heads, 5, 64)
    assert (got - want).abs().max() <= 1e-5
    out = torch.full_like(q, 3.0)
    dfattn.kv8_attention(cache, q, table, start, seq, heads, 2, 700, out=out)
    assert (out[:2] - want[:2]).abs().max() <= 1e-5 and (out[2:] == 3.0).all()


def test_results_repeat_bit_for_bit(device):
    lens = [3000, 50, 1]
    cache, table, seq, _ = build(device, lens, 4, 64, 16, "e4m3", 7)
    q = torch.randn(3, 4 * 64, device=device)
    first = dfattn.kv8_attention(cache, q, table, i32([0, 1, 2, 3], device), seq, 4, 1, 3000)
    for _ in range(3):
        again = dfattn.kv8_attention(cache, q, table, i32([0, 1, 2, 3], device), seq, 4, 1, 3000)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


# ---------------------------------------------------------------- together
def serve(device, graph, steps=20, fmt="i8", stream=None):
    """A small serving loop: three prompts in one step, then one token a step; q, k, v and logits made from a
    fixed table of vectors by token. Returns what each step answered."""
    heads, d, page, vocab, r = 4, 32, 16, 211, 3
    g = torch.Generator(device=device).manual_seed(11)
    emb = torch.randn(vocab, 3 * heads * d, generator=g, device=device)
    head = torch.randn(heads * d, vocab, generator=g, device=device)
    n_pages, width, cap = 40, 8, 64
    cache = dfattn.kv8_cache(n_pages, heads, d, page, ref.DTYPE[fmt], device)
    table = torch.full((r, width), -1, dtype=torch.int32, device=device)
    free = torch.randperm(n_pages, generator=g, device=device).int()
    first = torch.zeros(1, dtype=torch.int32, device=device)
    cached = torch.zeros(r, dtype=torch.int32, device=device)
    prompts = [[5, 9, 200, 7], [1] * 17, [3, 4]]
    ids = torch.zeros(cap, dtype=torch.int32, device=device)
    new = torch.zeros(r, dtype=torch.int32, device=device)

    def step(max_q):
        seq, start, slots, counts = dfattn.paged_plan(cached, new, table, free, first, page, n_pages, cap, stream=stream)
        x = emb[ids.long()]
        q, k, v = (x[:, i * heads * d:(i + 1) * heads * d] for i in range(3))
        dfattn.kv8_append(cache, k, v, slots, stream=stream)
        out, _ = dfattn.kv8_attention(cache, q, table, start, seq, heads, max_q, width * page, stream=stream)
        last = out[(start[1:] - 1).long()]
        logits = last @ head
        best = logits.argmax(1).int()
        lp, ent, _, top, top_lp = ops.token_logprobs_forward(logits, best, 5)
        cached.copy_(seq)
        first.copy_(counts[2:])
        ids[:r] = best
        return best, lp, ent, top, top_lp

    flat = [t for p in prompts for t in p]
    ids[:len(flat)] = i32(flat, device)
    new.copy_(i32([len(p) for p in prompts], device))
    history = [list(p) for p in prompts]
    answers = [[t.clone() for t in step(17)]]
    new.fill_(1)
    if graph:
        keep = [t.clone() for t in (*[c.view(torch.int8) if i < 2 else c for i, c in enumerate(cache)], table, first,
                                    cached, ids)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(1)
        torch.cuda.current_stream().wait_stream(side)
        rec = torch.cuda.CUDAGraph()
        with torch.cuda.graph(rec):
            held = step(1)
        for t, o in zip((cache.k.view(torch.int8), cache.v.view(torch.int8), cache.k_scale, cache.v_scale, table, first,
                         cached, ids), keep):
            t.copy_(o)
    for _ in range(steps):
        if graph:
            rec.replay()
            torch.cuda.synchronize()
            answers.append([t.clone() for t in held])
        else:
            answers.append([t.clone() for t in step(1)])
    for a in answers:
        for i, t in enumerate(a[0].tolist()):
            history[i].append(t)
    return answers, history, cache, table, cached, emb, head, (heads, d, page)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_serving_loop(device, fmt):
    """Plan, append, attention and log probabilities together, against the whole history in float64 from the
    values the cache holds at the end of each request."""
    say("serving loop", fmt)
    answers, history, cache, table, cached, emb, head, (heads, d, page) = serve(device, False, fmt=fmt)
    assert cached.tolist() == [len(h) - 1 for h in history]
    for i, h in enumerate(history):
        n = len(h) - 1
        pos = np.arange(n)
        slots = i32(table[i].cpu().numpy()[pos // page] * page + pos % page, device)
        k, v = (x.double().cpu().view(n, heads, d) for x in dfattn.kv8_read(cache, slots, d))
        q = emb[h[n - 1], :heads * d].double().cpu().view(heads, d)
        p = torch.softmax((k * q).sum(-1) * d ** -0.5, 0)
        out = (p[:, :, None] * v).sum(0).reshape(-1)
        logits = out @ head.double().cpu()
        logp = torch.log_softmax(logits, 0)
        best, lp, ent, top, top_lp = (t[i].cpu() for t in answers[-1])
        # Attention's error (2^-20 of |v| sums at most here) times the head's row sums, twice for the softmax.
        tol = 2 * 2.0 ** -18 * float(head.abs().sum(0).max())
        assert abs(float(lp) - float(logp[h[-1]])) <= tol
        assert abs(float(ent) + float((logp.exp() * logp).sum())) <= tol * 8
        assert top[0] == best and (top_lp.double() - logp[top.long()]).abs().max() <= tol


def test_serving_loop_replayed_from_a_graph(device):
    """The generating step captured once and replayed, every replay against the eager loop."""
    say("graph")
    eager = serve(device, False)
    replayed = serve(device, True)
    assert eager[1] == replayed[1]
    for a, b in zip(eager[0], replayed[0]):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_two_graphs_share_a_workspace_in_turn(device):
    lens = [2600, 900]
    cache, table, seq, _ = build(device, lens, 4, 64, 16, "i8", 3)
    start = i32([0, 1, 2], device)
    need = dfattn.kv8_attention_workspace_bytes(2, 2, 1, 2600, 4, 4, 64)
    assert need > 0
    ws = torch.empty(need // 4, device=device)
    qs = [torch.randn(2, 4 * 64, device=device) for _ in range(2)]
    want = [dfattn.kv8_attention(cache, q, table, start, seq, 4, 1, 2600) for q in qs]
    graphs, outs = [], []
    for q in qs:
        out, lse = torch.empty_like(q), torch.empty(4, 2, device=device)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            dfattn.kv8_attention(cache, q, table, start, seq, 4, 1, 2600, out=out, lse=lse, workspace=ws)
        graphs.append(g)
        outs.append((out, lse))
    for _ in range(3):
        for i in (0, 1, 1, 0):
            for t in outs[i]:
                t.zero_()
            graphs[i].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i]))


def test_calls_on_another_stream(device):
    """The stream argument: the call and what it allocates belong to that stream."""
    lens = [2500, 100]
    cache, table, seq, _ = build(device, lens, 4, 64, 16, "i8", 12)
    start, q = i32([0, 1, 2], device), torch.randn(2, 4 * 64, device=device)
    want = dfattn.kv8_attention(cache, q, table, start, seq, 4, 1, 2500)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = [dfattn.kv8_attention(cache, q, table, start, seq, 4, 1, 2500, stream=s) for _ in range(4)]
    other = [torch.zeros(1 << 20, device=device) for _ in range(8)]  # (the main stream allocates meanwhile)
    s.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))
    del other


def test_wrapper_refusals(device):
    cache = dfattn.kv8_cache(2, 2, 64, 16, device=device)
    k = torch.zeros(3, 128, device=device)
    slots = i32([0, 1, 2], device)
    with pytest.raises(ValueError):
        dfattn.kv8_append(cache, k, k.bfloat16(), slots)
    with pytest.raises(ValueError):
        dfattn.kv8_append(cache, k.double(), k.double(), slots)
    with pytest.raises(ValueError):
        dfattn.kv8_append(cache, k, k, slots.long())
    with pytest.raises(ValueError):
        dfattn.kv8_append(cache, k, k, slots[:2])
    with pytest.raises(ValueError):
        dfattn.kv8_append(cache, k[:, :64], k[:, :64], slots)
    with pytest.raises(ValueError):
        dfattn.kv8_append(cache, k.t().contiguous().t(), k, slots)
    with pytest.raises(ValueError):
        dfattn.kv8_read(cache, slots, 32)
    with pytest.raises(ValueError):
        dfattn.kv8_attention(cache, k, i32([[0]], device), i32([0], device), i32([3], device), 2, 3, 3)
    with pytest.raises(ValueError):
        dfattn.kv8_attention(cache, k, i32([[0]], device), i32([0, 3], device), i32([3], device), 2, 3, 3,
                             out=torch.empty(3, 64, device=device))
    with pytest.raises(dfattn.DfattnError):
        dfattn.kv8_attention(cache, torch.zeros(3, 3 * 64, device=device), i32([[0]], device), i32([0, 3], device),
                             i32([3], device), 3, 3, 3)


def test_a_stream_of_another_device_is_refused(device):
    class Elsewhere:
        device_index, cuda_stream = torch.cuda.current_device() + 1, 0

    cache = dfattn.kv8_cache(2, 2, 64, 16, device=device)
    x, slots, start = torch.zeros(1, 128, device=device), i32([0], device), i32([0, 1], device)
    table, one = i32([[0, 1]], device), i32([1], device)
    for call in (lambda: dfattn.kv8_append(cache, x, x, slots, stream=Elsewhere),
                 lambda: dfattn.kv8_read(cache, slots, 64, stream=Elsewhere),
                 lambda: dfattn.kv8_attention(cache, x, table, start, one, 2, 1, 1, stream=Elsewhere),
                 lambda: dfattn.paged_plan(one, one, table, slots, slots, 16, 2, 4, stream=Elsewhere)):
        with pytest.raises(ValueError):
            call()
