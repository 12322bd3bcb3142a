"""The paged 8-bit cache at the limits of its numbers, against float64 (kv8_reference.py): pages whose scales lie far
apart, infinities and NaN beside rows that do not see them, slots that do not follow each other, scores up to
2^100."""
import math

import numpy as np
import pytest
import torch

import dfattn
import kv8_reference as ref

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


def i32(x, device):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=device)


def filled(device, k, v, page, fmt, seed):
    """A cache that holds k and v [n, heads, d] of one request in scattered pages: (cache, table, K and V as the cache has
    them, float64)."""
    n, heads, d = k.shape
    pages = -(-n // page)
    table = np.random.RandomState(seed).permutation(pages)
    cache = dfattn.kv8_cache(pages, heads, d, page, ref.DTYPE[fmt], device)
    pos = np.arange(n)
    slots = i32(table[pos // page] * page + pos % page, device)
    dfattn.kv8_append(cache, *(torch.tensor(x.reshape(n, -1), dtype=torch.float32, device=device) for x in (k, v)), slots)
    kr, vr = (x.double().cpu().numpy().reshape(n, heads, d) for x in dfattn.kv8_read(cache, slots, d))
    return cache, i32(table[None], device), kr, vr


# ---------------------------------------------------------------- pages whose scales lie far apart
FAR = [
    # cached, queries, heads, kv heads, d, page
    (77, 1, 2, 2, 64, 16),
    (77, 30, 2, 2, 64, 16),      # every part of the pages masked
    (300, 20, 4, 2, 128, 32),
    (3000, 1, 2, 2, 64, 16),     # cut between workgroups
    (1300, 20, 2, 1, 128, 64),   # ... with more columns
    (1200, 200, 1, 1, 64, 16),   # ... 48 of them
    (20000, 1, 1, 1, 16, 16),    # ... in more pieces than one wave of the merge takes
]


@pytest.mark.parametrize("fmt,act", [("i8", "f32"), ("e4m3", "bf16"), ("e4m3", "f32"), ("i8", "bf16")])
@pytest.mark.parametrize("case", range(len(FAR)))
def test_scales_far_apart(device, case, fmt, act):
    """The largest score in pages of zeros or tiny values (whose scale is 2^-126 or near it), the other pages' scores
    `gap` below it and their values up to 2^121 times larger: their weights, far below fp32's smallest number, may
    still be what counts.

    The bound is kv8_reference's and what fp32 and bf16 lose below their normal numbers, half of 2^-149 at a time: each
    of the four waves of at most 64 pieces once, and each piece once in the merge, times its sum of probabilities,
    which all together are at most n; bf16 half of its 2^-133."""
    n, nq, heads, kv_heads, d, page = FAR[case]
    for low, high in ((None, 0), (None, 100), (-121, 0), (-20, 100)):
        rng = np.random.RandomState(case)
        small = np.isin(np.arange(n) // page, (1, -(-n // page) // 2))
        k, v = (rng.randn(n, kv_heads, d) for _ in range(2))
        k[:, :, 0] = np.where(small, 4.0, 0.0)[:, None]
        v *= np.where(small, 0.0 if low is None else 2.0 ** low, 2.0 ** high)[:, None, None]
        cache, table, kr, vr = filled(device, k, v, page, fmt, case)
        for gap in (60.0, 80.0, 110.0, 200.0):
            say("far apart", FAR[case], fmt, act, low, high, gap)
            q = 0.1 * rng.randn(nq, heads, d)
            q[:, :, 0] = gap / 4
            q = torch.tensor(q.reshape(nq, -1), device=device).to(ref.ACT[act])
            ok = np.ones(n, bool)
            want, wlse, tol, ltol = ref.attention(
                q.double().cpu().numpy(), lambda r: (kr, ok), lambda r: (vr, ok), [0, nq], [n], heads, kv_heads, d, 1.0,
                True, nq, 2.0 ** -22 if act == "f32" else 2.0 ** -11, 0.0 if act == "f32" else 2.0 ** -8, page)
            tol += (n + 256) * 2.0 ** -150 + (0.0 if act == "f32" else 2.0 ** -134)
            for workspace in ("auto", None):
                out, lse = dfattn.kv8_attention(cache, q, table, i32([0, nq], device), i32([n], device), heads, nq, n, 1.0,
                                                workspace=workspace)
                err = np.abs(out.double().cpu().numpy() - want)
                assert (err <= tol).all(), (low, high, gap, float(np.nanmax(err / tol)), bool(np.isnan(err).any()))
                assert (np.abs(lse.double().cpu().numpy() - wlse) <= ltol).all()


# ---------------------------------------------------------------- infinities and NaN
UNSEEN = [
    # cached, queries, heads, kv heads, d, page, the bad position
    (40, 16, 2, 2, 64, 16, 36),      # 16 columns
    (70, 70, 2, 2, 64, 16, 20),      # 32
    (70, 70, 2, 2, 64, 16, 50),
    (70, 35, 4, 2, 128, 32, 66),
    (230, 230, 2, 2, 64, 16, 19),    # 48
    (230, 230, 2, 2, 33, 16, 215),
    (1300, 20, 2, 2, 64, 16, 1290),  # tiles cut between workgroups
    (1300, 200, 2, 2, 64, 16, 1205),
    (1300, 80, 2, 2, 100, 48, 1280),
]


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("case", range(len(UNSEEN)))
def test_rows_that_do_not_see_a_bad_page(device, case, bad, fmt):
    """Queries before a page of NaN, in one tile with queries behind it, get what they get without it, bit for bit;
    the page's head gives NaN to those that see it, the other head nothing. So it stays when rows are added."""
    n, nq, heads, kv_heads, d, page, at = UNSEEN[case]
    say("unseen", UNSEEN[case], bad, fmt)
    rng = np.random.RandomState(case)
    k, v = (rng.randn(n, kv_heads, d) for _ in range(2))
    start, seq = i32([0, nq], device), i32([n], device)
    for act in (torch.float32, torch.bfloat16):
        q = torch.tensor(rng.randn(nq, heads * d), device=device).to(act)
        for in_k, in_v in ((False, True), (True, False), (True, True)):
            for later in (False, True):
                got = []
                for x in (0.0, bad):
                    kx, vx = k.copy(), v.copy()
                    if in_k:
                        kx[at, 1, d // 3] = x
                    if in_v:
                        vx[at, 1, d // 2] = x
                    first = at + 1 if later else n  # (the rest comes in a call of its own, behind the bad row)
                    pos = np.arange(n)
                    cache = dfattn.kv8_cache(-(-n // page), kv_heads, d, page, ref.DTYPE[fmt], device)
                    for a, b in ((0, first), (first, n)):
                        dfattn.kv8_append(cache, *(torch.tensor(y[a:b].reshape(b - a, kv_heads * d), dtype=torch.float32, device=device)
                                                   for y in (kx, vx)), i32(pos[a:b], device))
                    got.append(dfattn.kv8_attention(cache, q, i32([range(-(-n // page))], device), start, seq, heads, nq, n))
                (want, wlse), (out, lse) = got
                assert torch.isfinite(want).all()
                sees = torch.arange(n - nq, n, device=device) >= at // page * page
                group = torch.arange(heads, device=device) // (heads // kv_heads) == 1
                hit = sees[:, None] & group[None, :]
                bits = out.view(nq, heads, d)
                assert torch.isnan(bits[hit]).all() and torch.equal(bits[~hit], want.view(nq, heads, d)[~hit])
                assert torch.isnan(lse.t()[hit]).all() if in_k else torch.equal(lse, wlse)
                assert torch.equal(lse.t()[~hit], wlse.t()[~hit])


# ---------------------------------------------------------------- slots that do not follow each other
JUMPS = [[3, 5, 6], [3, 3], [5, 3], [2, 4, 6], [7, 8, 9, 12, 13], [0, 2], [15, 0]]


@pytest.mark.parametrize("fmt,act", [("i8", "f32"), ("e4m3", "bf16")])
@pytest.mark.parametrize("heads,d,page", [(2, 64, 16), (12, 100, 32), (2, 33, 64)])
@pytest.mark.parametrize("ahead", [0, 43, 44, 45, 46, 47, 48, 61, 62, 63, 64])
def test_append_of_slots_that_jump(device, ahead, heads, d, page, fmt, act):
    """A row whose slot does not follow the one before it in the same page is left out with those that follow it: the
    page's rows up to there, and every other page, hold what they hold without them."""
    say("jump", ahead, heads, d, page, fmt, act)
    rng = np.random.RandomState(ahead)
    pages = ahead + len(JUMPS)
    cache = dfattn.kv8_cache(pages, heads, d, page, ref.DTYPE[fmt], device)
    refs = [ref.Cache(pages, heads, page, d, fmt) for _ in range(2)]
    base = [(ahead + i) * page for i in range(len(JUMPS))]
    calls = [[b + o for b in base for o in range(page)]]                    # whole pages
    calls.append([i * page for i in range(ahead)] + [b + o for b, jump in zip(base, JUMPS) for o in jump])
    written = [[s for s in calls[0]], [i * page for i in range(ahead)]]
    for b, jump in zip(base, JUMPS):
        n = next((j for j in range(1, len(jump)) if jump[j] != jump[j - 1] + 1), len(jump))
        written[1] += [b + o for o in jump[:n]] + [-1] * (len(jump) - n)
    for n, (slots, kept) in enumerate(zip(calls, written)):
        k, v = (torch.tensor(rng.randn(len(slots), heads * d) * 4.0 ** n, device=device).to(ref.ACT[act]) for _ in range(2))
        for r, x in zip(refs, (k, v)):
            r.append(x.double().cpu().numpy().reshape(len(slots), heads, d), kept)
        dfattn.kv8_append(cache, k, v, i32(slots, device))
    at = [i * page for i in range(ahead)]
    for b, jump in zip(base, JUMPS):
        n = next(j for j in range(1, len(jump)) if jump[j] != jump[j - 1] + 1)
        at += [b + o for o in range(jump[n - 1] + 1)]
    for g, w in zip(dfattn.kv8_read(cache, i32(at, device), d), refs):
        assert np.array_equal(g.double().cpu().numpy(), w.read(at))
    for t, w in zip(cache[2:], refs):
        assert np.array_equal(t.double().cpu().numpy(), w.scale)


# ---------------------------------------------------------------- large scores
@pytest.mark.parametrize("fmt,act", [("i8", "f32"), ("e4m3", "bf16"), ("e4m3", "f32"), ("i8", "bf16")])
@pytest.mark.parametrize("power", [16, 21, 24, 27, 30, 40, 60, 100])
def test_large_scores(device, power, fmt, act):
    """Scores of about 2^power, of either sign: each row's largest two keys are the same and lie far above the others, so
    that the output is the mean of their values and lse the score and ln 2.

    The bound: a score's products and sums are off by (u + (d + 4) 2^-24) sum|q||k| alike for the two, so their
    weights are both 1 but for the exponential's 2^-22; the values' sum is fp32's of fp16 terms (u). lse is off by what
    the score is, and 2^-22 of its size."""
    heads, d, page = 2, 64, 16
    u = 2.0 ** -22 if act == "f32" else 2.0 ** -11
    step = 0.0 if act == "f32" else 2.0 ** -8
    for n, nq in ((70, 1), (70, 20), (3000, 1), (1300, 200), (300, 300)):
        for sign in (1.0, -1.0):
            say("large scores", power, fmt, act, n, nq, sign)
            rng = np.random.RandomState(power)
            k, v = (rng.randn(n, heads, d) for _ in range(2))
            k[:, :, 0] = np.where(np.arange(n) == 3, -1.0, -3.0)[:, None]  # all scores of one sign, key 3's next to 0
            twins = [0, n - nq - 1 if nq < n else 1]
            k[twins[1]] = k[twins[0]]
            k[twins, :, 0] = 4.0
            k[:, :, 1:] *= 2.0 ** -6
            if sign < 0:  # (all scores negative, the twins' the least so)
                k[:, :, 0] = -6.0
                k[3, :, 0] = -5.0
                k[twins, :, 0] = -1.0
            cache, table, kr, vr = filled(device, k, v, page, fmt, power)
            q = rng.randn(nq, heads, d) * 2.0 ** -6
            q[:, :, 0] = rng.uniform(1, 2, (nq, heads))
            q = torch.tensor(q.reshape(nq, -1), device=device).to(ref.ACT[act])
            qd = q.double().cpu().numpy().reshape(nq, heads, d)
            same = np.array_equal(kr[twins[0]], kr[twins[1]])
            scale = 2.0 ** power
            out, lse = dfattn.kv8_attention(cache, q, table, i32([0, nq], device), i32([n], device), heads, nq, n, scale)
            out, lse = out.double().cpu().numpy().reshape(nq, heads, d), lse.double().cpu().numpy()
            assert np.isfinite(out).all() and np.isfinite(lse).all()
            for j in range(nq):
                see = n - nq + j + 1
                for h in range(heads):
                    x = scale * (kr[:see, h] @ qd[j, h])
                    err = scale * (np.abs(kr[:see, h]) @ np.abs(qd[j, h])).max() * (u + (d + 4) * 2.0 ** -24)
                    err += 2.0 ** -22 * np.abs(x).max()
                    top = np.nonzero(x >= x.max() - 2 * err - 60)[0]
                    assert abs(lse[h, j] - x.max()) <= err + np.log(len(top)) + 1e-5
                    if len(top) == 1 or (same and list(top) == twins):
                        want = vr[top, h].mean(0)
                        tol = np.abs(vr[top, h]).mean(0) * (2.0 ** -20 + u + step) + 2.0 ** -38 * np.abs(vr[:, h]).max()
                        assert (np.abs(out[j, h] - want) <= tol).all(), (j, h, top)
                    else:  # (a value between those of the keys that cannot be told apart)
                        lo, hi = vr[top, h].min(0), vr[top, h].max(0)
                        slack = (np.abs(lo) + np.abs(hi)) * (2.0 ** -20 + u + step) + 1e-6
                        assert (out[j, h] >= lo - slack).all() and (out[j, h] <= hi + slack).all()
