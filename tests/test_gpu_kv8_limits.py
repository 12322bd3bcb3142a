"""The paged 8-bit cache at the limits of its numbers, against float64 (kv8_reference.py): pages whose scales lie far
apart."""
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
