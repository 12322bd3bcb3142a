"""The paged 8-bit cache's operators in float64 on the CPU, straight from their definitions: plan, append
(with its scales), and attention with the bound that its rounding may reach."""
import math

import numpy as np
import torch

LIMIT = {"i8": 127.0, "e4m3": 448.0}
DTYPE = {"i8": torch.int8, "e4m3": torch.float8_e4m3fn}
ACT = {"f32": torch.float32, "bf16": torch.bfloat16}


def pow2_scale(amax, fmt):
    """The smallest power of two s >= 2^-126 with amax <= LIMIT * s."""
    e = -126
    if amax > 0:
        e = max(-126, math.frexp(amax)[1] - 10)
        while amax > LIMIT[fmt] * math.ldexp(1.0, e):
            e += 1
    return math.ldexp(1.0, e)


def round_code(y, fmt):
    if fmt == "i8":
        return np.round(y)  # ties to even
    step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -6))) - 3)
    return np.round(y / step) * step


class Cache:
    """values[page, kv head, row, d] and scale[page, kv head] of K or V, in float64."""

    def __init__(self, pages, heads, page, d, fmt):
        self.fmt, self.p = fmt, page
        self.codes, self.scale = np.zeros((pages, heads, page, d)), np.zeros((pages, heads))

    def append(self, x, slots):
        """x [n, heads, d] (float64) into the slots, runs of one page consecutive."""
        pages = len(self.codes)
        i, n = 0, len(slots)
        while i < n:
            page, off = divmod(int(slots[i]), self.p)
            if not 0 <= slots[i] < pages * self.p:
                i += 1
                continue
            j = i + 1
            while j < n and slots[j] == slots[j - 1] + 1 and slots[j] % self.p:
                j += 1
            for h in range(self.codes.shape[1]):
                rows = x[i:j, h]
                old = self.scale[page, h] if off else 0.0
                if not np.all(np.isfinite(rows)) or np.isnan(old):
                    s = np.nan
                    self.codes[page, h, :off + j - i] = 0
                else:
                    s = max(pow2_scale(float(np.abs(rows).max()), self.fmt), old)
                    self.codes[page, h, off:off + j - i] = round_code(rows / s, self.fmt)
                    if off:
                        self.codes[page, h, :off] = round_code(self.codes[page, h, :off] * (old / s), self.fmt)
                self.scale[page, h] = s
            i = j

    def read(self, slots):
        out = np.zeros((len(slots), self.codes.shape[1], self.codes.shape[3]))
        for i, s in enumerate(slots):
            if 0 <= s < len(self.codes) * self.p:
                page, off = divmod(int(s), self.p)
                out[i] = self.codes[page, :, off] * self.scale[page][:, None]
        return out.reshape(len(slots), -1)


def plan(cached, new, table, free, free_start, page, n_pages, capacity):
    """dfattn_paged_plan, one request after the other."""
    table, r, width = table.copy(), len(cached), table.shape[1]
    seq, start, slots, taken = list(cached), [0], [], free_start
    admitted, open_ = 0, True
    for i in range(r):
        had, want = -(-cached[i] // page), -(-(cached[i] + new[i]) // page)
        open_ = open_ and cached[i] + new[i] <= width * page and taken + want - had <= len(free) and \
            start[-1] + new[i] <= capacity
        if open_:
            admitted += 1
            table[i, had:want] = free[taken:taken + want - had]
            taken += want - had
            seq[i] = cached[i] + new[i]
            for t in range(cached[i], seq[i]):
                p = int(table[i, t // page])
                slots.append(p * page + t % page if 0 <= p < n_pages else -1)
        start.append(len(slots))
    return {"table": table, "seq_lens": np.array(seq), "query_start": np.array(start),
            "slots": np.array(slots + [-1] * (capacity - len(slots))), "counts": np.array([admitted, len(slots), taken])}


def attention(q, k_of, v_of, query_start, seq_lens, heads, kv_heads, d, scale, causal, n_rows, u, out_step, page):
    """(out, lse, bound of out, bound of lse), float64. k_of(r), v_of(r): the request's cached values [L, kv heads,
    d], a position in a bad page NaN-free and listed in neither (None rows are left out by the caller's mask). u:
    the relative rounding of one operand of a product; out_step: half a step of the output type.

    The bound: a score is off by e = scale sum|q||k| (u + (d + 4) 2^-24) (its operands' rounding and its sum's), and
    by 2^-22 of the largest score's size for its scaling by log2 e and the difference from the maximum; a
    probability by twice that, 2^-22 for the exponential, u for its own rounding; a sum of L products by L 2^-24.
    The smallest numbers: what is multiplied with a code is w = p * scale(page), as fp16 terms whose smallest step
    is 2^-24 and whose largest value lies at 2^14 or above, so a weight may also be off by 2^-39 of the largest
    one, whatever its own size. A scale is below 2 amax(page) / LIMIT and a code at most LIMIT, so the sum over L
    positions is off by at most L 2^-39 LIMIT max(p 2 amax(page) / LIMIT) = L 2^-38 max(p amax(page)). (fp32's own
    smallest number, 2^-126, is far below that.)"""
    out, lse = np.zeros((n_rows, heads, d)), np.full((heads, n_rows), -np.inf)
    tol, ltol = np.zeros_like(out), np.zeros_like(lse)
    for r in range(len(seq_lens)):
        a, b = int(query_start[r]), int(query_start[r + 1])
        kr, vr, ok = k_of(r)[0], v_of(r)[0], k_of(r)[1]
        length = int(seq_lens[r])
        amax = np.array([np.abs(vr[t // page * page:t // page * page + page]).max((0, 2)) for t in range(len(vr))])
        for j in range(b - a):
            last = min(length, length - (b - a) + j + 1) if causal else length
            see = np.nonzero(ok[:max(last, 0)])[0]
            if not len(see):
                continue
            for h in range(heads):
                hk = h // (heads // kv_heads)
                x = q[a + j, h * d:(h + 1) * d]
                kk, vv = kr[see, hk], vr[see, hk]
                s = scale * (kk @ x)
                m = s.max()
                e = np.exp(s - m)
                p = e / e.sum()
                out[a + j, h] = p @ vv
                lse[h, a + j] = m + np.log(e.sum())
                err = abs(scale) * (np.abs(kk) @ np.abs(x)).max() * (u + (d + 4) * 2.0 ** -24) + \
                    2.0 ** -22 * max(1.0, np.abs(s).max())
                tol[a + j, h] = (p @ np.abs(vv)) * (2 * err + 2.0 ** -22 + u + (len(see) + 8) * 2.0 ** -24) + \
                    np.abs(out[a + j, h]) * out_step + len(see) * 2.0 ** -38 * (p * amax[see, hk]).max()
                ltol[h, a + j] = err + (len(see) + 8) * 2.0 ** -24 + 2.0 ** -22 * abs(lse[h, a + j])
    return out.reshape(n_rows, -1), lse, tol.reshape(n_rows, -1), ltol
