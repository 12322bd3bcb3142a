"""The serving operators' performance cases: paged tables built on the device, the 8-bit paged cache
(append, read back, attention) and the log probabilities of given tokens with their gradient.

listed() names twelve calls, draw() gives more of the same ranges. prepare() makes what a program has
in hand before the call, run() is one pass: in plain torch operations, or, where `own` is true, through
the library's entry points. exact() gives the same results in 64 bits.

Cache layout: codes K [pages, kv heads, page size, Dp] and V [pages, kv heads, Dp, page size] (Dp: the
head size rounded up to 16), one scale per page and kv head for each; value = code * scale.
"""
import math
import os
import sys

import torch

DEVICE = "cuda"
own = False

FORMATS = {"i8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # One step's tables for a small batch of generating requests: one new token each.
        {"name": "plan_decode_r48", "kind": "plan", "requests": 48, "cached": 1000, "new": 1, "page": 16,
         "capacity": 64, "short": False},
        # A step that admits many prompts of mixed lengths beside generating requests.
        {"name": "plan_mixed_r500", "kind": "plan", "requests": 500, "cached": 2000, "new": 160, "page": 16,
         "capacity": 65536, "short": False},
        # The new keys and values of one layer for 40 generating requests, and the cache read back.
        {"name": "append_decode_r40_h12_d64", "kind": "append", "requests": 40, "cached": 40, "new": 1, "page": 16,
         "kv_heads": 12, "d_head": 64, "fmt": "i8", "act": "f32"},
        # Prompts of odd lengths written into the cache of one layer (shared heads of 128), and read back.
        {"name": "append_prompts_t8197_h8_d128", "kind": "append", "requests": 7, "cached": 100, "new": 1171,
         "page": 32, "kv_heads": 8, "d_head": 128, "fmt": "e4m3", "act": "bf16"},
        # One generated token of one request over a cache of GPT-2's length: latency.
        {"name": "decode_r1_l1024_h12_d64", "kind": "attention", "requests": 1, "low": 1024, "high": 1024, "q": 1,
         "page": 16, "heads": 12, "kv_heads": 12, "d_head": 64, "fmt": "i8", "act": "f32"},
        # A generating batch with ragged lengths, bf16 activations.
        {"name": "decode_r64_l4096_h12_d64_bf16", "kind": "attention", "requests": 64, "low": 100, "high": 4096,
         "q": 1, "page": 16, "heads": 12, "kv_heads": 12, "d_head": 64, "fmt": "e4m3", "act": "bf16"},
        # Long contexts, few rows: the benchmark's longest sequence.
        {"name": "decode_r2_l131072_h12_d64", "kind": "attention", "requests": 2, "low": 65000, "high": 131072,
         "q": 1, "page": 64, "heads": 12, "kv_heads": 12, "d_head": 64, "fmt": "i8", "act": "f32"},
        # Shared key and value heads of 128, the usual shape of larger models.
        {"name": "decode_r32_l8192_h32_8_d128", "kind": "attention", "requests": 32, "low": 500, "high": 8192,
         "q": 1, "page": 32, "heads": 32, "kv_heads": 8, "d_head": 128, "fmt": "i8", "act": "bf16"},
        # Chunks of prompts against what the cache already holds.
        {"name": "chunk_r3_q500_l4096_h12_d64", "kind": "attention", "requests": 3, "low": 900, "high": 4096,
         "q": 500, "page": 16, "heads": 12, "kv_heads": 12, "d_head": 64, "fmt": "e4m3", "act": "f32"},
        # What an answer's tokens return: a small batch's log probabilities with five alternatives.
        {"name": "logprobs_r8_v50257_k5", "kind": "logprobs", "rows": 8, "vocab": 50257, "top": 5, "type": "f32"},
        # Scoring given texts, with twenty alternatives, bf16 logits.
        {"name": "logprobs_r2048_v50257_k20_bf16", "kind": "logprobs", "rows": 2048, "vocab": 50257, "top": 20,
         "type": "bf16"},
        # Training on the log probabilities and an entropy bonus: forward and the logits' gradient.
        {"name": "logprobs_grad_r1000_v50257", "kind": "logprobs_grad", "rows": 1000, "vocab": 50257, "top": 0,
         "type": "f32"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choices(("plan", "append", "attention", "logprobs", "logprobs_grad"), weights=(14, 20, 40, 16, 10))[0]
    if kind == "plan":
        requests = _log_int(rng, 1, 2000)
        new = 1 if rng.random() < 0.5 else _log_int(rng, 2, max(2, 60000 // requests))
        return {"kind": kind, "requests": requests, "cached": _log_int(rng, 1, 4000), "new": new,
                "page": rng.choice((16, 32, 64, 128)), "capacity": requests * new + rng.randint(0, 1000),
                "short": rng.random() < 0.3}
    if kind == "append":
        kv_heads, d_head = rng.choice((1, 2, 4, 8, 12, 16)), rng.choice((32, 64, 64, 80, 100, 128))
        most = min(8000, (1 << 23) // (kv_heads * d_head))
        requests = _log_int(rng, 1, 200)
        new = 1 if rng.random() < 0.5 else _log_int(rng, 2, max(2, most // requests))
        return {"kind": kind, "requests": requests, "cached": _log_int(rng, 1, 60), "new": new,
                "page": rng.choice((16, 16, 32, 64, 128)), "kv_heads": kv_heads, "d_head": d_head,
                "fmt": rng.choice(("i8", "e4m3")), "act": rng.choice(("f32", "bf16"))}
    if kind == "attention":
        group, d_head = rng.choice((1, 1, 1, 2, 4, 8)), rng.choice((32, 64, 64, 64, 80, 100, 128, 128))
        kv_heads = rng.choice((1, 2, 4, 8, 12))
        c = {"kind": kind, "page": rng.choice((16, 16, 32, 64, 128)), "heads": group * kv_heads,
             "kv_heads": kv_heads, "d_head": d_head, "fmt": rng.choice(("i8", "e4m3")),
             "act": rng.choice(("f32", "bf16"))}
        width = 2 * kv_heads * d_head
        if rng.random() < 0.75:  # generating: one token a request
            high = _log_int(rng, 64, 131072)
            most = max(1, min(128, 300_000_000 // (width * high)))
            return {**c, "requests": _log_int(rng, 1, most), "low": rng.randint(1, high), "high": high, "q": 1}
        q = rng.choice((2, 5)) if rng.random() < 0.4 else _log_int(rng, 16, 700)
        high = _log_int(rng, max(64, q), 4096)
        most = max(1, min(16, 4_500_000_000 // (c["heads"] * d_head * q * high)))
        return {**c, "requests": _log_int(rng, 1, most), "low": rng.randint(q, high), "high": high, "q": q}
    vocab = _log_int(rng, 1000, 131072)
    rows = _log_int(rng, 1, min(4096, 50_000_000 // vocab))
    return {"kind": kind, "rows": rows, "vocab": vocab, "top": rng.randint(0, 20) if kind == "logprobs" else 0,
            "type": rng.choice(("f32", "bf16"))}


# ---------------------------------------------------------------- sizes that follow from a case
def _pad16(d):
    return -(-d // 16) * 16


def _lengths(c):
    """The cached lengths of an attention case: evenly spread from low to high."""
    r = c["requests"]
    if r == 1:
        return [c["high"]]
    return [c["low"] + round(i * (c["high"] - c["low"]) / (r - 1)) for i in range(r)]


def _spread(most, n):
    """n lengths from 1 to 2 * most - 1 (all `most` where it is 1), `most` on average."""
    return [most if n == 1 or most == 1 else 1 + round(i * (2 * most - 2) / (n - 1)) for i in range(n)]


# ---------------------------------------------------------------- inputs, from the seed alone
def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE)


def _shuffled(g, values):
    t = torch.tensor(values, dtype=torch.int32, device=DEVICE)
    return t[torch.randperm(len(values), generator=g, device=DEVICE)].contiguous()


def _activations(g, rows, heads, d):
    """Keys or queries as layers give them: a few channels of a head larger than the others."""
    x = _randn(g, rows, heads, d)
    x[:, :, :: 16] *= 3.0
    return x.view(rows, heads * d)


def _pow2(amax, limit):
    """The smallest power of two s >= 2^-126 with amax <= limit * s, exactly."""
    m, e = torch.frexp(amax.float())
    top, bits = math.frexp(limit)
    e = torch.clamp(e - bits + (m > top).to(e.dtype), min=-126)
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _codes(x, scale, fmt):
    y = x / scale
    return (torch.round(y) if fmt == "i8" else y).to(FORMATS[fmt][0])


def _filled_cache(g, pages, c):
    """A cache whose pages all hold values: random ones of the usual spread, each page and head at its scale."""
    hk, d, p = c["kv_heads"], c["d_head"], c["page"]
    dp, dtype = _pad16(d), FORMATS[c["fmt"]][0]
    k = torch.zeros(pages, hk, p, dp, dtype=torch.int8, device=DEVICE).view(dtype)
    v = torch.zeros(pages, hk, dp, p, dtype=torch.int8, device=DEVICE).view(dtype)
    ks, vs = (torch.zeros(pages, hk, device=DEVICE) for _ in range(2))
    step = max(1, (1 << 26) // (hk * p * dp))
    for a in range(0, pages, step):
        n = min(step, pages - a)
        x = _randn(g, n, hk, p, d)
        x[..., :: 16] *= 3.0
        ks[a:a + n] = _pow2(x.abs().amax((2, 3)), FORMATS[c["fmt"]][1])
        k.view(torch.int8)[a:a + n, :, :, :d] = _codes(x, ks[a:a + n, :, None, None], c["fmt"]).view(torch.int8)
        x = _randn(g, n, hk, d, p)
        vs[a:a + n] = _pow2(x.abs().amax((2, 3)), FORMATS[c["fmt"]][1])
        v.view(torch.int8)[a:a + n, :, :d] = _codes(x, vs[a:a + n, :, None, None], c["fmt"]).view(torch.int8)
    return k, v, ks, vs


def _plan_inputs(c, seed):
    g, r, p = _generator(seed), c["requests"], c["page"]
    cached, new = _shuffled(g, _spread(c["cached"], r)), _shuffled(g, _spread(c["new"], r))
    pages_had = (cached + p - 1) // p
    pages_need = (cached + new + p - 1) // p - pages_had
    width = -(-(2 * c["cached"] + 2 * c["new"]) // p)
    had, need = int(pages_had.sum()), int(pages_need.sum())
    free_start = int(torch.randint(0, 50, (1,), generator=g, device=DEVICE))
    n_free = free_start + (need * 2 // 3 if c["short"] else need + 7)
    order = torch.randperm(had + n_free, generator=g, device=DEVICE).int()
    table = torch.full((r, width), -1, dtype=torch.int32, device=DEVICE)
    holds = torch.arange(width, device=DEVICE)[None, :] < pages_had[:, None]
    table[holds] = order[:had]
    return {"cached": cached, "new": new, "table": table, "free": order[had:].contiguous(),
            "free_start": torch.tensor([free_start], dtype=torch.int32, device=DEVICE), "n_pages": had + n_free,
            "page": p, "capacity": c["capacity"]}


def _append_inputs(c, seed):
    g, r, p, hk, d = _generator(seed), c["requests"], c["page"], c["kv_heads"], c["d_head"]
    cached, new = _shuffled(g, _spread(c["cached"], r)).long(), _shuffled(g, _spread(c["new"], r)).long()
    start = cached % p  # rows of the last page that hold tokens already; full pages stay outside the call
    pages = (start + new + p - 1) // p
    first = torch.cumsum(pages, 0) - pages
    n_pages = int(pages.sum())
    order = torch.randperm(n_pages, generator=g, device=DEVICE)
    cache = _filled_cache(g, n_pages, c)
    for t in cache[2:]:  # the rows already there are smaller than the new ones in some pages: their scale grows
        t *= torch.exp2(-torch.randint(0, 3, t.shape, generator=g, device=DEVICE).float())

    def slots(begin, count):
        total = int(count.sum())
        which = torch.repeat_interleave(torch.arange(r, device=DEVICE), count)
        at = torch.arange(total, device=DEVICE) - torch.repeat_interleave(torch.cumsum(count, 0) - count, count)
        row = begin[which] + at
        return (order[first[which] + row // p] * p + row % p).int()

    act = TYPES[c["act"]]
    n = int(new.sum())
    return {"cache": cache, "slots": slots(start, new), "all": slots(torch.zeros_like(start), start + new),
            "k": _activations(g, n, hk, d).to(act), "v": _randn(g, n, hk * d).to(act), "d_head": d, "fmt": c["fmt"]}


def _attention_inputs(c, seed):
    g, r, p, d = _generator(seed), c["requests"], c["page"], c["d_head"]
    lens = _shuffled(g, _lengths(c))
    width = -(-c["high"] // p)
    pages = (lens.long() + p - 1) // p
    n_pages = int(pages.sum())
    table = torch.full((r, width), -1, dtype=torch.int32, device=DEVICE)
    table[torch.arange(width, device=DEVICE)[None, :] < pages[:, None]] = \
        torch.randperm(n_pages, generator=g, device=DEVICE).int()
    n = r * c["q"]
    q = (1.5 * _randn(g, n, c["heads"] * d)).to(TYPES[c["act"]])
    return {"q": q, "cache": _filled_cache(g, n_pages, c), "table": table, "seq_lens": lens,
            "query_start": torch.arange(0, n + 1, c["q"], dtype=torch.int32, device=DEVICE), "heads": c["heads"],
            "d_head": d, "max_q": c["q"], "max_len": c["high"], "scale": d ** -0.5, "fmt": c["fmt"]}


def _logprobs_inputs(c, seed):
    g, (r, v) = _generator(seed), (c["rows"], c["vocab"])
    x = 2.0 * _randn(g, r, v)
    u = torch.rand(r, generator=g, device=DEVICE, dtype=torch.float64)
    tokens = (torch.exp(u * math.log(v + 1.0)) - 1.0).long().clamp_(0, v - 1)
    x[torch.arange(r, device=DEVICE), tokens] += 6.0  # a model mostly expects the token that comes
    s = {"logits": x.to(TYPES[c["type"]]), "tokens": tokens.int(), "top": c["top"], "grad": c["kind"] == "logprobs_grad"}
    if s["grad"]:
        s["g_logprob"], s["g_entropy"] = _randn(g, r) / r, -0.01 / r * torch.ones(r, device=DEVICE)
    return s


_INPUTS = {"plan": _plan_inputs, "append": _append_inputs, "attention": _attention_inputs,
           "logprobs": _logprobs_inputs, "logprobs_grad": _logprobs_inputs}


def prepare(case, seed):
    return {"kind": case["kind"], **_INPUTS[case["kind"]](case, seed)}


# ---------------------------------------------------------------- the operators in plain form
def _plan_plain(s):
    p, table, cap = s["page"], s["table"].long(), s["capacity"]
    cached, new, width = s["cached"].long(), s["new"].long(), s["table"].shape[1]
    had = (cached + p - 1) // p
    need = (cached + new + p - 1) // p - had
    free = s["free"].numel() - s["free_start"].long()
    fits = ((cached + new) <= width * p) & (torch.cumsum(need, 0) <= free) & (torch.cumsum(new, 0) <= cap)
    in_ = torch.cumprod(fits.long(), 0)
    new, need = new * in_, need * in_
    start = torch.cat([torch.zeros_like(new[:1]), torch.cumsum(new, 0)])
    before = s["free_start"].long() + torch.cumsum(need, 0) - need
    col = torch.arange(width, device=DEVICE)[None, :]
    fresh = (col >= had[:, None]) & (col < (had + need)[:, None])
    at = (before[:, None] + col - had[:, None]).clamp(0, s["free"].numel() - 1)
    table = torch.where(fresh, s["free"].long()[at], table)
    t = torch.arange(cap, device=DEVICE)
    r = torch.searchsorted(start[1:], t, right=True).clamp(max=new.numel() - 1)
    pos = (cached[r] + t - start[r]).clamp(max=width * p - 1)
    slot = torch.where(t < start[-1], table[r, pos // p] * p + pos % p, torch.full_like(t, -1))
    counts = torch.stack([in_.sum(), start[-1], s["free_start"].long()[0] + need.sum()])
    return {"table": table.int(), "seq_lens": (cached + new).int(), "query_start": start.int(), "slots": slot.int(),
            "counts": counts.int()}


def _plain_values(codes, scale):
    return codes.float() * scale[:, :, None, None]


def _plain_append(k_new, old, old_scale, slots, p, fmt):
    """One side of the cache as values [pages, page size, kv heads, d] after the new rows [n, kv heads, d]."""
    pages = old.shape[0]
    slots = slots.long()
    page, off = slots // p, slots % p
    rows = torch.zeros_like(old).index_put((page, off), k_new.float())
    begin = torch.full((pages,), p, dtype=torch.long, device=DEVICE).scatter_reduce(0, page, off, "amin")
    written = torch.zeros(pages, p, dtype=torch.bool, device=DEVICE).index_put((page, off), torch.ones_like(page, dtype=torch.bool))
    kept = (torch.arange(p, device=DEVICE)[None, :] < begin[:, None])[:, :, None, None]
    scale = _pow2(rows.abs().amax((1, 3)), FORMATS[fmt][1])
    scale = torch.where((begin > 0)[:, None], torch.maximum(scale, old_scale), scale)
    scale = torch.where((begin < p)[:, None], scale, old_scale)[:, None, :, None]
    values = torch.where(kept, old, rows)
    return torch.where(written[:, :, None, None] | kept, _codes(values, scale, fmt).float() * scale, torch.zeros_like(old))


def _append_plain(s):
    k, v, ks, vs = s["cache"]
    p, hk, d = k.shape[2], k.shape[1], s["d_head"]
    old_k = _plain_values(k, ks)[..., :d].transpose(1, 2).contiguous()
    old_v = _plain_values(v, vs)[:, :, :d].permute(0, 3, 1, 2).contiguous()
    new_k = _plain_append(s["k"].view(-1, hk, d), old_k, ks, s["slots"], p, s["fmt"])
    new_v = _plain_append(s["v"].view(-1, hk, d), old_v, vs, s["slots"], p, s["fmt"])
    at = s["all"].long()
    return {"k": new_k.view(-1, hk * d)[at], "v": new_v.view(-1, hk * d)[at]}


def _attention_plain(s):
    k, v, ks, vs = s["cache"]
    hk, p, d, h = k.shape[1], k.shape[2], s["d_head"], s["heads"]
    r, width = s["table"].shape
    table = s["table"].long().clamp(min=0)
    start, lens, n, most = s["query_start"].long(), s["seq_lens"].long(), s["q"].shape[0], s["max_q"]
    kk = k.view(torch.uint8)[table].view(k.dtype).float() * ks[table][..., None, None]  # [r, width, hk, p, dp]
    kk = kk[..., :d].permute(0, 2, 4, 1, 3).reshape(r, hk, d, width * p)
    row = start[:-1, None] + torch.arange(most, device=DEVICE)[None, :]
    q = s["q"].float()[row.clamp(max=n - 1)].view(r, most, hk, h // hk, d).permute(0, 2, 3, 1, 4)
    q = q.reshape(r, hk, (h // hk) * most, d)
    x = torch.matmul(q * s["scale"], kk).view(r, hk, h // hk, most, width * p)
    del kk
    at = lens[:, None] - (start[1:] - start[:-1])[:, None] + torch.arange(most, device=DEVICE)[None, :]
    sees = torch.arange(width * p, device=DEVICE)[None, None, :] <= at[:, :, None]
    x = x.masked_fill(~sees[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True).clamp(min=-3.4e38)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    vv = v.view(torch.uint8)[table].view(v.dtype).float() * vs[table][..., None, None]  # [r, width, hk, dp, p]
    vv = vv[..., :d, :].permute(0, 2, 1, 4, 3).reshape(r, hk, width * p, d)
    in_cache = torch.arange(width * p, device=DEVICE)[None, :] < lens[:, None]
    vv = torch.where(in_cache[:, None, :, None], vv, torch.zeros_like(vv[:1]))
    out = torch.matmul(e.view(r, hk, -1, width * p), vv).view(r, hk, h // hk, most, d)
    out = torch.where(total > 0, out / total, torch.zeros_like(out)).permute(0, 3, 1, 2, 4).reshape(r * most, h * d)
    lse = (m + torch.log(total)).squeeze(-1).permute(1, 2, 0, 3).reshape(h, r * most)
    return {"out": out.to(s["q"].dtype), "lse": lse}  # every request of a case has `most` rows


def _logprobs_plain(s):
    x, t = s["logits"].float(), s["tokens"].long()
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(1, keepdim=True)
    logp = x - m - torch.log(total)
    p = e / total
    entropy = -(p * torch.where(p > 0, logp, torch.zeros_like(logp))).sum(1)
    out = {"logprob": logp.gather(1, t[:, None])[:, 0], "entropy": entropy}
    if s["top"]:
        _, ids = torch.sort(x, dim=1, descending=True, stable=True)
        ids = ids[:, :s["top"]]
        out["top_ids"], out["top_logprobs"] = ids.int(), logp.gather(1, ids)
    if s["grad"]:
        hit = torch.zeros_like(x).scatter_(1, t[:, None], 1.0)
        grad = s["g_logprob"][:, None] * (hit - p) - s["g_entropy"][:, None] * p * (logp + entropy[:, None])
        out["grad"] = grad.to(s["logits"].dtype)
    return out


_PLAIN = {"plan": _plan_plain, "append": _append_plain, "attention": _attention_plain, "logprobs": _logprobs_plain,
          "logprobs_grad": _logprobs_plain}


# ---------------------------------------------------------------- the library's calls
def _library():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dark-forest_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import dfattn
    from dfattn import ops

    return dfattn, ops


def _run_own(s):
    dfattn, ops = _library()
    kind = s["kind"]
    if kind == "plan":
        seq_lens, query_start, slots, counts = dfattn.paged_plan(
            s["cached"], s["new"], s["table"], s["free"], s["free_start"], s["page"], s["n_pages"], s["capacity"])
        return {"table": s["table"], "seq_lens": seq_lens, "query_start": query_start, "slots": slots,
                "counts": counts}
    if kind == "append":
        dfattn.kv8_append(s["cache"], s["k"], s["v"], s["slots"])
        k, v = dfattn.kv8_read(s["cache"], s["all"], s["d_head"])
        return {"k": k, "v": v}
    if kind == "attention":
        out, lse = dfattn.kv8_attention(s["cache"], s["q"], s["table"], s["query_start"], s["seq_lens"], s["heads"],
                                        s["max_q"], s["max_len"], s["scale"])
        return {"out": out, "lse": lse}
    logprob, entropy, stats, ids, top = ops.token_logprobs_forward(s["logits"], s["tokens"], s["top"])
    out = {"logprob": logprob, "entropy": entropy}
    if s["top"]:
        out["top_ids"], out["top_logprobs"] = ids, top
    if s["grad"]:
        out["grad"] = ops.token_logprobs_backward(s["logits"], s["tokens"], stats, entropy, s["g_logprob"],
                                                  s["g_entropy"])
    return out


def run(state):
    return _run_own(state) if own else _PLAIN[state["kind"]](state)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    if c["kind"] == "plan":
        tokens = min(sum(_spread(c["new"], c["requests"])), c["capacity"])
        pages = tokens / c["page"]
        return {"bytes": 8 * c["requests"] + 8 * c["requests"] + 8 * pages + 4 * c["capacity"], "flops": 0}
    if c["kind"] == "append":
        new = sum(_spread(c["new"], c["requests"]))
        rows = new + c["requests"] * c["page"] / 2
        width, item = 2 * c["kv_heads"] * c["d_head"], 4 if c["act"] == "f32" else 2
        return {"bytes": new * width * (item + 1) + rows * width * 5, "flops": 0}
    if c["kind"] == "attention":
        lens, item = _lengths(c), 4 if c["act"] == "f32" else 2
        width, rows = 2 * c["kv_heads"] * c["d_head"], c["requests"] * c["q"]
        pairs = sum(c["q"] * n - c["q"] * (c["q"] - 1) // 2 for n in lens)
        return {"bytes": sum(lens) * (width + 8 * c["kv_heads"] / c["page"]) + 2 * rows * c["heads"] * c["d_head"] * item,
                "flops": 4 * c["heads"] * c["d_head"] * pairs}
    n, item = c["rows"] * c["vocab"], 4 if c["type"] == "f32" else 2
    return {"bytes": n * item * (2 if c["kind"] == "logprobs_grad" else 1) + c["rows"] * (12 + 8 * c["top"]), "flops": 0}


# ---------------------------------------------------------------- in 64 bits, from the definitions
def _round8(y, fmt):
    """y (float64, within range) to the nearest code of the format, ties to even."""
    if fmt == "i8":
        return torch.round(y)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def _exact_append(x, codes, scales, slots, p, fmt, at):
    """x [n, hk, d] float64; codes [pages, p, hk, d] float64: the rows `at` after the append."""
    limit, scales = FORMATS[fmt][1], scales.double().clone()
    page, off = slots.long() // p, slots.long() % p
    values = codes * scales[:, None, :, None]
    for i in torch.unique(page).tolist():
        new = page == i
        begin = int(off[new].min())
        amax = x[new].abs().amax((0, 2))
        e = torch.ceil(torch.log2(amax / limit).clamp(min=-126))
        e = torch.where(amax <= limit * torch.exp2(e - 1), e - 1, e).clamp(min=-126)
        e = torch.where(amax > limit * torch.exp2(e), e + 1, e)
        s = torch.exp2(e)
        if begin:
            s = torch.maximum(s, scales[i])
            values[i, :begin] = _round8(values[i, :begin] / s[None, :, None], fmt) * s[None, :, None]
        values[i, off[new]] = _round8(x[new] / s[None, :, None], fmt) * s[None, :, None]
    return values.reshape(-1, codes.shape[2] * codes.shape[3])[at.long()]


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["kind"] == "plan":
        return None
    if c["kind"] == "append":
        k, v, ks, vs = s["cache"]
        p, hk, d = c["page"], c["kv_heads"], c["d_head"]
        side = lambda x, codes, sc: _exact_append(x.double().view(-1, hk, d), codes, sc, s["slots"], p, c["fmt"], s["all"])
        return {"k": side(s["k"], k.double()[..., :d].permute(0, 2, 1, 3).contiguous(), ks),
                "v": side(s["v"], v.double()[:, :, :d].permute(0, 3, 1, 2).contiguous(), vs)}
    if c["kind"] == "attention":
        k, v, ks, vs = s["cache"]
        d, hk, group, nq = c["d_head"], c["kv_heads"], c["heads"] // c["kv_heads"], c["q"]
        out = torch.zeros(s["q"].shape[0], c["heads"], d, dtype=torch.float64, device=DEVICE)
        lse = torch.zeros(c["heads"], s["q"].shape[0], dtype=torch.float64, device=DEVICE)
        for r, n in enumerate(s["seq_lens"].tolist()):
            pages = s["table"][r, :-(-n // c["page"])].long()
            for j in range(hk):
                kj = (k[:, j].view(torch.uint8)[pages].view(k.dtype).double() * ks[pages, j].double()[:, None, None])
                vj = (v[:, j].view(torch.uint8)[pages].view(v.dtype).double() * vs[pages, j].double()[:, None, None])
                kj = kj.reshape(-1, kj.shape[2])[:n, :d].t().contiguous()
                vj = vj.transpose(1, 2).reshape(-1, vj.shape[1])[:n, :d].contiguous()
                for g in range(group):
                    h = j * group + g
                    q = s["q"][r * nq:(r + 1) * nq, h * d:(h + 1) * d].double()
                    x = (q @ kj) * s["scale"]
                    last = n - nq + torch.arange(nq, device=DEVICE)
                    x[torch.arange(n, device=DEVICE)[None, :] > last[:, None]] = -math.inf
                    top = torch.logsumexp(x, 1)
                    lse[h, r * nq:(r + 1) * nq] = top
                    out[r * nq:(r + 1) * nq, h] = torch.exp(x - top[:, None]) @ vj
        return {"out": out.view(-1, c["heads"] * d), "lse": lse}
    parts = {}
    for a in range(0, c["rows"], 256):
        x, t = s["logits"][a:a + 256].double(), s["tokens"][a:a + 256].long()
        logp = torch.log_softmax(x, 1)
        p = torch.exp(logp)
        entropy = -(p * logp).sum(1)
        got = {"logprob": logp.gather(1, t[:, None])[:, 0], "entropy": entropy}
        if c["top"]:
            got["top_logprobs"] = torch.topk(logp, c["top"], 1).values
        if s["grad"]:
            hit = torch.nn.functional.one_hot(t, c["vocab"]).double()
            gl, ge = s["g_logprob"][a:a + 256, None].double(), s["g_entropy"][a:a + 256, None].double()
            got["grad"] = gl * (hit - p) - ge * p * (logp + entropy[:, None])
        for name, value in got.items():
            parts.setdefault(name, []).append(value)
    out = {name: torch.cat(values) for name, values in parts.items()}
    if c["top"]:
        out["top_ids"] = None
    return out
