"""Performance cases of the operators between and inside the steps of a generating program: pages of a paged cache
(forking, freeing, compacting, with the copies) and linear layers with 4-bit weights (quantising, products).

listed() names twelve calls, draw() gives more of the same ranges. prepare() makes what a program has in hand
before the call, run() is one pass: in plain torch operations, or, where `own` is true, through the library's
entry points. exact() gives the computed numbers in 64 bits.

Tables: page ids [requests, max_pages], -1 behind a request's pages. 4-bit weights: codes [outputs, bytes] with input 2 b in the
low half of byte b (rows of whole 16 bytes), scales bf16 [groups, outputs], zeros [groups, outputs] for "u4";
value = (code - zero) * scale ("i4": zero 8), or the e2m1 number of the code times the scale.
"""
import math
import os
import sys

import torch

DEVICE = "cuda"
own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "i8": torch.int8}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def listed():
    return [
        # A beam step of two prompts with four beams each, 12 layers of an 8-bit cache of GPT-2 small's heads.
        {"name": "fork_beams_r8_l1000", "kind": "fork", "requests": 8, "children": 8, "share": 4, "length": 1000, "page": 16,
         "pages": 1500, "pool": "i8", "layers": 12, "width": 768, "keep": False},
        # Sixty prompts of mixed lengths, eight answers to each, bf16 pools.
        {"name": "fork_answers_r60_n480_l3000", "kind": "fork", "requests": 60, "children": 480, "share": 1, "length": 3000,
         "page": 16, "pages": 24000, "pool": "bf16", "layers": 4, "width": 768, "keep": False},
        # A few of a small batch's requests have ended.
        {"name": "free_r48_l1000", "kind": "free", "requests": 48, "share": 1, "length": 1000, "page": 16, "pages": 4096},
        # A large server: two thousand requests, groups of four with a common prefix.
        {"name": "free_r2000_l3000", "kind": "free", "requests": 2000, "share": 4, "length": 3000, "page": 16,
         "pages": 500000},
        # A small cache is made dense, to be cut short.
        {"name": "compact_r20_l500", "kind": "compact", "requests": 20, "share": 1, "length": 500, "page": 16, "pages": 1400,
         "pool": "i8", "layers": 2, "width": 768},
        # A large one, after half of its requests have gone.
        {"name": "compact_r300_l1500", "kind": "compact", "requests": 300, "share": 3, "length": 1500, "page": 32,
         "pages": 30001, "pool": "bf16", "layers": 2, "width": 512},
        # One matrix of a small model, from its fp32 checkpoint.
        {"name": "quantize_768x768_i4", "kind": "quantize", "out": 768, "in": 768, "group": 64, "fmt": "i4", "type": "f32"},
        # A large layer, with zero points.
        {"name": "quantize_16384x4096_u4_bf16", "kind": "quantize", "out": 16384, "in": 4096, "group": 128, "fmt": "u4",
         "type": "bf16"},
        # One token's fused query, key and value projection: latency.
        {"name": "linear_r1_768x2304_i4", "kind": "linear", "rows": 1, "out": 2304, "in": 768, "group": 64, "fmt": "i4",
         "type": "f32", "bias": True, "gelu": False, "residual": False},
        # One token through a large layer: the weights' bytes.
        {"name": "linear_r1_4096x16384_u4_bf16", "kind": "linear", "rows": 1, "out": 16384, "in": 4096, "group": 128,
         "fmt": "u4", "type": "bf16", "bias": False, "gelu": False, "residual": False},
        # The logits of sixteen generating requests, an odd vocabulary.
        {"name": "linear_r16_768x50257_e2m1", "kind": "linear", "rows": 16, "out": 50257, "in": 768, "group": 32,
         "fmt": "e2m1", "type": "f32", "bias": False, "gelu": False, "residual": False},
        # A chunk of a prompt through a layer with its GELU.
        {"name": "linear_r500_4096x4096_i4_bf16", "kind": "linear", "rows": 500, "out": 4096, "in": 4096, "group": 128,
         "fmt": "i4", "type": "bf16", "bias": True, "gelu": True, "residual": False},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    kind = rng.choices(("fork", "free", "compact", "quantize", "linear"), weights=(20, 12, 14, 14, 40))[0]
    if kind in ("fork", "free", "compact"):
        page = rng.choice((16, 16, 32, 64, 128, 20))
        most = {"fork": 1_000_000, "free": 6_000_000, "compact": 1_000_000}[kind]  # tokens of all requests
        length = _log_int(rng, 20, 20000)
        requests = _log_int(rng, 1, max(1, min(2000, most // length)))
        c = {"kind": kind, "requests": requests, "share": rng.choice((1, 1, 2, 4)), "length": length, "page": page}
        used = requests * (2 * length // page + 2)
        if kind == "free":
            return {**c, "pages": used + rng.randint(0, used)}
        c.update(pool=rng.choice(("i8", "bf16", "f32")), layers=rng.choice((1, 2, 4, 12)), width=64 * rng.randint(1, 16))
        c["children"] = _log_int(rng, 1, 600)
        item = {"i8": 1, "bf16": 2, "f32": 4}[c["pool"]]
        each = 2 * c["layers"] * page * c["width"] * item  # bytes of a page
        if kind == "compact":
            del c["children"]
            c["pages"] = min(used + rng.randint(0, used), max(100, 1_500_000_000 // each))
            c["requests"] = max(1, min(requests, c["pages"] // (2 * length // page + 2)))
            c["pages"] = max(c["pages"], c["requests"] * (2 * length // page + 2))
            return c
        c["children"] = max(1, min(c["children"], 200_000_000 // each, most // length))
        return {**c, "pages": used + c["children"] + rng.randint(0, used), "keep": rng.random() < 0.3}
    c = {"kind": kind, "in": _log_int(rng, 64, 12000), "group": rng.choice((32, 64, 128)), "fmt": rng.choice(("i4", "u4", "e2m1")),
         "type": rng.choice(("f32", "bf16"))}
    c["out"] = _log_int(rng, 64, min(60000, 60_000_000 // c["in"]))
    if kind == "quantize":
        return c
    rows = rng.choice((1, 1, 2, 4, 8)) if rng.random() < 0.5 else _log_int(rng, 3, 600)
    c["rows"] = max(1, min(rows, 8_000_000_000 // (c["in"] * c["out"])))
    c.update(bias=rng.random() < 0.5, gelu=rng.random() < 0.3, residual=rng.random() < 0.3)
    return c


# ---------------------------------------------------------------- inputs, from the seed alone
def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE)


def _randint(g, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=g, device=DEVICE)


def _lengths(c):
    """Tokens of each request: from 1 to 2 * length - 1, evenly spread."""
    n, most = c["requests"], c["length"]
    return [most if n == 1 else 1 + round(i * (2 * most - 2) / (n - 1)) for i in range(n)]


def _tables(c, g):
    """(block table, lengths): `share` requests at a time have the whole pages of the first half in common."""
    r, p, share = c["requests"], c["page"], c["share"]
    lens = torch.tensor(_lengths(c), device=DEVICE)[torch.randperm(r, generator=g, device=DEVICE)]
    pages = (lens + p - 1) // p
    width = (2 * c["length"]) // p + 2
    col = torch.arange(width, device=DEVICE)[None, :]
    first = torch.arange(r, device=DEVICE) // share * share
    common = torch.minimum(lens, lens[first]) // p // 2  # whole pages that a request has of its group's first
    common[first == torch.arange(r, device=DEVICE)] = 0
    mine = (col < pages[:, None]) & (col >= common[:, None])
    table = torch.full((r, width), -1, dtype=torch.int64, device=DEVICE)
    table[mine] = torch.randperm(c["pages"], generator=g, device=DEVICE)[:int(mine.sum())]
    table = torch.where((col < pages[:, None]) & ~mine, table[first], table)
    return table.int().contiguous(), lens.int()


def _pools(c, g):
    """Two pools a layer, [pages, page size, width], as layers give their keys and values; 8-bit ones have a scale a page beside them."""
    one = _randn(g, 2 * c["layers"], c["page"], c["width"])
    pools = []
    for i in range(2 * c["layers"]):
        some = torch.empty(c["pages"], c["page"], c["width"], dtype=TYPES[c["pool"]], device=DEVICE)
        step = max(1, (1 << 26) // (c["page"] * c["width"]))
        for a in range(0, c["pages"], step):
            n = min(step, c["pages"] - a)
            f = 0.5 + torch.rand(n, 1, 1, generator=g, device=DEVICE)
            some[a:a + n] = (one[i] * f * (25.0 if c["pool"] == "i8" else 1.0)).clamp_(-127, 127).to(some.dtype)
        pools.append(some)
        if c["pool"] == "i8":
            pools.append(torch.exp2(-_randint(g, 0, 12, c["pages"], c["width"] // 64).float()))
    return pools


def _paged_inputs(c, seed):
    g = _generator(seed)
    table, lens = _tables(c, g)
    r, p = c["requests"], c["page"]
    s = {"table": table, "lens": lens, "page": p, "pages": c["pages"]}
    if c["kind"] == "free":
        s["ended"] = (_randint(g, 0, 4, r) == 0).int()
        return s
    s["pools"] = _pools(c, g)
    if c["kind"] == "compact":
        s["lens"] = torch.where(_randint(g, 0, 2, r) == 0, torch.zeros_like(lens), lens)  # half of them have gone
        s["new_table"] = table.clone()
        return s
    n = c["children"]
    if n > r and c["share"] == 1:
        s["parents"] = (torch.arange(n, device=DEVICE) * r // n).int()  # answers to each prompt
    else:
        s["parents"] = _randint(g, 0, r, n).int()  # beams: some go on, some more than once, some end
    if c["keep"]:
        s["keep"] = _randint(g, 0, 2 * c["length"], n).int()
    s["new_table"] = torch.full((n, table.shape[1]), -1, dtype=torch.int32, device=DEVICE)
    return s


def _bytes_of(k):
    """Bytes of a row of k codes."""
    return -(-k // 32) * 16


def _weights(c, g):
    """(codes, scales, zeros or None) as quantised layers have them."""
    n, k, group = c["out"], c["in"], c["group"]
    groups = -(-k // group)
    q = torch.empty(n, 2 * _bytes_of(k), dtype=torch.uint8, device=DEVICE)
    step = max(1, (1 << 26) // q.shape[1])
    for a in range(0, n, step):
        x = _randn(g, min(step, n - a), q.shape[1])
        q[a:a + step] = (torch.round(x * 2.5) + 8).clamp_(0, 15).to(torch.uint8) if c["fmt"] != "e2m1" else \
            (torch.round(x.abs() * 2.5).clamp_(0, 7) + 8 * (x < 0)).to(torch.uint8)
    codes = q[:, 0::2] | (q[:, 1::2] << 4)
    scales = (0.02 * (0.5 + torch.rand(groups, n, generator=g, device=DEVICE))).bfloat16()
    zeros = _randint(g, 5, 11, groups, n).to(torch.uint8) if c["fmt"] == "u4" else None
    return codes.contiguous(), scales, zeros


def _quantize_inputs(c, seed):
    g = _generator(seed)
    w = 0.02 * _randn(g, c["out"], c["in"])
    return {"w": w.to(TYPES[c["type"]]), "group": c["group"], "fmt": c["fmt"]}


def _linear_inputs(c, seed):
    g, act = _generator(seed), TYPES[c["type"]]
    x = _randn(g, c["rows"], c["in"])
    x[:, :: 61] *= 8.0  # a few channels larger than the others
    codes, scales, zeros = _weights(c, g)
    return {"x": x.to(act), "codes": codes, "scales": scales, "zeros": zeros, "group": c["group"], "fmt": c["fmt"],
            "in": c["in"], "gelu": c["gelu"], "bias": 0.1 * _randn(g, c["out"]) if c["bias"] else None,
            "residual": _randn(g, c["rows"], c["out"]).to(act) if c["residual"] else None}


_INPUTS = {"fork": _paged_inputs, "free": _paged_inputs, "compact": _paged_inputs, "quantize": _quantize_inputs,
           "linear": _linear_inputs}


def prepare(case, seed):
    return {"kind": case["kind"], **_INPUTS[case["kind"]](case, seed)}


# ---------------------------------------------------------------- pages in plain form
def _refs(table, lens, p, pages):
    """How often each page is in the first ceil(lens / p) places of a row."""
    held = (torch.arange(table.shape[1], device=DEVICE)[None, :] < ((lens + p - 1) // p)[:, None])
    held &= (table >= 0) & (table < pages)
    at = torch.where(held, table, torch.full_like(table, pages)).flatten()
    return torch.zeros(pages + 1, dtype=torch.int64, device=DEVICE).index_add_(0, at, torch.ones_like(at))[:pages]


def _by_use(refs):
    """(pages with references, ascending, then those without, ascending; how many have)"""
    free = (refs == 0).long()
    return torch.sort(free, stable=True)[1], refs.numel() - free.sum()


def _copy(pools, src, dst):
    """The pages src of every pool to its pages dst; -1: none."""
    real = src >= 0
    src, dst = src[real], dst[real]
    return [x.index_copy_(0, dst, x[src]) for x in pools]


def _fork_plain(s):
    p, pages, table = s["page"], s["pages"], s["table"].long()
    width, parents = table.shape[1], s["parents"].long()
    lens = s["lens"].long().clamp(max=width * p)[parents]
    if "keep" in s:
        lens = torch.minimum(lens, s["keep"].long())
    rows = table[parents]
    refs = _refs(rows, lens, p, pages)
    n = parents.numel()
    child = torch.arange(n, device=DEVICE)
    last = ((lens + p - 1) // p - 1).clamp(min=0)
    partial = lens % p != 0
    old = torch.where(partial, rows[child, last], torch.full_like(last, pages))
    lasts = torch.zeros(pages + 1, dtype=torch.int64, device=DEVICE).index_add_(0, old, torch.ones_like(old))
    lowest = torch.full((pages + 1,), n, device=DEVICE).scatter_reduce(0, old, child, "amin")
    alone = torch.cat([refs, refs[:1]])[old] == lasts[old]
    need = partial & ~((lowest[old] == child) & alone)
    order, used = _by_use(refs)
    rank = torch.cumsum(need.long(), 0) - 1
    got = need & (rank < pages - used)
    new = torch.where(got, order[(used + rank).clamp(0, pages - 1)], old)
    refs = torch.cat([refs, refs[:1]])
    refs.index_add_(0, torch.where(need, old, torch.full_like(old, pages)), -torch.ones_like(old))
    refs[torch.where(got, new, torch.full_like(new, pages))] = 1
    held = torch.arange(width, device=DEVICE)[None, :] < ((lens + p - 1) // p)[:, None]
    rows[child, last] = torch.where(got, new, rows[child, last])
    s["new_table"].copy_(torch.where(held, rows, s["new_table"].long()))
    at = torch.where(got, rank, torch.full_like(rank, n))
    src, dst = (torch.full((n + 1,), -1, device=DEVICE).index_copy_(0, at, x)[:n] for x in (old, new))
    src, dst = torch.where(child < got.sum(), src, -1), torch.where(child < got.sum(), dst, -1)
    counts = torch.stack([got.sum(), (need & ~got).sum()])
    return {"table": s["new_table"], "lens": torch.where(need & ~got, lens // p * p, lens).int(), "refs": refs[:pages].int(),
            "free_pages": order.int(), "free_start": (used + got.sum()).int()[None], "src": src.int(), "dst": dst.int(),
            "counts": counts.int(), "pools": _copy(s["pools"], src, dst)}


def _free_plain(s):
    lens = torch.where(s["ended"] != 0, torch.zeros_like(s["lens"]), s["lens"])
    s["lens"].copy_(lens)
    refs = _refs(s["table"].long(), lens.long(), s["page"], s["pages"])
    order, used = _by_use(refs)
    return {"lens": s["lens"], "refs": refs.int(), "free_pages": order.int(), "free_start": used.int()[None]}


def _compact_plain(s):
    p, pages, table = s["page"], s["pages"], s["table"].long()
    refs = _refs(table, s["lens"].long(), p, pages)
    held = torch.arange(table.shape[1], device=DEVICE)[None, :] < ((s["lens"].long() + p - 1) // p)[:, None]
    page = torch.arange(pages, device=DEVICE)
    used = (refs > 0).sum()
    far, hole = (refs > 0) & (page >= used), (refs == 0) & (page < used)
    moves, most = far.sum(), pages // 2
    listed_ = lambda m: torch.sort((~m).long(), stable=True)[1][:most]
    src = torch.where(page[:most] < moves, listed_(far), -1)
    dst = torch.where(page[:most] < moves, listed_(hole), -1)
    to = page.clone()
    to[far] = listed_(hole)[(torch.cumsum(far.long(), 0) - 1)[far]]
    ids = torch.where(held & (table >= 0) & (table < pages), to[table.clamp(0, pages - 1)], table)
    s["new_table"].copy_(torch.where(held, ids, s["new_table"].long()))
    new_refs = torch.zeros_like(refs).index_copy_(0, to[refs > 0], refs[refs > 0])
    return {"table": s["new_table"], "refs": new_refs.int(), "free_pages": page.int(), "free_start": used.int()[None],
            "src": src.int(), "dst": dst.int(), "counts": moves.int()[None], "pools": _copy(s["pools"], src, dst)}


# ---------------------------------------------------------------- 4-bit weights in plain form
def _nearest_bf16(x):
    """x >= 0 (64 bits) to the nearest bf16 number, ties to even."""
    _, e = torch.frexp(x)
    step = torch.exp2((e - 8).clamp(min=-133).double())
    return (torch.round(x / step) * step).bfloat16()


def _quantize_plain(s):
    w, group, fmt = s["w"], s["group"], s["fmt"]
    n, k = w.shape
    groups = -(-k // group)
    x = torch.nn.functional.pad(w.double(), (0, groups * group - k)).view(n, groups, group)
    lo, hi = x.amin(2).clamp(max=0), x.amax(2).clamp(min=0)
    top = torch.maximum(-lo, hi)
    scale = _nearest_bf16({"i4": top / 7, "u4": (hi - lo) / 15, "e2m1": top / 6}[fmt])
    d = scale.double()[:, :, None]
    y = torch.where(d > 0, x / torch.where(d > 0, d, torch.ones_like(d)), torch.zeros_like(x))
    out = {"scales": scale.t().contiguous()}
    if fmt == "e2m1":
        a = y.abs()
        step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
        v = torch.copysign((torch.round(a / step) * step).clamp(max=6), y)
    elif fmt == "i4":
        v = torch.round(y).clamp(-8, 7)
    else:
        zero = torch.where(d[:, :, 0] > 0, torch.round(-lo / torch.where(d[:, :, 0] > 0, d[:, :, 0], 1.0)), 0.0).clamp(0, 15)
        v = (torch.round(y) + zero[:, :, None]).clamp(0, 15) - zero[:, :, None]
        out["zeros"] = zero.t().to(torch.uint8).contiguous()
    out["values"] = (v * d).view(n, -1)[:, :k].float()
    return out


def _values(s, dtype):
    """The weights of codes, [outputs, inputs]."""
    n, k, group = s["codes"].shape[0], s["in"], s["group"]
    q = torch.stack([s["codes"] & 15, s["codes"] >> 4], 2).view(n, -1)[:, :k]
    g = torch.arange(k, device=DEVICE) // group
    scale = s["scales"].to(dtype).t()[:, g]
    if s["fmt"] == "e2m1":
        return torch.tensor(E2M1, dtype=dtype, device=DEVICE)[q.int()] * scale
    return (q.to(dtype) - (8 if s["zeros"] is None else s["zeros"].to(dtype).t()[:, g])) * scale


def _linear_plain(s):
    y = torch.matmul(s["x"].float(), _values(s, torch.float32).t())
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["gelu"]:
        y = 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"out": y.to(s["x"].dtype)}


_PLAIN = {"fork": _fork_plain, "free": _free_plain, "compact": _compact_plain, "quantize": _quantize_plain,
          "linear": _linear_plain}


# ---------------------------------------------------------------- the library's calls
def _library():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dark-forest_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import dfattn
    from dfattn import w4

    return dfattn, w4


def _run_own(s):
    dfattn, w4 = _library()
    kind = s["kind"]
    if kind == "fork":
        f = dfattn.paged_fork(s["table"], s["lens"], s["parents"], s["page"], s["pages"], s.get("keep"),
                              new_table=s["new_table"])
        dfattn.paged_copy(s["pools"], f.copy_src, f.copy_dst, f.counts)
        return {"table": f.block_table, "lens": f.seq_lens, "refs": f.refs, "free_pages": f.free_pages,
                "free_start": f.free_start, "src": f.copy_src, "dst": f.copy_dst, "counts": f.counts, "pools": s["pools"]}
    if kind == "free":
        refs, free_pages, free_start = dfattn.paged_free(s["table"], s["lens"], s["page"], s["pages"], s["ended"])
        return {"lens": s["lens"], "refs": refs, "free_pages": free_pages, "free_start": free_start}
    if kind == "compact":
        f = dfattn.paged_compact(s["table"], s["lens"], s["page"], s["pages"], new_table=s["new_table"])
        dfattn.paged_copy(s["pools"], f.copy_src, f.copy_dst, f.counts)
        return {"table": f.block_table, "refs": f.refs, "free_pages": f.free_pages, "free_start": f.free_start,
                "src": f.copy_src, "dst": f.copy_dst, "counts": f.counts, "pools": s["pools"]}
    if kind == "quantize":
        w = w4.quantize(s["w"], s["group"], s["fmt"])
        out = {"scales": w.scales, "values": w4.dequantize(w)}
        if s["fmt"] == "u4":
            out["zeros"] = w.zeros
        return out
    w = w4.Weight(s["codes"], s["scales"], s["zeros"], s["in"], s["group"], s["fmt"])
    return {"out": w4.linear(s["x"], w, bias=s["bias"], residual=s["residual"], gelu=s["gelu"])}


def run(state):
    return _run_own(state) if own else _PLAIN[state["kind"]](state)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    if c["kind"] in ("fork", "free", "compact"):
        held = sum(-(-n // c["page"]) for n in _lengths(c))
        if c["kind"] == "free":
            return {"bytes": 4 * held * 3 / 4 + 8 * c["pages"] + 12 * c["requests"], "flops": 0}
        each = 2 * c["layers"] * c["page"] * c["width"] * {"i8": 1, "bf16": 2, "f32": 4}[c["pool"]]
        if c["kind"] == "compact":
            used = held / 2 * (1 - (c["share"] - 1) / c["share"] / 4)
            moves = used * (1 - used / c["pages"])
            return {"bytes": 4 * held + 8 * c["pages"] + moves * (2 * each + 8), "flops": 0}
        kept = held / c["requests"] * c["children"]
        copies = c["children"] * 0.4 if c["share"] > 1 or c["children"] <= c["requests"] else c["children"] - c["requests"]
        return {"bytes": 8 * kept + 8 * c["pages"] + copies * (2 * each + 8), "flops": 0}
    n, k, item = c["out"], c["in"], 4 if c["type"] == "f32" else 2
    weights = n * k / 2 + -(-k // c["group"]) * n * (3 if c["fmt"] == "u4" else 2)
    if c["kind"] == "quantize":  # the weights read, the codes written and read, their values written
        return {"bytes": n * k * (item + 4) + 2 * weights, "flops": 0}
    extra = (4 * n if c["bias"] else 0) + (c["rows"] * n * item if c["residual"] else 0)
    return {"bytes": weights + c["rows"] * (k + n) * item + extra, "flops": 2 * c["rows"] * n * k}


# ---------------------------------------------------------------- in 64 bits, from the definitions
def _exact_quantize(s):
    w, group, fmt = s["w"].double(), s["group"], s["fmt"]
    n, k = w.shape
    grid = torch.tensor(E2M1[:8], dtype=torch.float64, device=DEVICE)
    values, scales = torch.empty_like(w), []
    for a in range(0, k, group):
        x = w[:, a:a + group]
        lo, hi = x.min(1).values.clamp(max=0), x.max(1).values.clamp(min=0)
        want = (hi - lo) / 15 if fmt == "u4" else torch.maximum(hi, -lo) / (7 if fmt == "i4" else 6)
        e = torch.floor(torch.log2(want.clamp(min=1e-300)))
        unit = torch.exp2(e - 7)
        d = (torch.round(want / unit) * unit)[:, None]
        if fmt == "e2m1":
            far = (x.abs()[:, :, None] - grid * d[:, :, None]).abs()
            even = torch.tensor([0, 1] * 4, device=DEVICE) * 1e-12
            v = grid[(far + even * d[:, :, None]).argmin(2)] * torch.sign(x)
        elif fmt == "i4":
            v = torch.round(x / d).clamp(-8, 7)
        else:
            zero = torch.round(-lo[:, None] / d).clamp(0, 15)
            v = (torch.round(x / d) + zero).clamp(0, 15) - zero
        values[:, a:a + group] = v * d
        scales.append(d[:, 0])
    out = {"scales": torch.stack(scales), "values": values}
    if fmt == "u4":
        out["zeros"] = None
    return out


def exact(case, seed):
    if case["kind"] not in ("quantize", "linear"):
        return None
    s = prepare(case, seed)
    if case["kind"] == "quantize":
        return _exact_quantize(s)
    x, group, parts = s["x"].double(), s["group"], []
    for a in range(0, case["out"], 4096):
        codes = s["codes"][a:a + 4096].int()
        y = torch.zeros(case["rows"], codes.shape[0], dtype=torch.float64, device=DEVICE)
        for g, b in enumerate(range(0, case["in"], group)):
            k = min(group, case["in"] - b)
            part = codes[:, b // 2:(b + k + 1) // 2]
            q = torch.cat([(part & 15)[:, :, None], (part >> 4)[:, :, None]], 2).flatten(1)[:, :k]
            if s["fmt"] == "e2m1":
                size = torch.where(q % 8 < 2, (q % 8) * 0.5, (1 + 0.5 * (q % 2)) * torch.exp2((q % 8 // 2 - 1).double()))
                v = torch.where(q >= 8, -size, size).double()
            else:
                v = q.double() - (8.0 if s["zeros"] is None else s["zeros"][g, a:a + 4096, None].double())
            y += (x[:, b:b + k] @ v.t().contiguous()) * s["scales"][g, a:a + 4096].double()
        parts.append(y)
    y = torch.cat(parts, 1)
    if s["bias"] is not None:
        y += s["bias"].double()
    if s["gelu"]:
        y = 0.5 * y * (1 + torch.tanh((2 / math.pi) ** 0.5 * (y + 0.044715 * y ** 3)))
    if s["residual"] is not None:
        y += s["residual"].double()
    return {"out": y}
