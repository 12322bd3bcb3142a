"""Linear layers with 4-bit weights (dfgpt2_w4_*) against 64-bit references.

Tolerances. Values and scales are exact. A product's error: with bf16 or fp32 activations every term code * x is exact in
the products' inputs, so what is left is the fp32 sums. Summing K terms in fp32 in any order with partial sums
grouped as the kernel likes is off by at most (K + groups) * 2^-24 * sum |code - zero| |x| scale, where a zero point may
take part as its own term (code x - zero x: 2 * 15 in place of |code - zero|), so 4 K 2^-24 * 15 * sum |x| scale bounds it with room
for the group's scale and bias. GELU's slope is at most 1.13 and its own fp32 error a few units of |y| + 1 (2^-20 taken). The result is
rounded once: half a unit of the type.
"""
import math

import pytest
import torch

from dfattn import w4

pytestmark = pytest.mark.gpu

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def weight(seed, n, k, group, fmt):
    """A Weight of random codes: all sixteen, zeros of 0..15, scales of many sizes."""
    g = generator(seed)
    codes = torch.randint(0, 256, (n, w4.row_bytes(k)), generator=g, device="cuda", dtype=torch.uint8)
    groups = -(-k // group)
    scales = torch.exp2(torch.randint(-9, 3, (groups, n), generator=g, device="cuda").float()) * \
        (1 + torch.rand(groups, n, generator=g, device="cuda"))
    zeros = torch.randint(0, 16, (groups, n), generator=g, device="cuda", dtype=torch.uint8) if fmt == "u4" else None
    return w4.Weight(codes, scales.bfloat16(), zeros, k, group, fmt)


def values(w):
    """The weights in 64 bits."""
    n, k = w.codes.shape[0], w.in_features
    q = torch.stack([w.codes & 15, w.codes >> 4], 2).reshape(n, -1)[:, :k].long()
    g = torch.arange(k, device="cuda") // w.group
    if w.format == "e2m1":
        v = torch.tensor(E2M1, device="cuda", dtype=torch.float64)[q % 8] * (1 - 2 * (q // 8))
    else:
        v = q.double() - (8 if w.zeros is None else w.zeros.double().t()[:, g])
    return v * w.scales.double().t()[:, g]


def gelu64(y):
    return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))


def check(x, w, bias=None, residual=None, gelu=False, out=None, **kw):
    want, g = values(w), torch.arange(w.in_features, device="cuda") // w.group
    y = x.double() @ want.t().contiguous()
    size = x.double().abs() @ w.scales.double().t()[:, g].t().contiguous() * 15
    bound = 4 * w.in_features * 2.0 ** -24 * size
    if bias is not None:
        y = y + bias.double()
        bound = bound + 2.0 ** -24 * y.abs()
    if gelu:
        bound = 1.13 * bound + 2.0 ** -20 * (y.abs() + 1)
        y = gelu64(y)
    if residual is not None:
        y = y + residual.double()
        bound = bound + 2.0 ** -24 * y.abs()
    got = w4.linear(x, w, bias, residual, gelu, out, **kw)
    assert got.dtype == x.dtype and got.shape == y.shape
    far = (got.double() - y).abs() - bound - HALF[x.dtype] * (y.abs() + bound)
    assert far.max() <= 0, (far.max().item(), y.abs().max().item())
    return got


FORMATS = [(f, g) for f in ("i4", "u4", "e2m1") for g in (32, 64, 128)]


@pytest.mark.parametrize("fmt,group", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,k", [(1, 1), (5, 31), (16, 32), (17, 129), (40, 256), (33, 1000), (130, 515)])
def test_quantize(device, fmt, group, dtype, n, k):
    g = generator(n * k)
    w = (torch.randn(n, k, generator=g, device="cuda") * torch.exp2(torch.randint(-20, 20, (n, 1), generator=g, device="cuda").float()))
    w = w.to(dtype)
    w[0, :min(k, group)] = 0
    if n > 8:
        w[1] = w[1].abs()
        w[2] = -w[2].abs()
        w[3] = torch.round(w[3] / w[3].abs().max().clamp(min=1e-30) * 14) * 0.5  # halves: many ties
        w[4] = torch.sign(w[4]) * 3.0
    got = w4.quantize(w, group, fmt)
    groups = -(-k // group)
    x = torch.nn.functional.pad(w.double(), (0, groups * group - k)).view(n, groups, group)
    lo, hi = x.amin(2).clamp(max=0), x.amax(2).clamp(min=0)
    top = {"i4": torch.maximum(hi, -lo) / 7, "e2m1": torch.maximum(hi, -lo) / 6, "u4": (hi - lo) / 15}[fmt]
    unit = torch.exp2(torch.floor(torch.log2(top.clamp(min=1e-300))) - 7)
    scale = torch.round(top / unit) * unit
    assert torch.equal(got.scales.double(), scale.t())
    v = values(got)
    s = scale[:, torch.arange(k, device="cuda") // group]
    # Each value is the nearest one that the codes offer.
    if fmt == "e2m1":
        offered = torch.tensor([-x for x in E2M1] + list(E2M1), device="cuda", dtype=torch.float64) * s[..., None]
    elif fmt == "i4":
        offered = torch.arange(-8, 8, device="cuda").double() * s[..., None]
    else:
        zero = torch.where(scale > 0, torch.round(-lo / scale.clamp(min=1e-300)), 0).clamp(0, 15)
        assert torch.equal(got.zeros.double(), zero.t())
        offered = (torch.arange(16, device="cuda").double() - zero[:, torch.arange(k, device="cuda") // group, None]) * s[..., None]
    best = (offered - w.double()[..., None]).abs().amin(2)
    assert torch.equal((v - w.double()).abs(), best)
    if fmt == "i4":  # ties go to even codes
        tie = (w.double() / s.clamp(min=1e-300)).frac().abs() == 0.5
        assert not ((v / s.clamp(min=1e-300)).round().long()[tie & (s > 0)] % 2).any()
    for t in (torch.float32, torch.bfloat16):
        assert torch.equal(w4.dequantize(got, t), v.float().to(t))


def test_quantize_far(device):
    """Scales next to bf16's range, groups with an infinity or NaN, rows as a column block."""
    w = torch.ones(6, 64, device="cuda")
    w[0] *= 2.0 ** -126
    w[1] *= 2.0 ** -140
    w[2] *= 3.3e38
    w[3, 40] = math.inf
    w[4, 3] = math.nan
    w[5] = 0
    for fmt in ("i4", "u4", "e2m1"):
        q = w4.quantize(w, 32, fmt)
        v = w4.dequantize(q)
        assert torch.isnan(v[3, 32:]).all() and torch.isnan(v[4, :32]).all()
        assert not torch.isnan(v[3, :32]).any() and not torch.isnan(v[4, 32:]).any() and not v[5].any()
        for r in (0, 2):
            assert ((v[r].double() - w[r].double()).abs() <= 0.08 * w[r].double()).all(), (fmt, r)
        assert (v[1].double() - w[1].double()).abs().max() <= 2.0 ** -134 * 7.5  # half a unit of the last bf16 scale, 7 times over, and half a step
    g = generator(5)
    wide = torch.randn(37, 300, generator=g, device="cuda")
    a, b = w4.quantize(wide[:, 11:240], 64, "u4"), w4.quantize(wide[:, 11:240].contiguous(), 64, "u4")
    assert all(torch.equal(x, y) for x, y in zip(a[:3], b[:3]))


@pytest.mark.parametrize("fmt,group", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 2, 7, 16, 17, 33, 64, 65, 130, 1025, 1060])
def test_linear(device, fmt, group, dtype, rows):
    n, k = 72, 392
    x = torch.randn(rows, k, generator=generator(rows), device="cuda").to(dtype)
    check(x, weight(1, n, k, group, fmt))


@pytest.mark.parametrize("fmt,group", [("i4", 32), ("u4", 128), ("e2m1", 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (3, 15, 7), (2, 16, 31), (5, 17, 33), (1, 2304, 768), (1, 100, 4097), (20, 31, 127), (40, 300, 1111),
                                      (1, 6000, 40), (16, 5001, 768), (200, 130, 260), (1, 40, 20000), (9, 2000, 2000), (300, 260, 1000),
                                      (1100, 31, 127), (1030, 300, 1111), (1024, 130, 260), (2000, 33, 300), (1100, 600, 700),
                                      (1100, 600, 300)])
def test_linear_sizes(device, fmt, group, dtype, rows, n, k):
    x = torch.randn(rows, k, generator=generator(k), device="cuda").to(dtype)
    bias = torch.randn(n, generator=generator(n), device="cuda") if k % 2 else None
    check(x, weight(2, n, k, group, fmt), bias)


@pytest.mark.parametrize("fmt,group", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n,k", [(1, 70, 4500), (2, 70, 2100), (4, 70, 5000), (16, 40, 9000), (33, 140, 4321), (200, 1100, 2048),
                                      (1030, 140, 4321), (100, 1000, 2300), (20, 700, 9000)])
def test_linear_many_inputs(device, fmt, group, dtype, rows, n, k):
    """Many tiles of inputs, whole and shared out, and without a workspace."""
    x = torch.randn(rows, k, generator=generator(k), device="cuda").to(dtype)
    w = weight(3, n, k, group, fmt)
    check(x, w)
    check(x, w, workspace=None)


@pytest.mark.parametrize("fmt,group", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n,k", [(2, 33000, 300), (2, 8200, 4100), (5, 8210, 4100), (9, 40, 8200), (16, 70, 8300)])
def test_linear_few_rows(device, fmt, group, dtype, rows, n, k):
    """Wide layers, large ones and many inputs, where few rows share out the inputs; and without a workspace."""
    x = torch.randn(rows, k, generator=generator(k + n), device="cuda").to(dtype)
    w = weight(5, n, k, group, fmt)
    check(x, w)
    check(x, w, workspace=None)


@pytest.mark.parametrize("fmt,group", [("i4", 128), ("u4", 64), ("e2m1", 32)])
@pytest.mark.parametrize("rows", [2, 3])
def test_linear_few_rows_bf16(device, fmt, group, rows):
    n, k = 16400, 8200
    check(torch.randn(rows, k, generator=generator(k + n), device="cuda").bfloat16(), weight(6, n, k, group, fmt))


@pytest.mark.parametrize("fmt,group", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n,k", [(1, 16389, 300), (2, 16389, 300), (1, 16399, 1000), (2, 16399, 1000), (1, 16390, 1100), (2, 9000, 2200),
                                      (3, 16401, 300), (16, 16401, 300), (5, 8300, 900), (9, 33000, 300), (34, 16401, 300), (70, 4100, 300), (20, 8300, 60), (33, 33000, 60)])
def test_linear_many_outputs(device, fmt, group, dtype, rows, n, k):
    """Layers wide enough for the forms that give a wave more outputs."""
    x = torch.randn(rows, k, generator=generator(k + rows), device="cuda").to(dtype)
    check(x, weight(4, n, k, group, fmt), torch.randn(n, generator=generator(n), device="cuda"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n,k", [(1, 768, 768), (4, 1000, 640), (50, 77, 300), (150, 200, 512), (1100, 200, 512), (1100, 600, 512)])
def test_epilogue(device, dtype, rows, n, k):
    g = generator(7)
    x = torch.randn(rows, k, generator=g, device="cuda").to(dtype)
    w = weight(3, n, k, 64, "i4")
    w = w._replace(scales=(w.scales.float() * 0.02).bfloat16())
    bias, residual = torch.randn(n, generator=g, device="cuda"), torch.randn(rows, n, generator=g, device="cuda").to(dtype)
    check(x, w, gelu=True)
    check(x, w, bias, residual)
    want = check(x, w, bias, residual, gelu=True)
    out = residual.clone()
    assert w4.linear(x, w, bias, out, True, out) is out and torch.equal(out, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,k", [(1, 200), (5, 200), (20, 201), (70, 768), (1040, 520)])
def test_rows_of_a_wider_tensor(device, dtype, rows, k):
    wide = torch.randn(rows, 3 * k + 9, generator=generator(3), device="cuda").to(dtype)
    w = weight(4, 50, k, 32, "u4")
    for start in (0, 1, 8, k):
        x = wide[:, start:start + k]
        assert torch.equal(w4.linear(x, w), w4.linear(x.contiguous(), w))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [19, 1029])
def test_rows_alone(device, dtype, rows):
    """A row's result does not depend on what the other rows hold, not-numbers among them, nor on what
    stands behind the inputs' codes."""
    n, k = 90, 300
    x = torch.randn(rows, k, generator=generator(3), device="cuda").to(dtype)
    for fmt in ("i4", "u4", "e2m1"):
        w = weight(5, n, k, 64, fmt)
        want = w4.linear(x, w)
        y = x.clone()
        y[4, 7], y[11, 299], y[18] = math.inf, math.nan, -math.inf
        got = w4.linear(y, w)
        bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
        bad[[4, 11, 18]] = True
        assert torch.equal(got[~bad], want[~bad])
        assert not torch.isfinite(got[11]).any()
        nonzero = values(w)[:, 7] != 0
        assert not torch.isfinite(got[4][nonzero]).any()
        other = w.codes.clone()
        other[:, 150:] = 255 - other[:, 150:]
        assert torch.equal(w4.linear(x, w._replace(codes=other)), want)
    # A code of NaN scale reaches its output only.
    w.scales[1, 20] = math.nan
    got = w4.linear(x, w)
    assert torch.isnan(got[:, 20]).all() and torch.equal(got[:, 21:], want[:, 21:])


@pytest.mark.parametrize("fmt,group", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n,k", [(1030, 96, 5), (1030, 32, 33), (1100, 160, 70), (2, 32800, 31), (40, 32768, 96), (3, 64, 20), (1, 32, 8)])
def test_short_rows_of_codes(device, fmt, group, dtype, rows, n, k):
    """Rows of 16, 32 and 48 bytes of codes, in the middle of a tensor whose other bytes are no part of them."""
    x = torch.randn(rows, k, generator=generator(k), device="cuda").to(dtype)
    w = weight(9, n, k, group, fmt)
    want = check(x, w)
    whole = torch.full((n * w4.row_bytes(k) + 128,), 0xff, dtype=torch.uint8, device="cuda")
    codes = whole[64:-64].view(n, -1).copy_(w.codes)
    assert torch.equal(w4.linear(x, w._replace(codes=codes)), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_far_values(device, dtype):
    """Large and small activations, and fp32 ones whose last bits matter."""
    n, k = 64, 256
    g = generator(9)
    w = weight(6, n, k, 64, "i4")
    for size in (1e-25, 1e30):
        check((torch.randn(3, k, generator=g, device="cuda") * size).to(dtype), w)
    check((1 + torch.rand(5, k, generator=g, device="cuda") * 2.0 ** -10).to(dtype), w)
    e = torch.randint(-30, 30, (4, k), generator=g, device="cuda").float()
    check((torch.randn(4, k, generator=g, device="cuda") * torch.exp2(e)).to(dtype), w)


@pytest.mark.parametrize("fmt,group", FORMATS)
@pytest.mark.parametrize("rows,n", [(1, 40), (2, 16400), (16, 40), (16, 16400), (16, 32800), (1024, 40), (1024, 150), (1056, 40), (1056, 150)])
def test_exact_products(device, fmt, group, rows, n):
    """fp32 activations of 24 bits, one at a time in each of 1024 places: nothing of them is lost, wherever it stands.

    The code's product (28 bits, added up from three) is rounded at most twice to 24 bits at up to 15 |x| scale, the zero point's share and
    the scaled sum once each: 3 * 15 |x| scale and |result|, times 2^-24."""
    k = 1024
    w = weight(8, n, k, group, fmt)
    v = (torch.randint(2 ** 23, 2 ** 24, (k,), generator=generator(1), device="cuda") | 1).float()
    exact, g = values(w), torch.arange(k, device="cuda") // group
    for first in range(0, k, rows if rows > 2 else 37):
        at = (first + torch.arange(rows, device="cuda")) % k
        x = torch.zeros(rows, k, device="cuda")
        x[torch.arange(rows), at] = v[at]
        got = w4.linear(x, w).double()
        size = v[at].double()[:, None]
        want = size * exact[:, at].t()
        assert ((got - want).abs() <= 2.0 ** -24 * (3 * 15 * size * w.scales.double()[g[at]] + want.abs())).all(), first


def test_streams_and_capture(device):
    rows, n, k = 3, 700, 520
    w = weight(1, n, k, 64, "u4")
    x = torch.randn(rows, k, generator=generator(2), device="cuda")
    want = w4.linear(x, w)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    got = w4.linear(x, w, stream=stream)
    stream.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        y = w4.linear(x, w)
        z = w4.quantize(x, 32, "e2m1")
    for seed in range(3):
        x.copy_(torch.randn(rows, k, generator=generator(20 + seed), device="cuda"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, w4.linear(x, w)) and torch.equal(z.codes, w4.quantize(x, 32, "e2m1").codes)


def test_no_rows(device):
    w = weight(1, 8, 40, 32, "i4")
    assert w4.linear(torch.empty(0, 40, device="cuda"), w).shape == (0, 8)


def test_large_offsets(device):
    """Outputs and codes past 2^31 bytes, rows of x past 2^31 elements."""
    n, k = 70000, 65536
    w = weight(1, 1, k, 128, "i4")
    codes = w.codes.expand(n, -1).contiguous()
    codes[:, 0] = (torch.arange(n, device="cuda") % 256).to(torch.uint8)
    big = w4.Weight(codes, w.scales.expand(-1, n).contiguous(), None, k, 128, "i4")
    x = torch.randn(2, k, generator=generator(2), device="cuda").bfloat16()
    got = w4.linear(x, big)
    pick = torch.tensor([0, 1, 40000, 65535, 65536, 69999], device="cuda")
    small = big._replace(codes=codes[pick].contiguous(), scales=big.scales[:, pick].contiguous())
    check(x, small)
    bound = 2.0 ** -7 * got[:, pick].abs().float()  # (a sum's order may differ with the number of outputs: one unit)
    assert ((got[:, pick].float() - w4.linear(x, small).float()).abs() <= bound + 2.0 ** -12).all()
    del codes, big
    wide = torch.empty(9, 1 << 28, dtype=torch.bfloat16, device="cuda")
    rows = torch.randn(9, 300, generator=generator(3), device="cuda").bfloat16()
    wide[:, :300] = rows
    w = weight(3, 40, 300, 32, "i4")
    assert torch.equal(w4.linear(wide[:, :300], w), w4.linear(rows, w))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_two_streams(device, dtype):
    """Products that share out their inputs, on two streams at once: each call has its own sums."""
    w = weight(1, 300, 2300, 64, "u4")
    xs = [torch.randn(1100, 2300, generator=generator(seed), device="cuda").to(dtype) for seed in range(2)]
    assert w4.linear_workspace_bytes(1100, 2300, 300) > 0
    want = [w4.linear(x, w) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[w4.linear(x, w, stream=s) for x, s in zip(xs, streams)] for _ in range(10)]
    torch.cuda.synchronize()
    for each in got:
        for y, z in zip(each, want):
            assert torch.equal(y, z)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n,k", [(1, 700, 520), (1100, 300, 2300), (40, 700, 520), (2, 33000, 300)])
def test_captured_forms(device, dtype, rows, n, k):
    """Every product's kernels as a graph, replayed on other inputs between eager calls."""
    w = weight(2, n, k, 128, "i4")
    x, bias = torch.randn(rows, k, generator=generator(1), device="cuda").to(dtype), torch.randn(n, generator=generator(2), device="cuda")
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        w4.linear(x, w, bias, gelu=True)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        y = w4.linear(x, w, bias, gelu=True)
    for seed in range(4):
        x.copy_(torch.randn(rows, k, generator=generator(30 + seed), device="cuda"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, w4.linear(x, w, bias, gelu=True))
