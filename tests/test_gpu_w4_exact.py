"""Linear layers with 4-bit weights (dfgpt2_w4_linear) over many inputs, with bounds that do not grow with their number.

test_whole_numbers. Activations are whole numbers of up to 3, scales 1/2, 1 or 2, bias and residual whole numbers of up to 100. Every
term code x scale and zero x scale is a multiple of 1/4 of at most 90, so that with up to 20000 inputs each partial sum, in whatever
order and however grouped, is a multiple of 1/4 below 1.8 * 2^20: fp32 holds them all, and the result is exact (bf16: rounded once).

test_one_at_a_time. One activation a row: bf16 ones of 8 bits make exact results, since code x has 12 bits and its scale 8 more; for fp32 ones of 24
bits the code's product (28 bits, added up from three) is rounded at most twice to 24 bits at up to 15 |x| scale, the zero point's share and
the scaled sum once each: 3 * 15 |x| scale and |result|, times 2^-24.

test_many_terms. Random fp32 activations. A group's sum has up to `group` roundings, of partial sums whose squares are at most the
group's sum of squares S_g on the mean (terms of random sign), the sum over the n groups n more, of at most all of S = sum S_g. A
rounding is off by at most 2^-23 of its partial sum (nearest: half of that). Errors of random sign add up in squares: group * sum S_g + n S,
times 2^-46, plus the result's own rounding. The mean over all outputs of error^2 over that is at most 1.
"""
import pytest
import torch

from dfattn import w4
from test_gpu_w4 import generator, values, weight

pytestmark = pytest.mark.gpu

FORMATS = [(f, g) for f in ("i4", "u4", "e2m1") for g in (32, 64, 128)]

# By the forms that the sizes reach: one and two rows, 3 to 16, up to 1024 of small layers, 17 and more with the inputs shared out over
# workgroups, over two halves of a workgroup (bf16; 500 rows in one launch, 128 in two) and not at all; K even and odd in tiles of 128.
SIZES = [(1, 140, 2048), (2, 140, 4321), (1, 33, 20000), (2, 33, 20000), (2, 33000, 2048), (7, 70, 4321), (16, 140, 9000), (16, 33, 20000), (9, 8210, 4321),
         (17, 33, 20000), (64, 300, 2048), (200, 140, 4321), (64, 1100, 4321), (200, 1100, 9000), (128, 2300, 4000), (500, 1700, 2048),
         (500, 1700, 3900), (500, 4096, 2900), (1030, 140, 4321), (1030, 33, 20000), (2100, 1100, 2048)]


def whole(seed, n, k, group, fmt):
    w = weight(seed, n, k, group, fmt)
    steps = torch.randint(-1, 2, w.scales.shape, generator=generator(seed + 1), device="cuda")
    return w._replace(scales=torch.exp2(steps.float()).bfloat16())


@pytest.mark.parametrize("fmt,group", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n,k", SIZES)
def test_whole_numbers(device, fmt, group, dtype, rows, n, k):
    g = generator(rows + k)
    small = lambda most, *shape: torch.randint(-most, most + 1, shape, generator=g, device="cuda").float()
    w, x = whole(21, n, k, group, fmt), small(3, rows, k)
    want = x.double() @ values(w).t().contiguous()
    assert torch.equal(w4.linear(x.to(dtype), w), want.to(dtype))
    bias, residual = small(100, n), small(100, rows, n)
    want = want + bias.double() + residual.double()
    assert torch.equal(w4.linear(x.to(dtype), w, bias, residual.to(dtype)), want.to(dtype))
    assert torch.equal(w4.linear(x.to(dtype), w, bias, residual.to(dtype), workspace=None), want.to(dtype))


@pytest.mark.parametrize("fmt,group", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n", [(1, 70), (2, 70), (16, 70), (64, 70), (200, 1100), (500, 1700), (1030, 140)])
def test_one_at_a_time(device, fmt, group, dtype, rows, n):
    k = 2300
    w = weight(22, n, k, group, fmt)
    bits = 24 if dtype is torch.float32 else 8
    v = (torch.randint(2 ** (bits - 1), 2 ** bits, (k,), generator=generator(1), device="cuda") | 1).to(dtype)
    exact, g = values(w), torch.arange(k, device="cuda") // group
    for first in range(0, k, rows if rows > 2 else 37):
        at = (first + torch.arange(rows, device="cuda")) % k
        x = torch.zeros(rows, k, device="cuda", dtype=dtype)
        x[torch.arange(rows), at] = v[at]
        got = w4.linear(x, w)
        size = v[at].double()[:, None]
        want = size * exact[:, at].t()
        if dtype is torch.bfloat16:
            assert torch.equal(got, want.bfloat16()), first
        else:
            assert ((got.double() - want).abs() <= 2.0 ** -24 * (3 * 15 * size * w.scales.double()[g[at]] + want.abs())).all(), first


def squares(x, w):
    """Sum of the squares of a row's terms code x scale and zero x scale, for each output."""
    n, k = w.codes.shape[0], w.in_features
    q = torch.stack([w.codes & 15, w.codes >> 4], 2).reshape(n, -1)[:, :k].double()
    g = torch.arange(k, device=x.device) // w.group
    s = w.scales.double().t()[:, g]
    if w.format == "e2m1":
        t = values(w) ** 2
    else:
        z = torch.full_like(s, 8) if w.zeros is None else w.zeros.double().t()[:, g]
        t = (q ** 2 + z ** 2) * s ** 2
    return (x.double() ** 2) @ t.t().contiguous()


def mean_square(got, x, w):
    """The mean of error^2 over what roundings explain."""
    want = x.double() @ values(w).t().contiguous()
    groups = w.scales.shape[0]
    explained = 2.0 ** -46 * (w.group + groups) * squares(x, w) + (2.0 ** -24 * want) ** 2
    return ((got.double() - want) ** 2 / explained).mean().item()


@pytest.mark.parametrize("fmt,group", FORMATS)
@pytest.mark.parametrize("rows,n,k", [(1, 2000, 2048), (2, 2000, 4321), (2, 1000, 20000), (16, 300, 9000), (16, 140, 20000), (200, 140, 4321), (64, 1100, 4321),
                                      (500, 1700, 2048), (1030, 140, 9000), (1030, 33, 20000)])
def test_many_terms(device, fmt, group, rows, n, k):
    x, w = torch.randn(rows, k, generator=generator(k), device="cuda"), weight(23, n, k, group, fmt)
    assert mean_square(w4.linear(x, w), x, w) <= 1
    assert mean_square(w4.linear(x, w, workspace=None), x, w) <= 1
