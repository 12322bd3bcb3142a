"""The 4-bit quantiser's codes at and next to ties, as codes: scales are exact there, so each expected code is the rule's."""
import pytest
import torch

from dfattn import w4

pytestmark = pytest.mark.gpu

# Scales with at most 4 bits: every value below is a bf16 number.
SCALES = [1.0, 1.5, 0.875, 2.0 ** -20, 1.25 * 2.0 ** 30, 2.0 ** -110]
GROUPS = (32, 64, 128)


def codes_of(rows, group, fmt, dtype):
    """(codes, scales, zeros) of lists of values, a group each, filled with zeros."""
    w = torch.zeros(len(rows), group, dtype=torch.float64)
    for i, r in enumerate(rows):
        w[i, :len(r)] = torch.tensor(r, dtype=torch.float64)
    got = w.to(dtype).cuda()
    assert torch.equal(got.double().cpu(), w)  # (the values are the type's)
    q = w4.quantize(got, group, fmt)
    codes = torch.stack([q.codes & 15, q.codes >> 4], 2).reshape(len(rows), -1).tolist()
    return [c[:len(r)] for c, r in zip(codes, rows)], q.scales[0].double().tolist(), None if q.zeros is None else q.zeros[0].tolist()


def next_to(x, up):
    t = torch.tensor(x, dtype=torch.float32)
    return torch.nextafter(t, torch.tensor(float("inf") if up else float("-inf"))).item()


@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_e2m1(device, group, dtype):
    """Half way between two of the numbers the even code is taken; next to it (fp32) the nearer one."""
    ties = [(0.25, 0, 1), (0.75, 2, 1), (1.25, 2, 3), (1.75, 4, 3), (2.5, 4, 5), (3.5, 6, 5), (5.0, 6, 7)]  # value, even code, odd code
    rows, want = [], []
    for s in SCALES:
        for sign in (1, -1):
            row, codes = [6 * s], [7]
            for v, even, odd in ties:
                row.append(sign * v * s)
                codes.append(even + (8 if sign < 0 else 0))
                if dtype is torch.float32:
                    low, high = min(even, odd), max(even, odd)
                    for up, code in ((True, high if sign > 0 else low), (False, low if sign > 0 else high)):
                        row.append(next_to(sign * v * s, up))
                        codes.append(code + (8 if sign < 0 else 0))
            rows.append(row)
            want.append(codes)
    got, scales, _ = codes_of(rows, group, "e2m1", dtype)
    assert scales == [s for s in SCALES for _ in range(2)]
    zero = lambda codes: [0 if c == 8 else c for c in codes]  # (0 has two codes)
    assert [zero(c) for c in got] == [zero(c) for c in want]


@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_i4(device, group, dtype):
    rows, want = [], []
    for s in SCALES:
        for sign in (1, -1):
            halves = [sign * (j + 0.5) for j in range(7)]
            rows.append([7 * s] + [h * s for h in halves])
            want.append([15] + [round(h) + 8 for h in halves])
            if dtype is torch.float32:
                rows.append([-7 * s] + [next_to(h * s, up) for h in halves for up in (True, False)])
                want.append([1] + [(int(h + 0.5) if up else int(h - 0.5)) + 8 for h in halves for up in (True, False)])
    got, scales, _ = codes_of(rows, group, "i4", dtype)
    assert got == want and set(scales) == set(SCALES)


@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_u4(device, group, dtype):
    """A range of exactly 15 scales: zero is -low / scale rounded, a code the quotient rounded (each to the nearest, ties to even)
    plus zero, in 0..15."""
    rows, want, zeros, steps = [], [], [], []
    for s in SCALES:
        for twice in range(31):
            low = twice / 2  # 0, 1/2, .. 15
            zero = round(low)
            inside = [j + 0.5 - 15 for j in range(30) if -low <= j + 0.5 - 15 <= 15 - low] + [j - 15 for j in range(31) if -low <= j - 15 <= 15 - low][::5]
            rows.append([-low * s, (15 - low) * s] + [x * s for x in inside])
            want.append([min(15, max(0, round(x) + zero)) for x in [-low, 15 - low] + inside])
            zeros.append(zero)
            steps.append(s)
    assert max(map(len, rows)) <= 32
    got, scales, z = codes_of(rows, group, "u4", dtype)
    assert scales == steps and z == zeros and got == want


def test_past_32_bits(device):
    """A matrix of more than 2^32 weights: rows of it against the same rows by themselves, quantised and read back."""
    n, k, rows = 70000, 65536, 6
    pick = [0, 1, 32768, 65535, 65536, n - 1]
    g = torch.Generator(device="cuda").manual_seed(2)
    few = torch.randn(rows, k, generator=g, device="cuda").bfloat16()
    w = torch.zeros(n, k, dtype=torch.bfloat16, device="cuda")
    assert w.numel() > 1 << 32
    w[pick] = few
    for fmt in ("i4", "u4", "e2m1"):
        q, small = w4.quantize(w, 128, fmt), w4.quantize(few, 128, fmt)
        assert torch.equal(q.codes[pick], small.codes) and torch.equal(q.scales[:, pick], small.scales)
        assert q.zeros is None or torch.equal(q.zeros[:, pick], small.zeros)
        for dtype in (torch.bfloat16, torch.float32):
            values = w4.dequantize(q, dtype)
            assert torch.equal(values[pick], w4.dequantize(small, dtype))
            values[pick] = 0
            assert not values.any()
            del values
