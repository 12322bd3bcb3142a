"""dfgpt2_token_logprobs and its backward on the GPU against float64 on the CPU: log probabilities, entropy,
alternatives (ties by the lowest id) and the logits' gradient, at odd sizes, masks and strides."""
import math

import numpy as np
import pytest
import torch

from dfattn import ops

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


def log_p(x):
    """(ln p, p, m, ln sum exp(x - m)) of rows x, the maximum taken off first: a row at -3.4e38 has no place for ln
    sum exp beside it, in 64 bits neither. A row of nothing but -inf: ln p = -inf, p = 0."""
    m = x.amax(1, keepdim=True)
    dead = torch.isneginf(m)
    d = torch.where(dead, torch.full_like(x, -math.inf), x - m)
    ln_s = torch.where(dead, torch.zeros_like(m), torch.log(torch.exp(d).sum(1, keepdim=True)))
    logp = d - ln_s
    return logp, torch.exp(logp), m, ln_s


def reference(x, tokens, k):
    """x float64 [rows, n] without NaN or +inf: (logprob, entropy, (m, ln S), ids, top logprobs)."""
    rows, n = x.shape
    logp, p, m, ln_s = log_p(x)
    ent = -(p * torch.where(p > 0, logp, torch.zeros_like(p))).sum(1)
    ids = torch.stack([torch.tensor(sorted(range(n), key=lambda i: (-r[i], i))[:k], dtype=torch.long)
                       for r in x.tolist()]) if k else torch.zeros(rows, 0, dtype=torch.long)
    inside = (tokens >= 0) & (tokens < n)
    lp = torch.where(inside, logp.gather(1, tokens.clamp(0, n - 1)[:, None])[:, 0], torch.zeros(rows, dtype=x.dtype))
    return lp, ent, torch.cat([m, ln_s], 1), ids, logp.gather(1, ids)


def tolerances(x):
    """Bounds of ln S (and a log probability but for its own rounding) and entropy, a row each, from their rounding: exp(x - m) is off by
    2^-22 and |x - m| 2^-23 relatively, S = sum by n 2^-24 at worst, of which a tree over threads leaves 64 + n /
    1024 steps; ln and the two additions round to 2^-24 of their size."""
    n = x.shape[1]
    m = x.amax(1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    d = torch.where(torch.isinf(x), torch.zeros_like(x), x - m)
    e = torch.where(torch.isneginf(x), torch.zeros_like(x), torch.exp(x - m))
    s = e.sum(1).clamp(min=1e-300)
    rel = ((2.0 ** -22 + d.abs() * 2.0 ** -23) * e).sum(1) / s + (64 + n / 1024) * 2.0 ** -24
    t_lse = rel + 2.0 ** -22 * (1 + torch.log(s).abs())
    # T = sum e d: each term off by rel plus 2^-23, sum of |e d|.
    big = (e * d.abs()).sum(1) / s
    t_ent = rel * (1 + 2 * big) + ((2.0 ** -21 + d.abs() * 2.0 ** -22) * e * d.abs()).sum(1) / s + 2.0 ** -22 * (1 + big)
    return t_lse, t_ent


def check(x, tokens, k, device, wide=0, shift=0):
    rows, n = x.shape
    if wide or shift:
        w = torch.zeros(rows, n + wide + shift, dtype=x.dtype, device=device)
        w[:, shift:shift + n] = x.to(device)
        dev = w[:, shift:shift + n]
    else:
        dev = x.to(device)
    got = ops.token_logprobs_forward(dev, tokens.int().to(device), k)
    xd = x.double()
    want = reference(xd, tokens, k)
    t_lse, t_ent = tolerances(xd)
    lp, ent, stats, ids, top = (t.cpu() for t in got)
    assert torch.equal(stats[:, 0].double(), want[2][:, 0]), "maximum"
    assert torch.equal(ids.long(), want[3]), "alternatives"
    for name, g, w, t in (("logprob", lp, want[0], t_lse + want[0].abs().nan_to_num(posinf=0) * 2.0 ** -23), ("ln S", stats[:, 1], want[2][:, 1], t_lse),
                          ("entropy", ent, want[1], t_ent),
                          ("top", top, want[4], (t_lse[:, None] + want[4].abs().nan_to_num(posinf=0) * 2.0 ** -23))):
        inf = torch.isneginf(w)
        assert torch.equal(torch.isneginf(g), inf), name
        err = torch.where(inf, torch.zeros_like(w), (g.double() - w).abs())
        assert (err <= t).all(), (name, float((err / t).max()))
    return dev, got, want


SIZES = [(1, 1, 1), (1, 2, 2), (3, 5, 3), (2, 63, 5), (2, 64, 64), (2, 65, 64), (3, 1000, 20), (2, 1023, 7), (2, 4096, 0),
         (5, 4097, 33), (2, 16384, 20), (2, 50257, 20), (3, 50304, 64), (2, 51201, 5), (2, 65537, 20), (1, 131072, 64),
         (1, 262147, 20)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n,k", SIZES)
def test_forward(device, rows, n, k, dtype):
    """bf16 logits tie often: the order of the alternatives is that of their ids."""
    say("forward", rows, n, k, dtype)
    g = torch.Generator().manual_seed(n)
    x = (torch.randn(rows, n, generator=g) * 2).to(dtype)
    tokens = torch.randint(0, n, (rows,), generator=g)
    check(x, tokens, k, device)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_in_a_wider_tensor(device, dtype):
    g = torch.Generator().manual_seed(1)
    for n, wide, shift in ((1000, 24, 0), (1001, 3, 1), (50257, 47, 0), (50257, 2, 3), (2050, 6, 2)):
        say("wide", n, wide, shift)
        check((torch.randn(3, n, generator=g) * 2).to(dtype), torch.tensor([0, n - 1, n // 2]), 9, device, wide, shift)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [700, 5000, 50257, 70000])
def test_masks_and_ties(device, n, dtype):
    """Rows of one value, masks of -inf and of the type's lowest value that leave a run, a few, one or nothing,
    and many equal largest values."""
    low = torch.finfo(dtype).min
    g = torch.Generator().manual_seed(n)
    base = torch.randn(n, generator=g)
    rows = [torch.zeros(n), torch.full((n,), low), torch.full((n,), -math.inf), torch.full((n,), -1e9)]
    for fill in (-math.inf, low, -1e9):
        for keep in (slice(0, 300), slice(n - 300, n), slice(n // 2, n // 2 + 3), slice(n - 1, n), slice(3, n, 97)):
            r = torch.full((n,), fill)
            r[keep] = base[keep]
            rows.append(r)
    r = torch.round(base)                      # many ties everywhere
    rows.append(r)
    rows.append(torch.where(base > 0, 5.0, base))  # half the row is the largest value
    rows.append(torch.where(base > 2, 50.0, base))
    rows.append(torch.arange(n) / n)           # rising and falling
    rows.append(-torch.arange(n) / n)
    rows.append(torch.arange(n) % 256 / 8.0)   # the large values at fixed places of every block
    rows.append(torch.arange(n) % 4096 / 64.0)
    z = torch.zeros(n)
    z[::2] = -0.0                              # both zeros are one value
    rows.append(z)
    x = torch.stack(rows).to(dtype)
    tokens = torch.randint(0, n, (len(rows),), generator=g)
    for k in (20, 64, 1):
        say("masks", n, dtype, k)
        check(x, tokens, k, device)


def test_nan_and_infinity(device):
    """A NaN makes its row's statistics NaN and stands first among the alternatives; +inf gives NaN too. Rows
    beside it are not touched."""
    for n in (100, 9000, 60000):
        x = torch.randn(4, n)
        clean = x.clone()
        x[1, 7], x[1, 50] = math.nan, math.nan
        x[2, 11] = math.inf
        lp, ent, stats, ids, top = (t.cpu() for t in ops.token_logprobs_forward(x.to(device), torch.zeros(4, dtype=torch.int32, device=device), 3))
        assert all(torch.isnan(t[1]).all() for t in (lp, ent, stats, top)) and ids[1, :2].tolist() == [7, 50]
        assert torch.isnan(ent[2]) and ids[2, 0] == 11
        want = ops.token_logprobs_forward(clean.to(device), torch.zeros(4, dtype=torch.int32, device=device), 3)
        for g, w in zip((lp, ent, stats, ids, top), want):
            assert torch.equal(g[[0, 3]], w.cpu()[[0, 3]])


def test_tokens_outside_the_row(device):
    x = torch.randn(4, 300)
    tokens = torch.tensor([-1, 300, 2 ** 31 - 1, 299])
    _, got, _ = check(x, tokens, 2, device)
    assert got[0][:3].tolist() == [0.0, 0.0, 0.0]
    grad = ops.token_logprobs_backward(x.to(device), tokens.int().to(device), got[2], got[1], torch.ones(4, device=device))
    assert not grad[:3].any() and grad[3].any()


def test_no_rows(device):
    x, t = torch.empty(0, 10, device=device), torch.empty(0, dtype=torch.int32, device=device)
    got = ops.token_logprobs_forward(x, t, 3)
    assert [tuple(g.shape) for g in got] == [(0,), (0,), (0, 2), (0, 3), (0, 3)]
    assert ops.token_logprobs_backward(x, t, got[2], got[1]).shape == (0, 10)


def grad_reference(x, tokens, gl, ge):
    """(gradient, p, ln p with 0 where p is 0, entropy)"""
    n = x.shape[1]
    logp, p, m, _ = log_p(x)
    ent = reference(x, tokens, 0)[1]
    logp = torch.where(p > 0, logp, torch.zeros_like(p))
    inside = ((tokens >= 0) & (tokens < n) & ~torch.isneginf(m[:, 0])).double()
    hit = torch.zeros_like(x).scatter_(1, tokens.clamp(0, n - 1)[:, None], 1.0)
    return gl[:, None] * inside[:, None] * (hit - p) - ge[:, None] * p * (logp + ent[:, None]), p, logp, ent


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n", [(1, 1), (2, 7), (3, 64), (2, 1001), (4, 4096), (2, 50257), (2, 51205), (1, 131071)])
def test_backward(device, rows, n, dtype):
    say("backward", rows, n, dtype)
    g = torch.Generator().manual_seed(n + 1)
    x = (torch.randn(rows, n, generator=g) * 3).to(dtype)
    if n > 50:
        x[0, 10:20] = -math.inf
        x[0, 21] = torch.finfo(dtype).min
    tokens = torch.randint(0, n, (rows,), generator=g)
    gl, ge = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
    t_lse, t_ent = tolerances(x.double())
    dev, td = x.to(device), tokens.int().to(device)
    _, ent, stats, _, _ = ops.token_logprobs_forward(dev, td)
    half = torch.finfo(dtype).eps / 2
    for a, b in ((gl, ge), (gl, None), (None, ge), (None, None)):
        d = lambda t: None if t is None else t.to(device)
        zero = torch.zeros(rows, dtype=torch.float64)
        a64, b64 = (zero if t is None else t.double() for t in (a, b))
        want, p, logp, h = grad_reference(x.double(), tokens, a64, b64)
        # p is off relatively by what lse is, 2^-22 for exp and |ln p| 2^-23; ln p + H by both of theirs.
        rel = t_lse[:, None] + 2.0 ** -21 + logp.abs() * 2.0 ** -22
        tol = a64.abs()[:, None] * (p * rel + 2.0 ** -22) + b64.abs()[:, None] * p * (
            (logp + h[:, None]).abs() * (rel + 2.0 ** -22) + t_lse[:, None] + t_ent[:, None] + (logp.abs() + 1) * 2.0 ** -22)
        tol = tol + want.abs() * half + 1e-38
        if dtype == torch.bfloat16:
            tol = tol + tol * half
        got = ops.token_logprobs_backward(dev, td, stats, ent, d(a), d(b)).double().cpu()
        assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol).max())
    # In place, and from a column block.
    c = dev.clone()
    whole = ops.token_logprobs_backward(dev, td, stats, ent, gl.to(device), ge.to(device))
    ops.token_logprobs_backward(c, td, stats, ent, gl.to(device), ge.to(device), out=c)
    assert torch.equal(c, whole)
    wide = torch.zeros(rows, n + 5, dtype=dtype, device=device)
    wide[:, 3:3 + n] = dev
    assert torch.equal(ops.token_logprobs_backward(wide[:, 3:3 + n], td, stats, ent, gl.to(device), ge.to(device)), whole)


def test_gradient_of_masked_rows(device):
    """A row of nothing but -inf, and one of the lowest value, have no NaN in their gradient."""
    low = torch.finfo(torch.float32).min
    x = torch.stack([torch.full((500,), -math.inf), torch.full((500,), low), torch.full((500,), low)])
    x[2, 33] = 1.0
    t = torch.tensor([3, 4, 33])
    _, got, _ = check(x, t, 3, device)
    one = torch.ones(3, device=device)
    grad = ops.token_logprobs_backward(x.to(device), t.int().to(device), got[2], got[1], one, one).cpu()
    assert not grad[0].any() and not grad[2].any()
    want = grad_reference(x.double(), t, torch.ones(3).double(), torch.ones(3).double())[0]
    assert (grad - want).abs().max() <= 2.0 ** -20  # (entropy ln 500 and ln p cancel: 8 * 2^-23 / 500 beside p's 2^-22)


def test_autograd_against_differences(device):
    """token_logprobs' gradient of a weighted sum against central differences in float64."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn(3, 41, generator=g)
    tokens = torch.tensor([5, 40, 0])
    wl, we = torch.randn(3, generator=g), torch.randn(3, generator=g)

    def f(y):
        lp, ent, _, _, _ = reference(y, tokens, 0)
        return float((wl.double() * lp + we.double() * ent).sum())

    leaf = x.to(device).requires_grad_(True)
    lp, ent, ids, top = ops.token_logprobs(leaf, tokens.int().to(device), 4)
    assert not ids.requires_grad and not top.requires_grad
    (lp * wl.to(device) + ent * we.to(device)).sum().backward()
    step = 1e-4
    for r in range(3):
        for j in range(41):
            up, down = x.double().clone(), x.double().clone()
            up[r, j] += step
            down[r, j] -= step
            # The difference is off by step^2 / 6 of the third derivative (at most 10 here), the gradient as in
            # test_backward: about 2^-19.
            assert abs(float(leaf.grad[r, j]) - (f(up) - f(down)) / (2 * step)) <= 10 * step ** 2 / 6 + 2.0 ** -18
    # Only one of the outputs used, and neither.
    a = x.to(device).requires_grad_(True)
    ops.token_logprobs(a, tokens.int().to(device))[0].sum().backward()
    want = grad_reference(x.double(), tokens, torch.ones(3).double(), torch.zeros(3).double())[0]
    assert (a.grad.double().cpu() - want).abs().max() <= 2.0 ** -19
    b = x.to(device).to(torch.bfloat16).requires_grad_(True)
    ops.token_logprobs(b, tokens.int().to(device))[1].sum().backward()
    assert b.grad.dtype == torch.bfloat16


def test_a_second_derivative_is_refused(device):
    x = torch.randn(2, 30, device=device, requires_grad=True)
    lp = ops.token_logprobs(x, torch.zeros(2, dtype=torch.int32, device=device))[0]
    (g,) = torch.autograd.grad(lp.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.square().sum(), x)


@pytest.mark.parametrize("n", [16384, 16385])
def test_many_rows_at_once(device, n):
    """More rows than run at a time, of both sides of the size where a row gets more threads."""
    g = torch.Generator().manual_seed(n)
    x = (torch.randn(16, n, generator=g) * 2).bfloat16()
    tokens = torch.randint(0, n, (16,), generator=g)
    _, got, _ = check(x, tokens, 20, device)
    many = ops.token_logprobs_forward(x.to(device).repeat(160, 1), tokens.int().to(device).repeat(160), 20)
    for a, b in zip(many, got):
        assert torch.equal(a, b.repeat(160, *[1] * (b.dim() - 1)))


def test_two_streams_at_once(device):
    sets = [(torch.randn(300, 5001, device=device), torch.randint(0, 5001, (300,), device=device).int()) for _ in range(2)]
    want = [ops.token_logprobs_forward(x, t, 7) for x, t in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], []
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((ops.token_logprobs_forward(*sets[i], 7), want[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g, w in got for a, b in zip(g, w))


def test_replayed_from_a_graph(device):
    x = torch.randn(40, 3001, device=device)
    t = torch.randint(0, 3001, (40,), device=device).int()
    gl = torch.randn(40, device=device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.token_logprobs_forward(x, t, 8)
        grad = ops.token_logprobs_backward(x, t, held[2], held[1], gl)
    for seed in range(4):
        x.copy_(torch.randn(40, 3001, generator=torch.Generator().manual_seed(seed)) * 3)
        graph.replay()
        torch.cuda.synchronize()
        want = ops.token_logprobs_forward(x, t, 8)
        assert all(torch.equal(a, b) for a, b in zip(held, want))
        assert torch.equal(grad, ops.token_logprobs_backward(x, t, want[2], want[1], gl))


def test_a_large_row_offset(device):
    """Rows whose offset passes 2^31 elements."""
    n, stride, rows = 1000, 1 << 28, 10
    big = torch.empty((rows - 1) * stride + n, dtype=torch.bfloat16, device=device).as_strided((rows, n), (stride, 1))
    x = torch.randn(rows, n, device=device).bfloat16()
    big.copy_(x)
    t = torch.randint(0, n, (rows,), device=device).int()
    for a, b in zip(ops.token_logprobs_forward(big, t, 5), ops.token_logprobs_forward(x, t, 5)):
        assert torch.equal(a, b)
