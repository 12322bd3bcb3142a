"""dfgpt2_token_logprobs and its backward where the token itself is masked out, against float64; rows too far apart; the most
alternatives; a training step in a graph."""
import math

import pytest
import torch

import test_gpu_token_logprobs as base
from dfattn import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [2, 100, 5001, 50257])
def test_a_masked_token(device, n, dtype):
    """A token at -infinity or at the type's lowest value in a row that has others: it gets grad_logprob itself, the other
    columns what the formula says, as the gradient of a gather from log_softmax."""
    base.say("masked token", n, dtype)
    g = torch.Generator().manual_seed(n)
    x = (torch.randn(4, n, generator=g) * 3).to(dtype)
    tokens = torch.tensor([0, n - 1, n // 2, n - 1])
    for row, value in ((0, -math.inf), (1, -math.inf), (2, torch.finfo(dtype).min), (3, -math.inf)):
        x[row, tokens[row]] = value
    x[3, : n // 2] = -math.inf  # with other columns masked out beside it
    if n == 2:
        x[3, 0] = 1.0
    dev, (_, entropy, stats, _, _), want = base.check(x, tokens, 0, device)
    assert torch.isneginf(want[0][[0, 1, 3]]).all()
    gl, ge = torch.randn(4, generator=g), torch.randn(4, generator=g)
    got = ops.token_logprobs_backward(dev, tokens.int().to(device), stats, entropy, gl.to(device), ge.to(device)).cpu()
    at = torch.arange(4)
    assert torch.equal(got[at, tokens], gl.to(dtype))
    want, p, logp, h = base.grad_reference(x.double(), tokens, gl.double(), ge.double())
    # The bound of base.test_backward: half a step of each gradient's own value and what p and ln p are off by.
    t_lse, t_ent = base.tolerances(x.double())
    rel = t_lse[:, None] + 2.0 ** -21 + logp.abs() * 2.0 ** -22
    half = torch.finfo(dtype).eps / 2

    def bound(want, a, b):
        tol = a.abs()[:, None] * (p * rel + 2.0 ** -22) + b.abs()[:, None] * p * (
            (logp + h[:, None]).abs() * (rel + 2.0 ** -22) + t_lse[:, None] + t_ent[:, None] + (logp.abs() + 1) * 2.0 ** -22)
        tol = tol + want.abs() * half + 1e-38
        return tol + tol * half if dtype == torch.bfloat16 else tol

    assert ((got.double() - want).abs() <= bound(want, gl.double(), ge.double())).all()
    masked = torch.isneginf(x)
    masked[at, tokens] = False
    assert not got[masked].any()
    # torch's own answer, in float64.
    leaf = x.double().requires_grad_(True)
    torch.log_softmax(leaf, 1).gather(1, tokens[:, None])[:, 0].backward(gl.double())
    only = ops.token_logprobs_backward(dev, tokens.int().to(device), stats, entropy, gl.to(device)).double().cpu()
    assert ((only - leaf.grad).abs() <= bound(leaf.grad, gl.double(), torch.zeros(4))).all()


def test_rows_too_far_apart(device):
    """A row stride of 2^32 elements or more is refused: modulo 2^32 it is that of other rows."""
    n = 100
    far = torch.empty((1 << 32) + 4096 + n, dtype=torch.bfloat16, device=device).as_strided((2, n), ((1 << 32) + 4096, 1))
    t = torch.zeros(2, dtype=torch.int32, device=device)
    with pytest.raises(ValueError):
        ops.token_logprobs_forward(far, t)
    with pytest.raises(ValueError):
        ops.token_logprobs_backward(far, t, torch.zeros(2, 2, device=device), torch.zeros(2, device=device))
    assert ops.token_logprobs_forward(far[:1], t[:1])[0].shape == (1,)  # (one row has no stride)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_most_alternatives(device, dtype):
    """64 alternatives of many ordinary rows, of which some have more logits above the bound that 64 reach than the
    kernel keeps (7 of these in fp32)."""
    base.say("64 alternatives", dtype)
    g = torch.Generator().manual_seed(64)
    x = (torch.randn(256, 20011, generator=g) * 2).to(dtype)
    base.check(x, torch.randint(0, 20011, (256,), generator=g), 64, device)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_training_step_replayed_from_a_graph(device, dtype):
    """Forward and backward of the differentiable form captured together: every replay against the eager step."""
    rows, dim, n = 33, 16, 3001
    g = torch.Generator().manual_seed(5)
    x = torch.randn(rows, dim, generator=g).to(device).to(dtype)
    tokens = torch.randint(0, n, (rows,), generator=g).int().to(device)
    weights = [torch.randn(dim, n, generator=g).to(device).to(dtype) for _ in range(3)]

    def step(leaf):
        logprob, entropy, ids, _ = ops.token_logprobs(x @ leaf, tokens, 3)
        loss = -logprob.mean() - 0.01 * entropy.mean()
        (grad,) = torch.autograd.grad(loss, leaf)
        return loss.detach(), grad, ids

    eager = []
    for w in weights:
        base.say("eager", dtype)
        eager.append(step(w.clone().requires_grad_(True)))
    leaf = torch.zeros_like(weights[0]).requires_grad_(True)  # (no eager graph of it)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(leaf)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    base.say("capture")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(leaf)
    for _ in range(2):
        for w, want in zip(weights, eager):
            with torch.no_grad():
                leaf.copy_(w)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(held, want))
