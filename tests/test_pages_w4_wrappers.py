"""The wrappers of the page calls and the 4-bit linear layers, on tensors without a device: what they refuse before the
library is called."""
import pytest
import torch

import dfattn
from dfattn import kv8, w4

BIG = 1 << 32


@pytest.fixture
def here(monkeypatch):
    """Tensors without a device of their own count as being on the current one; nothing may reach the library but the
    questions for a workspace's size."""
    names = (torch, torch.int32, torch.float32, torch.bfloat16, torch.int8, torch.float8_e4m3fn, -1)
    for module in (kv8, w4):
        monkeypatch.setattr(module, "_names", lambda: names)
        monkeypatch.setattr(module, "_stream_ptr", lambda s: None)

    class Lib:
        def dfattn_paged_workspace_bytes(self, *_):
            return 64

        def dfgpt2_w4_linear_workspace_bytes(self, *_):
            return 0

        def __getattr__(self, name):
            def called(*_):
                raise AssertionError(f"{name} was called")

            return called

    monkeypatch.setattr(kv8, "lib", Lib)
    monkeypatch.setattr(w4, "ops_lib", Lib)


def meta(*shape, dtype=torch.int32):
    return torch.empty(shape, dtype=dtype, device="meta")


def weight(n=10, k=100, group=64):
    return w4.Weight(meta(n, w4.row_bytes(k), dtype=torch.uint8), meta(-(-k // group), n, dtype=torch.bfloat16), None, k, group, "i4")


# ---------------------------------------------------------------- sizes: the entry points take 32 bits, ctypes takes the rest off
@pytest.mark.parametrize("pools", [[meta(BIG + 4, 1, dtype=torch.int8)], [meta(BIG, 2, dtype=torch.bfloat16)] * 2])
def test_pools_of_too_many_pages(here, pools):
    with pytest.raises(ValueError):
        dfattn.page_pools(pools)
    with pytest.raises(ValueError):
        dfattn.paged_copy(pools, meta(3), meta(3))


def test_too_many_copies(here):
    with pytest.raises(ValueError):
        dfattn.paged_copy([meta(4, 2)], meta(BIG + 1), meta(BIG + 1))


@pytest.mark.parametrize("r,width,n", [(BIG + 4, 1, 3), (4, BIG + 8, 3), (4, 8, BIG + 3)])
def test_tables_too_large(here, r, width, n):
    table, lens = meta(r, width), meta(r)
    with pytest.raises(ValueError):
        dfattn.paged_fork(table, lens, meta(n), 16, 100)
    if n < BIG:
        with pytest.raises(ValueError):
            dfattn.paged_free(table, lens, 16, 100)
        with pytest.raises(ValueError):
            dfattn.paged_compact(table, lens, 16, 100)


@pytest.mark.parametrize("rows,n,k", [(BIG + 5, 10, 1), (3, BIG + 10, 1), (3, 1, BIG + 100)])
def test_layers_too_large(here, rows, n, k):
    w = weight(n, k)
    with pytest.raises(ValueError):
        w4.linear(meta(rows, k, dtype=torch.bfloat16), w)
    with pytest.raises(ValueError):
        w4.linear_workspace_bytes(rows, k, n)
    if rows < BIG:
        with pytest.raises(ValueError):
            w4.dequantize(w)
        with pytest.raises(ValueError):
            w4.quantize(meta(n, k, dtype=torch.bfloat16))


# ---------------------------------------------------------------- gradients: none is lost without a word
def activations(n, wants):
    t = torch.empty(3, n, device="meta")
    return t.requires_grad_() if wants else t


@pytest.mark.parametrize("wants", ["bias", "scales", "out"])
def test_linear_refuses_gradients(here, wants):
    bias = torch.empty(10, device="meta").requires_grad_(wants == "bias")
    w = weight()
    w.scales.requires_grad_(wants == "scales")
    out = activations(10, wants == "out")
    with pytest.raises(ValueError, match="gradient"):
        w4.linear(activations(100, False), w, bias, out=out)
    with torch.no_grad(), pytest.raises(AssertionError, match="was called"):
        w4.linear(activations(100, False), w, bias, out=out)


def test_dequantize_refuses_gradients(here):
    w = weight()
    w.scales.requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        w4.dequantize(w)
    with torch.no_grad(), pytest.raises(AssertionError, match="was called"):
        w4.dequantize(w)


@pytest.mark.parametrize("wants", ["x", "residual", "bias"])
@pytest.mark.parametrize("grad", [True, False])
def test_linear_refuses_tangents(here, wants, grad):
    """Forward mode goes on under torch.no_grad()."""
    from torch.autograd import forward_ad

    t = dict(x=activations(100, False), residual=activations(10, False), bias=torch.empty(10, device="meta"))
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(AssertionError, match="was called"):
            w4.linear(t["x"], weight(), t["bias"], t["residual"])
        t[wants] = forward_ad.make_dual(t[wants], torch.empty_like(t[wants]))
        with pytest.raises(ValueError, match="gradient"):
            w4.linear(t["x"], weight(), t["bias"], t["residual"])


# ---------------------------------------------------------------- memory
@pytest.mark.parametrize("n_pages", [131073, 500000])
def test_scratch_goes_with_the_call(here, monkeypatch, n_pages):
    """What a program keeps of a call from step to step keeps none of its workspace (8 bytes a page)."""
    class Lib:
        dfattn_paged_workspace_bytes = lambda self, rows, pages: 4 * (2 * pages + 1025 + rows)
        dfattn_paged_fork = dfattn_paged_free = dfattn_paged_compact = lambda self, *_: 0

    monkeypatch.setattr(kv8, "lib", Lib)
    table, lens = meta(4, 8), meta(4)
    for tensors in (dfattn.paged_fork(table, lens, meta(6), 16, n_pages)[1:], dfattn.paged_free(table, lens, 16, n_pages),
                    dfattn.paged_compact(table, lens, 16, n_pages)[1:]):
        held = {t.untyped_storage()._cdata: t.untyped_storage().nbytes() for t in tensors}
        assert sum(held.values()) == 4 * sum(t.numel() for t in tensors)
