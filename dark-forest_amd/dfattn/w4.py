"""Linear layers with 4-bit weights and a scale for each group of inputs (include/dfgpt2.h, dfgpt2_w4_*) for PyTorch
tensors:

    w = w4.quantize(weight, group=64, format="i4")      # once, from float32 or bfloat16 [outputs, inputs]
    y = w4.linear(x, w, bias=b, gelu=True)              # x [rows, inputs], one token or many
    x = w4.linear(y, w2, bias=b2, residual=x, out=x)

Weights made elsewhere are a Weight of their codes and scales. Nothing here has a gradient: where one would be wanted of an
argument of linear or dequantize (x, the scales, the bias, the residual, out) the call is refused, as it is where one has a
tangent of forward mode; a product that has one is torch's, with dequantize's values. Quantising rounds, and what it
returns is apart from the weight's graph. Tensors live on the current device; what a call allocates belongs to the stream it runs on.
"""
from __future__ import annotations

import collections

from . import _check, _stream_ptr
from .kv8 import _names, _on, _out, _ptr, _rows, _too_large, _u32
from .ops import ops_lib

FORMATS = {"i4": 0, "u4": 1, "e2m1": 2}  # DFGPT2_W4_I4, DFGPT2_W4_U4, DFGPT2_W4_E2M1

# codes uint8 [outputs, bytes] (input 2 b in the low half of byte b; rows of whole 16 bytes), scales bfloat16 [groups,
# outputs], zeros uint8 [groups, outputs] for "u4" (else None); value = (code - zero) * scale ("i4": zero 8), or the e2m1
# number of the code times the scale.
Weight = collections.namedtuple("Weight", "codes scales zeros in_features group format")


def row_bytes(in_features):
    """Bytes of one output's codes."""
    return -(-in_features // 32) * 16


def _weight(w, n):
    """(codes, scales, zeros pointers, format, group, outputs, inputs) of a Weight."""
    torch, dev = n[0], n[6]
    codes, scales, zeros, k, group, fmt = w
    if fmt not in FORMATS or group not in (32, 64, 128):
        raise ValueError("a weight's format is one of i4, u4 and e2m1, its group 32, 64 or 128")
    if k < 1 or codes.dim() != 2 or codes.shape[1] != row_bytes(k):
        raise ValueError(f"codes must be [outputs, {row_bytes(k)}] for {k} inputs")
    shape = (-(-k // group), codes.shape[0])
    if (shape[1] | k) >> 32:
        _too_large("codes")
    if scales.shape != shape or (fmt == "u4" and (zeros is None or zeros.shape != shape)):
        raise ValueError(f"scales (and the zeros of u4) must be {list(shape)}")
    return (_ptr(codes, "codes", torch.uint8, dev), _ptr(scales, "scales", n[3], dev),
            _ptr(zeros, "zeros", torch.uint8, dev) if fmt == "u4" else None, FORMATS[fmt], group, shape[1], k)


_forward_ad = None


def _no_gradient(torch, name, tensors):
    """Refuses a call that a gradient of one of `tensors`, or a tangent of forward mode (which torch.no_grad() leaves on),
    would be lost in."""
    global _forward_ad
    if _forward_ad is None:
        _forward_ad = torch.autograd.forward_ad
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{name} has no gradient: call it under torch.no_grad()")
    if _forward_ad._current_level >= 0 and any(t is not None and _forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError(f"{name} has no gradient of forward mode: give it the primals")


def quantize(w, group=64, format="i4", stream=None):
    """dfgpt2_w4_quantize: the Weight of w [outputs, inputs] (float32 or bfloat16, rows may be a column block)."""
    names = _names()
    torch, dev = names[0], names[6]
    if format not in FORMATS or group not in (32, 64, 128):
        raise ValueError("format is one of i4, u4 and e2m1, group 32, 64 or 128")
    if w.dim() != 2 or not w.numel():
        raise ValueError("w must be [outputs, inputs] and not empty")
    n, k = w.shape
    if (n | k) >> 32:
        _too_large("w")
    p, stride, dtype = _rows(w, "w", k, names)
    with _on(stream, dev):
        codes = torch.empty((n, row_bytes(k)), dtype=torch.uint8, device=w.device)
        scales = torch.empty((-(-k // group), n), dtype=names[3], device=w.device)
        zeros = torch.empty((-(-k // group), n), dtype=torch.uint8, device=w.device) if format == "u4" else None
    _check(ops_lib().dfgpt2_w4_quantize(p, codes.data_ptr(), scales.data_ptr(), None if zeros is None else zeros.data_ptr(),
                                        dtype, FORMATS[format], group, n, k, stride, _stream_ptr(stream)))
    return Weight(codes, scales, zeros, k, group, format)


def dequantize(w, dtype=None, out=None, stream=None):
    """dfgpt2_w4_dequantize: the values of a Weight, [outputs, inputs] in `dtype` (float32 by default, or bfloat16)."""
    names = _names()
    *ptrs, fmt, group, n, k = _weight(w, names)
    if dtype is None:
        dtype = names[2] if out is None else out.dtype
    if dtype is not names[2] and dtype is not names[3]:
        raise ValueError("values are read as float32 or bfloat16")
    _no_gradient(names[0], "dequantize", (w[1], out))
    with _on(stream, names[6]):
        out, p = _out(out, "out", (n, k), dtype, w.codes.device, names)
    _check(ops_lib().dfgpt2_w4_dequantize(*ptrs, p, 0 if dtype is names[2] else 1, fmt, group, n, k, _stream_ptr(stream)))
    return out


def linear_workspace_bytes(rows, in_features, out_features):
    _u32(rows, "rows"), _u32(in_features, "in_features"), _u32(out_features, "out_features")
    return ops_lib().dfgpt2_w4_linear_workspace_bytes(rows, in_features, out_features)


def linear(x, w, bias=None, residual=None, gelu=False, out=None, workspace="auto", stream=None):
    """dfgpt2_w4_linear: x W^T + bias, then GELU where gelu is true, then + residual; x [rows, inputs] (float32 or
    bfloat16, rows may be a column block), bias [outputs] float32, residual and out [rows, outputs] in x's type (out may be
    the residual). workspace: "auto" allocates dfgpt2_w4_linear_workspace_bytes, None does without."""
    names = _names()
    dev = names[6]
    *ptrs, fmt, group, n, k = _weight(w, names)
    px, stride, dtype = _rows(x, "x", k, names)
    _no_gradient(names[0], "linear", (x, w[1], bias, residual, out))
    shape = (x.shape[0], n)
    if shape[0] >> 32:
        _too_large("x")
    if bias is not None and bias.shape != (n,):
        raise ValueError(f"bias must be [{n}]")
    if residual is not None and residual.shape != shape:
        raise ValueError(f"residual must be {list(shape)}")
    with _on(stream, dev):
        out, po = _out(out, "out", shape, x.dtype, x.device, names)
        if isinstance(workspace, str):
            need = ops_lib().dfgpt2_w4_linear_workspace_bytes(shape[0], k, n) if shape[0] > 1 else 0
            workspace = names[0].empty((need // 4,), dtype=names[2], device=x.device) if need else None
    ws, ws_bytes = (None, 0) if workspace is None else (_ptr(workspace, "workspace", names[2], dev), workspace.numel() * 4)
    _check(ops_lib().dfgpt2_w4_linear(
        px, *ptrs, None if bias is None else _ptr(bias, "bias", names[2], dev),
        None if residual is None else _ptr(residual, "residual", x.dtype, dev), po, dtype, fmt, group, shape[0], k, n, stride,
        1 if gelu else 0, ws, ws_bytes, _stream_ptr(stream)))
    return out
