"""Serving batches of requests from a paged 8-bit cache (include/dfattn.h, dfattn_paged_plan and
dfattn_kv8_*) for PyTorch tensors.

A step of a serving loop, with nothing read on the host between the calls:

    cache = dfattn.kv8_cache(n_pages, n_kv_heads, d_head, page_size)            # once per layer
    seq_lens, query_start, slots, counts = dfattn.paged_plan(cached, new, block_table, free_pages, free_start,
                                                             page_size, n_pages, token_capacity)
    dfattn.kv8_append(cache, k, v, slots)                                       # each layer
    out, lse = dfattn.kv8_attention(cache, q, block_table, query_start, seq_lens, n_heads, max_q, max_len)
    cached.copy_(seq_lens); free_start.copy_(counts[2:])                        # before the next step

Ids and lengths are int32 tensors, activations float32 or bfloat16, a cache's codes int8 or
float8_e4m3fn. Tensors live on the current device. What a call allocates (outputs that are not given,
the workspace) belongs to the stream it runs on.
"""
from __future__ import annotations

import collections

from . import _check, _stream_ptr, _torch, lib

KV_I8, KV_E4M3 = 2, 3  # DFATTN_KV_I8, DFATTN_KV_E4M3

# Codes k [pages, kv heads, page size, Dp], v [pages, kv heads, Dp, page size] (Dp: d_head rounded up to
# 16) and their scales [pages, kv heads]; value = code * scale.
KV8Cache = collections.namedtuple("KV8Cache", "k v k_scale v_scale")


def kv8_cache(n_pages, n_kv_heads, d_head, page_size=16, dtype=None, device="cuda"):
    """An empty KV8Cache; dtype torch.int8 (the default) or torch.float8_e4m3fn."""
    torch = _torch()
    dtype = torch.int8 if dtype is None else dtype
    if dtype not in (torch.int8, torch.float8_e4m3fn):
        raise ValueError("an 8-bit cache holds int8 or float8_e4m3fn codes")
    if lib().dfattn_kv8_pool_bytes(n_pages, n_kv_heads, page_size, d_head) == 0:
        raise ValueError("n_pages and n_kv_heads must be >= 1, page_size a multiple of 16 up to 256 and d_head in "
                         "1..128")
    dp = (d_head + 15) // 16 * 16
    codes = lambda *shape: torch.zeros(shape, dtype=torch.int8, device=device).view(dtype)
    scale = lambda: torch.zeros((n_pages, n_kv_heads), dtype=torch.float32, device=device)
    return KV8Cache(codes(n_pages, n_kv_heads, page_size, dp), codes(n_pages, n_kv_heads, dp, page_size), scale(),
                    scale())


def _ptr(t, name, *dtypes):
    """Device pointer of a contiguous tensor of one of `dtypes` on the current device."""
    torch = _torch()
    if not t.is_cuda or t.dtype not in dtypes or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous device tensor of type {' or '.join(map(str, dtypes))}")
    if t.device.index != torch._C._cuda_getDevice():
        raise ValueError(f"{name} is not on the current device")
    return t.data_ptr()


def _rows(t, name, cols):
    """(pointer, row stride, type code) of a float32 or bfloat16 [rows, cols] tensor whose rows may be a
    column block of a wider one."""
    torch = _torch()
    if not t.is_cuda or t.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"{name} must be a float32 or bfloat16 device tensor")
    if t.device.index != torch._C._cuda_getDevice():
        raise ValueError(f"{name} is not on the current device")
    if t.dim() != 2 or t.shape[1] != cols or (t.stride(1) != 1 and cols > 1):
        raise ValueError(f"{name} must be [rows, {cols}] with contiguous rows")
    stride = t.stride(0) if t.shape[0] > 1 else cols
    if stride < cols:
        raise ValueError(f"{name} must be [rows, {cols}] with contiguous rows")
    return t.data_ptr(), stride, 0 if t.dtype == torch.float32 else 1


def _cache(cache, d_head=None):
    """(k, v, k_scale, v_scale pointers, kv type, kv heads, page size, pages) of a KV8Cache."""
    torch = _torch()
    k, v, ks, vs = cache
    if k.dim() != 4 or v.dim() != 4 or k.dtype != v.dtype:
        raise ValueError("a cache is (k [pages, kv heads, page size, Dp], v [pages, kv heads, Dp, page size], scales)")
    pages, heads, page, dp = k.shape
    if tuple(v.shape) != (pages, heads, dp, page) or tuple(ks.shape) != (pages, heads) or \
            tuple(vs.shape) != (pages, heads):
        raise ValueError("the cache's pools and scales disagree in shape")
    if d_head is not None and (d_head + 15) // 16 * 16 != dp:
        raise ValueError(f"the cache holds heads of {dp - 15}..{dp}, not {d_head}")
    code = torch.int8, torch.float8_e4m3fn
    return ((_ptr(k, "k codes", *code), _ptr(v, "v codes", *code), _ptr(ks, "k scales", torch.float32),
             _ptr(vs, "v scales", torch.float32)), KV_I8 if k.dtype == torch.int8 else KV_E4M3, heads, page, pages)


class _On:
    """Allocations under `stream` where one is given (memory then belongs to it)."""

    def __init__(self, stream):
        self.c = None if stream is None else _torch().cuda.stream(stream)

    def __enter__(self):
        if self.c is not None:
            self.c.__enter__()

    def __exit__(self, *e):
        if self.c is not None:
            self.c.__exit__(*e)


def _same(t, name, shape):
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must have the shape {list(shape)}")


def paged_plan(cached_lens, new_lens, block_table, free_pages, free_start, page_size, n_pages, token_capacity,
               seq_lens=None, query_start=None, slot_map=None, counts=None, stream=None):
    """dfattn_paged_plan: cached_lens, new_lens [R]; block_table [R, max_pages], whose new entries are written;
    free_pages [n] and free_start [1]. Returns (seq_lens [R], query_start [R+1], slot_map [token_capacity], counts
    [3] = requests admitted, tokens, the next free_start)."""
    torch = _torch()
    i32 = torch.int32
    r, dev = cached_lens.numel(), cached_lens.device
    if block_table.dim() != 2 or block_table.shape[0] != r or new_lens.numel() != r or free_start.numel() != 1:
        raise ValueError("cached_lens and new_lens are [R], block_table [R, max_pages], free_start [1]")
    with _On(stream):
        seq_lens = torch.empty(r, dtype=i32, device=dev) if seq_lens is None else seq_lens
        query_start = torch.empty(r + 1, dtype=i32, device=dev) if query_start is None else query_start
        slot_map = torch.empty(token_capacity, dtype=i32, device=dev) if slot_map is None else slot_map
        counts = torch.empty(3, dtype=i32, device=dev) if counts is None else counts
    _same(seq_lens, "seq_lens", (r,))
    _same(query_start, "query_start", (r + 1,))
    _same(slot_map, "slot_map", (token_capacity,))
    _same(counts, "counts", (3,))
    _check(lib().dfattn_paged_plan(
        _ptr(cached_lens, "cached_lens", i32), _ptr(new_lens, "new_lens", i32), _ptr(free_pages, "free_pages", i32),
        _ptr(free_start, "free_start", i32), _ptr(block_table, "block_table", i32), _ptr(seq_lens, "seq_lens", i32),
        _ptr(query_start, "query_start", i32), _ptr(slot_map, "slot_map", i32), _ptr(counts, "counts", i32),
        free_pages.numel(), r, block_table.shape[1], token_capacity, page_size, n_pages, _stream_ptr(stream)))
    return seq_lens, query_start, slot_map, counts


def kv8_append(cache, k, v, slot_map, stream=None):
    """dfattn_kv8_append: rows k, v [n, kv heads * d_head] (float32 or bfloat16; one row stride, so column blocks
    of a fused projection will do) into the slots slot_map [n] of `cache`."""
    heads = cache[0].shape[1]
    n, dm = k.shape
    if dm % heads:
        raise ValueError("k and v must be [n, kv heads * d_head]")
    ptrs, kv, heads, page, pages = _cache(cache, dm // heads)
    (pk, sk, tk), (pv, sv, tv) = _rows(k, "k", dm), _rows(v, "v", dm)
    if v.shape[0] != n or tk != tv or sk != sv:
        raise ValueError("k and v must share their shape, type and row stride")
    _same(slot_map, "slot_map", (n,))
    _check(lib().dfattn_kv8_append(pk, pv, _ptr(slot_map, "slot_map", _torch().int32), *ptrs, tk, kv, n, heads,
                                   dm // heads, page, pages, sk, _stream_ptr(stream)))


def kv8_read(cache, slots, d_head, dtype=None, k_out=None, v_out=None, stream=None):
    """dfattn_kv8_read: (k, v) [n, kv heads * d_head], the values in slots [n] of `cache`, in `dtype`
    (float32 by default, or bfloat16)."""
    torch = _torch()
    ptrs, kv, heads, page, pages = _cache(cache, d_head)
    shape = (slots.numel(), heads * d_head)
    dtype = (torch.float32 if k_out is None else k_out.dtype) if dtype is None else dtype
    with _On(stream):
        k_out = torch.empty(shape, dtype=dtype, device=slots.device) if k_out is None else k_out
        v_out = torch.empty(shape, dtype=dtype, device=slots.device) if v_out is None else v_out
    _same(k_out, "k_out", shape)
    _same(v_out, "v_out", shape)
    if dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("values are read as float32 or bfloat16")
    _check(lib().dfattn_kv8_read(*ptrs, _ptr(slots, "slots", torch.int32), _ptr(k_out, "k_out", dtype),
                                 _ptr(v_out, "v_out", dtype), 0 if dtype == torch.float32 else 1, kv, slots.numel(),
                                 heads, d_head, page, pages, _stream_ptr(stream)))
    return k_out, v_out


def kv8_attention_workspace_bytes(n_requests, n_tokens, max_query_len, max_seq_len, n_heads, n_kv_heads, d_head):
    return int(lib().dfattn_kv8_attention_workspace_bytes(n_requests, n_tokens, max_query_len, max_seq_len, n_heads,
                                                          n_kv_heads, d_head))


def kv8_attention(cache, q, block_table, query_start, seq_lens, n_heads, max_query_len, max_seq_len, scale=None,
                  causal=True, out=None, lse=None, workspace="auto", stream=None):
    """dfattn_kv8_attention: q [n, n_heads * d_head] (float32 or bfloat16, rows may be a column block), the tokens of
    R requests packed by query_start [R+1], against seq_lens [R] cached positions in block_table [R, max_pages].
    max_query_len, max_seq_len: bounds of the lengths. workspace: "auto" allocates
    dfattn_kv8_attention_workspace_bytes, None does not split the keys. Returns (out [n, n_heads * d_head] in q's type,
    lse [n_heads, n])."""
    torch = _torch()
    i32 = torch.int32
    if q.dim() != 2 or q.shape[1] % n_heads:
        raise ValueError("q must be [n, n_heads * d_head]")
    n, dm = q.shape
    d_head = dm // n_heads
    ptrs, kv, heads, page, pages = _cache(cache, d_head)
    r = seq_lens.numel()
    if block_table.dim() != 2 or block_table.shape[0] != r or query_start.numel() != r + 1:
        raise ValueError("seq_lens is [R], query_start [R+1], block_table [R, max_pages]")
    pq, sq, act = _rows(q, "q", dm)
    with _On(stream):
        out = torch.empty((n, dm), dtype=q.dtype, device=q.device) if out is None else out
        lse = torch.empty((n_heads, n), dtype=torch.float32, device=q.device) if lse is None else lse
        if isinstance(workspace, str):
            need = kv8_attention_workspace_bytes(r, n, max_query_len, max_seq_len, n_heads, heads, d_head)
            workspace = torch.empty(need // 4, dtype=torch.float32, device=q.device) if need else None
    _same(out, "out", (n, dm))
    _same(lse, "lse", (n_heads, n))
    ws, ws_bytes = (None, 0) if workspace is None else (_ptr(workspace, "workspace", torch.float32),
                                                        workspace.numel() * 4)
    _check(lib().dfattn_kv8_attention(
        pq, *ptrs, _ptr(block_table, "block_table", i32), _ptr(query_start, "query_start", i32),
        _ptr(seq_lens, "seq_lens", i32), _ptr(out, "out", q.dtype), _ptr(lse, "lse", torch.float32), act, kv, r, n,
        max_query_len, max_seq_len, n_heads, heads, d_head, page, pages, block_table.shape[1], sq,
        d_head ** -0.5 if scale is None else scale, int(bool(causal)), ws, ws_bytes, _stream_ptr(stream)))
    return out, lse
