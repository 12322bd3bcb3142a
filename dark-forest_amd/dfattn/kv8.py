"""Serving batches of requests from a paged 8-bit cache (include/dfattn.h, dfattn_paged_plan and
dfattn_kv8_*) for PyTorch tensors.

A step of a serving loop, with nothing read on the host between the calls:

    cache = dfattn.kv8_cache(n_pages, n_kv_heads, d_head, page_size)            # once per layer
    seq_lens, query_start, slots, counts = dfattn.paged_plan(cached, new, block_table, free_pages, free_start,
                                                             page_size, n_pages, token_capacity)
    dfattn.kv8_append(cache, k, v, slots)                                       # each layer
    out, lse = dfattn.kv8_attention(cache, q, block_table, query_start, seq_lens, n_heads, max_q, max_len)
    cached.copy_(seq_lens); free_start.copy_(counts[2:])                        # before the next step

Between steps requests go on more than once (beams, several answers to a prompt), or end, still with nothing read on
the host; the free list is made again from the tables:

    f = dfattn.paged_fork(block_table, cached, parents, page_size, n_pages)     # row i goes on from row parents[i]
    dfattn.paged_copy(caches, f.copy_src, f.copy_dst, f.counts)                 # all layers' caches
    block_table, cached, free_pages, free_start = f.block_table, f.seq_lens, f.free_pages, f.free_start
    refs, free_pages, free_start = dfattn.paged_free(block_table, cached, page_size, n_pages, ended)

Ids and lengths are int32 tensors, activations float32 or bfloat16, a cache's codes int8 or
float8_e4m3fn. Tensors live on the current device. What a call allocates (outputs that are not given,
the workspace) belongs to the stream it runs on.
"""
from __future__ import annotations

import array
import collections
import contextlib

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


# What every call does per argument is kept short, as in the other wrappers: a small call's kernels take 4-10 us.
# Checks go by attribute reads of 0.05 us each and by one look at the current device per call.
_torch_names = None


def _names():
    """(torch, int32, float32, bfloat16, int8, float8_e4m3fn, the current device's index)"""
    global _torch_names
    if _torch_names is None:
        torch = _torch()
        _torch_names = (torch, torch.int32, torch.float32, torch.bfloat16, torch.int8, torch.float8_e4m3fn,
                        torch._C._cuda_getDevice)
    n = _torch_names
    if not n[0].cuda.is_initialized():
        n[0].cuda.init()
    return n[:6] + (n[6](),)


def _refuse(t, name, what, dev):
    if t.is_cuda and t.get_device() != dev:
        raise ValueError(f"{name} is not on the current device")
    raise ValueError(f"{name} must be {what}")


def _ptr(t, name, dtype, dev):
    """Device pointer of a contiguous tensor of type dtype on the current device."""
    if not (t.get_device() == dev and t.dtype is dtype and t.is_contiguous()):  # (a CPU tensor's device is -1)
        _refuse(t, name, f"a contiguous device tensor of type {dtype}", dev)
    return t.data_ptr()


def _u32(x, name):
    """x, which ctypes would otherwise pass modulo 2^32."""
    if not 0 <= x < 1 << 32:
        raise ValueError(f"{name} must be at least 0 and below 2^32")
    return x


def _too_large(name):
    """For a tensor one of whose sizes ctypes would pass modulo 2^32."""
    raise ValueError(f"{name} has a size of 2^32 or more")


def _rows(t, name, cols, n):
    """(pointer, row stride, type code) of a float32 or bfloat16 [rows, cols] tensor whose rows may be a
    column block of a wider one."""
    dtype = t.dtype
    if not (t.get_device() == n[6] and (dtype is n[2] or dtype is n[3])):
        _refuse(t, name, "a float32 or bfloat16 device tensor", n[6])
    if t.dim() != 2 or t.shape[1] != cols:
        raise ValueError(f"{name} must be [rows, {cols}]")
    stride = cols
    if not t.is_contiguous():
        if t.shape[0] > 1:
            stride = t.stride(0)
        if (t.stride(1) != 1 and cols > 1) or stride < cols:
            raise ValueError(f"{name} must be [rows, {cols}] with contiguous rows")
        _u32(stride, f"{name}'s row stride")
    return t.data_ptr(), stride, 0 if dtype is n[2] else 1


def _cache(cache, d_head, n):
    """(k, v, k_scale, v_scale pointers, kv type, kv heads, page size, pages) of a KV8Cache."""
    k, v, ks, vs = cache
    if k.dim() != 4:
        raise ValueError("a cache is (k [pages, kv heads, page size, Dp], v [pages, kv heads, Dp, page size], scales)")
    pages, heads, page, dp = k.shape
    dtype, dev = k.dtype, n[6]
    if v.shape != (pages, heads, dp, page) or ks.shape != (pages, heads) or vs.shape != (pages, heads):
        raise ValueError("the cache's pools and scales disagree in shape")
    if (d_head + 15) // 16 * 16 != dp:
        raise ValueError(f"the cache holds heads of {dp - 15}..{dp}, not {d_head}")
    if dtype is not n[4] and dtype is not n[5]:
        raise ValueError("an 8-bit cache holds int8 or float8_e4m3fn codes")
    return ((_ptr(k, "k codes", dtype, dev), _ptr(v, "v codes", dtype, dev), _ptr(ks, "k scales", n[2], dev),
             _ptr(vs, "v scales", n[2], dev)), KV_I8 if dtype is n[4] else KV_E4M3, heads, page, pages)


def _check_stream(stream, dev):
    if stream is not None and stream.device_index != dev:
        raise ValueError("the stream is not on the current device")


_HERE = contextlib.nullcontext()


def _on(stream, dev):
    """Allocations under `stream` where one is given (memory then belongs to it)."""
    if stream is None:
        return _HERE
    _check_stream(stream, dev)
    return _torch().cuda.stream(stream)


def _same(t, name, shape):
    if t.shape != shape:
        raise ValueError(f"{name} must have the shape {list(shape)}")


def _out(t, name, shape, dtype, on, n):
    """(t, its pointer) of an output that the caller gave, or of a new one on device `on`."""
    if t is None:
        t = n[0].empty_strided(shape, (shape[1], 1) if len(shape) == 2 else (1,), dtype=dtype, device=on)
        return t, t.data_ptr()  # (empty takes 1.6 us, this 1.3)
    _same(t, name, shape)
    return t, _ptr(t, name, dtype, n[6])


def paged_plan(cached_lens, new_lens, block_table, free_pages, free_start, page_size, n_pages, token_capacity,
               seq_lens=None, query_start=None, slot_map=None, counts=None, stream=None):
    """dfattn_paged_plan: cached_lens, new_lens [R]; block_table [R, max_pages], whose new entries are written;
    free_pages [n] and free_start [1]. Returns (seq_lens [R], query_start [R+1], slot_map [token_capacity], counts
    [3] = requests admitted, tokens, the next free_start)."""
    names = _names()
    i32, dev = names[1], names[6]
    r = cached_lens.numel()
    if block_table.dim() != 2 or block_table.shape[0] != r or new_lens.numel() != r or free_start.numel() != 1:
        raise ValueError("cached_lens and new_lens are [R], block_table [R, max_pages], free_start [1]")
    _u32(page_size, "page_size"), _u32(n_pages, "n_pages"), _u32(token_capacity, "token_capacity")
    with _on(stream, dev):
        on = cached_lens.device
        if seq_lens is None and query_start is None and slot_map is None and counts is None:
            # One allocation in four parts (3.4 us instead of 5.2).
            whole = names[0].empty_strided((2 * r + token_capacity + 4,), (1,), dtype=i32, device=on)
            seq_lens, query_start, slot_map, counts = whole.split_with_sizes([r, r + 1, token_capacity, 3])
            ps, pq, pm, pc = seq_lens.data_ptr(), query_start.data_ptr(), slot_map.data_ptr(), counts.data_ptr()
        else:
            seq_lens, ps = _out(seq_lens, "seq_lens", (r,), i32, on, names)
            query_start, pq = _out(query_start, "query_start", (r + 1,), i32, on, names)
            slot_map, pm = _out(slot_map, "slot_map", (token_capacity,), i32, on, names)
            counts, pc = _out(counts, "counts", (3,), i32, on, names)
    _check(lib().dfattn_paged_plan(
        _ptr(cached_lens, "cached_lens", i32, dev), _ptr(new_lens, "new_lens", i32, dev),
        _ptr(free_pages, "free_pages", i32, dev), _ptr(free_start, "free_start", i32, dev),
        _ptr(block_table, "block_table", i32, dev), ps, pq, pm, pc, free_pages.numel(), r, block_table.shape[1],
        token_capacity, page_size, n_pages, _stream_ptr(stream)))
    return seq_lens, query_start, slot_map, counts


# A batch's rows after a fork: the new table and lengths, how often each page is held, the page ids (those held of the parents, the
# new ones, the free ones, each rising), the first free one's place, the pairs of pages to copy and counts [2] = pairs, rows cut for want of a page.
PagedFork = collections.namedtuple("PagedFork", "block_table seq_lens refs free_pages free_start copy_src copy_dst counts")
PagedCompact = collections.namedtuple("PagedCompact", "block_table refs free_pages free_start copy_src copy_dst counts")


def _table(block_table, seq_lens, names):
    """(pointers of both, R, max_pages) of a batch's table."""
    if block_table.dim() != 2 or seq_lens.shape != block_table.shape[:1]:
        raise ValueError("block_table is [R, max_pages], seq_lens [R]")
    i32, dev = names[1], names[6]
    r, width = block_table.shape
    if (r | width) >> 32:
        _too_large("block_table")
    return _ptr(block_table, "block_table", i32, dev), _ptr(seq_lens, "seq_lens", i32, dev), r, width


# A workspace of more words than this (1 MB, some 130000 pages) is an allocation of its own, so that a program that keeps the free list
# does not keep the scratch; up to there it stands behind the outputs, which saves a call 1.3 us on the host (10 to 14 in all).
_SCRATCH_WORDS = 1 << 18


def _parts(names, on, *sizes):
    """int32 tensors of these sizes but the last, the workspace's; the pointers of all; what must live until the call is made."""
    apart = sizes[-1] > _SCRATCH_WORDS
    new = lambda n: names[0].empty_strided((n,), (1,), dtype=names[1], device=on)
    scratch = new(sizes[-1]) if apart else None
    parts = new(sum(sizes[:-1]) if apart else sum(sizes)).split_with_sizes(sizes[:-1] if apart else sizes)
    ptrs = [t.data_ptr() for t in parts]
    return (parts, ptrs + [scratch.data_ptr()], scratch) if apart else (parts[:-1], ptrs, None)


def paged_fork(block_table, seq_lens, parents, page_size, n_pages, keep_lens=None, new_table=None, stream=None):
    """dfattn_paged_fork: row i of the result goes on from row parents[i] of block_table [R, max_pages] (none: an id
    outside 0..R-1), from its seq_lens[parents[i]] tokens or the first keep_lens[i]. new_table [n, max_pages] (allocated
    where it is not given) keeps what stands behind a row's pages. Returns a PagedFork; follow it with paged_copy."""
    names = _names()
    i32, dev = names[1], names[6]
    pt, pl, r, width = _table(block_table, seq_lens, names)
    _u32(page_size, "page_size"), _u32(n_pages, "n_pages")
    n = parents.numel()
    if n >> 32:
        _too_large("parents")
    if keep_lens is not None:
        _same(keep_lens, "keep_lens", (n,))
    ws = lib().dfattn_paged_workspace_bytes(n, n_pages)
    with _on(stream, dev):
        on = block_table.device
        if new_table is None:
            new_table = names[0].empty_strided((n, width), (width, 1), dtype=i32, device=on)
        _same(new_table, "new_table", (n, width))
        pages = n_pages if ws else 0  # (0: the call refuses the sizes)
        parts, ptrs, scratch = _parts(names, on, n, pages, pages, 1, n, n, 2, ws // 4)
    _check(lib().dfattn_paged_fork(
        pt, pl, _ptr(parents, "parents", i32, dev), None if keep_lens is None else _ptr(keep_lens, "keep_lens", i32, dev),
        _ptr(new_table, "new_table", i32, dev), *ptrs[:7], r, n, width, page_size, n_pages, ptrs[7], ws, _stream_ptr(stream)))
    return PagedFork(new_table, *parts)


def paged_free(block_table, seq_lens, page_size, n_pages, ended=None, stream=None):
    """dfattn_paged_free: seq_lens[r] becomes 0 where ended[r] is not 0 (int32). Returns (refs [n_pages], free_pages
    [n_pages], free_start [1]) of the rows that remain."""
    names = _names()
    pt, pl, r, width = _table(block_table, seq_lens, names)
    _u32(page_size, "page_size"), _u32(n_pages, "n_pages")
    if ended is not None:
        _same(ended, "ended", (r,))
    ws = lib().dfattn_paged_workspace_bytes(r, n_pages)
    with _on(stream, names[6]):
        pages = n_pages if ws else 0
        parts, ptrs, scratch = _parts(names, block_table.device, pages, pages, 1, ws // 4)
    _check(lib().dfattn_paged_free(pt, pl, None if ended is None else _ptr(ended, "ended", names[1], names[6]), *ptrs[:3],
                                   r, width, page_size, n_pages, ptrs[3], ws, _stream_ptr(stream)))
    return tuple(parts)


def paged_compact(block_table, seq_lens, page_size, n_pages, new_table=None, stream=None):
    """dfattn_paged_compact: the held pages move below their number. new_table [R, max_pages] may be block_table itself,
    which it is where it is not given. Returns a PagedCompact (counts [1]: pairs); follow it with paged_copy."""
    names = _names()
    pt, pl, r, width = _table(block_table, seq_lens, names)
    _u32(page_size, "page_size"), _u32(n_pages, "n_pages")
    new_table = block_table if new_table is None else new_table
    _same(new_table, "new_table", (r, width))
    ws = lib().dfattn_paged_workspace_bytes(r, n_pages)
    with _on(stream, names[6]):
        pages = n_pages if ws else 0
        parts, ptrs, scratch = _parts(names, block_table.device, pages, pages, 1, pages // 2, pages // 2, 1, ws // 4)
    _check(lib().dfattn_paged_compact(pt, pl, _ptr(new_table, "new_table", names[1], names[6]), *ptrs[:6], r, width,
                                      page_size, n_pages, ptrs[6], ws, _stream_ptr(stream)))
    return PagedCompact(new_table, *parts)


class PagePools:
    """The pools that paged_copy copies in (page_pools makes one): what the library takes, the tensors, their pages."""

    def __init__(self, fields, tensors, n_pages, device):
        self.fields, self.tensors, self.n_pages, self.device = fields, tensors, n_pages, device


def page_pools(pools):
    """PagePools of a list of tensors [n_pages, ...] (any type, contiguous) and of KV8Caches, to be kept by a program that
    copies in the same ones each step (the tensors must keep the memory they have now: no resize_, no new .data)."""
    if KV8Cache in map(type, pools):
        tensors = [t for p in pools for t in (p if type(p) is KV8Cache else (p,))]
    else:
        tensors = list(pools)
    dev = _names()[6]
    # (A list for each question: 48 pools 16 us, tensor after tensor 35.)
    n_pages = tensors[0].shape[0] if tensors and tensors[0].dim() else 0
    for t in [t for t in tensors if t.get_device() != dev or not t.is_contiguous()]:
        _ptr(t, "a pool", t.dtype, dev)
    sizes = [t.nbytes for t in tensors]
    try:
        same = not [t for t in tensors if t.shape[0] != n_pages]
    except IndexError:  # (a pool without dimensions)
        same = False
    if not same or n_pages == 0 or 0 in sizes:
        raise ValueError("there must be at least one pool, all [n_pages, ...] of one n_pages and not empty")
    if n_pages >> 32:
        _too_large("a pool")
    fields = array.array("Q", bytes(16 * len(tensors)))  # (a dfattn_page_pool is a pointer and a size)
    fields[0::2] = array.array("Q", [t.data_ptr() for t in tensors])
    fields[1::2] = array.array("Q", [s // n_pages for s in sizes])
    return PagePools(fields, tensors, n_pages, dev)


def paged_copy(pools, copy_src, copy_dst, n_copies=None, stream=None):
    """dfattn_paged_copy: page copy_src[m] to page copy_dst[m] of all pools (a list as page_pools takes, or what it
    returned), for the first n_copies[0] pairs (a device tensor, such as a fork's counts; None: all)."""
    names = _names()
    i32, dev = names[1], names[6]
    if not isinstance(pools, PagePools):
        pools = page_pools(pools)
    if pools.device != dev:
        raise ValueError("the pools are not on the current device")
    _check_stream(stream, dev)
    n = copy_src.numel()
    if n >> 32:
        _too_large("copy_src")
    _same(copy_src, "copy_src", (n,)), _same(copy_dst, "copy_dst", (n,))
    if n_copies is not None and n_copies.numel() < 1:
        raise ValueError("n_copies must have at least one entry")
    _check(lib().dfattn_paged_copy(
        pools.fields.buffer_info()[0], len(pools.tensors), _ptr(copy_src, "copy_src", i32, dev), _ptr(copy_dst, "copy_dst", i32, dev),
        None if n_copies is None else _ptr(n_copies, "n_copies", i32, dev), n, pools.n_pages, _stream_ptr(stream)))


def kv8_append(cache, k, v, slot_map, stream=None):
    """dfattn_kv8_append: rows k, v [n, kv heads * d_head] (float32 or bfloat16; one row stride, so column blocks
    of a fused projection will do) into the slots slot_map [n] of `cache`, each page's rows next to each other with
    consecutive slots (paged_plan's maps are so)."""
    names = _names()
    _check_stream(stream, names[6])
    n, dm = k.shape
    if dm % cache[0].shape[1]:
        raise ValueError("k and v must be [n, kv heads * d_head]")
    d_head = dm // cache[0].shape[1]
    ptrs, kv, heads, page, pages = _cache(cache, d_head, names)
    (pk, sk, tk), (pv, sv, tv) = _rows(k, "k", dm, names), _rows(v, "v", dm, names)
    if v.shape[0] != n or tk != tv or sk != sv:
        raise ValueError("k and v must share their shape, type and row stride")
    _same(slot_map, "slot_map", (n,))
    _check(lib().dfattn_kv8_append(pk, pv, _ptr(slot_map, "slot_map", names[1], names[6]), *ptrs, tk, kv, n, heads,
                                   d_head, page, pages, sk, _stream_ptr(stream)))


def kv8_read(cache, slots, d_head, dtype=None, k_out=None, v_out=None, stream=None):
    """dfattn_kv8_read: (k, v) [n, kv heads * d_head], the values in slots [n] of `cache`, in `dtype`
    (float32 by default, or bfloat16)."""
    names = _names()
    ptrs, kv, heads, page, pages = _cache(cache, d_head, names)
    n, dev = slots.numel(), names[6]
    shape = (n, heads * d_head)
    if dtype is None:
        dtype = names[2] if k_out is None else k_out.dtype
    if dtype is not names[2] and dtype is not names[3]:
        raise ValueError("values are read as float32 or bfloat16")
    with _on(stream, dev):
        k_out, pk = _out(k_out, "k_out", shape, dtype, slots.device, names)
        v_out, pv = _out(v_out, "v_out", shape, dtype, slots.device, names)
    _check(lib().dfattn_kv8_read(*ptrs, _ptr(slots, "slots", names[1], dev), pk, pv, 0 if dtype is names[2] else 1, kv, n,
                                 heads, d_head, page, pages, _stream_ptr(stream)))
    return k_out, v_out


def kv8_attention_workspace_bytes(n_requests, n_tokens, max_query_len, max_seq_len, n_heads, n_kv_heads, d_head):
    return lib().dfattn_kv8_attention_workspace_bytes(n_requests, n_tokens, max_query_len, max_seq_len, n_heads,
                                                      n_kv_heads, d_head)


def kv8_attention(cache, q, block_table, query_start, seq_lens, n_heads, max_query_len, max_seq_len, scale=None,
                  causal=True, out=None, lse=None, workspace="auto", stream=None):
    """dfattn_kv8_attention: q [n, n_heads * d_head] (float32 or bfloat16, rows may be a column block), the tokens of
    R requests packed by query_start [R+1], against seq_lens [R] cached positions in block_table [R, max_pages].
    max_query_len, max_seq_len: bounds of the lengths (a long chunk beside many requests of one token is faster in a call of
    its own). workspace: "auto" allocates
    dfattn_kv8_attention_workspace_bytes, None does not split the keys. Returns (out [n, n_heads * d_head] in q's type,
    lse [n_heads, n])."""
    names = _names()
    i32, f32, dev = names[1], names[2], names[6]
    if q.dim() != 2 or n_heads < 1 or q.shape[1] % n_heads:
        raise ValueError("q must be [n, n_heads * d_head]")
    _u32(max_query_len, "max_query_len"), _u32(max_seq_len, "max_seq_len")
    n, dm = q.shape
    d_head = dm // n_heads
    ptrs, kv, heads, page, pages = _cache(cache, d_head, names)
    r = seq_lens.numel()
    if block_table.dim() != 2 or block_table.shape[0] != r or query_start.numel() != r + 1:
        raise ValueError("seq_lens is [R], query_start [R+1], block_table [R, max_pages]")
    pq, sq, act = _rows(q, "q", dm, names)
    with _on(stream, dev):
        out, po = _out(out, "out", (n, dm), q.dtype, q.device, names)
        lse, pl = _out(lse, "lse", (n_heads, n), f32, q.device, names)
        if isinstance(workspace, str):
            need = kv8_attention_workspace_bytes(r, n, max_query_len, max_seq_len, n_heads, heads, d_head)
            workspace = names[0].empty((need // 4,), dtype=f32, device=q.device) if need else None
    ws, ws_bytes = (None, 0) if workspace is None else (_ptr(workspace, "workspace", f32, dev), workspace.numel() * 4)
    _check(lib().dfattn_kv8_attention(
        pq, *ptrs, _ptr(block_table, "block_table", i32, dev), _ptr(query_start, "query_start", i32, dev),
        _ptr(seq_lens, "seq_lens", i32, dev), po, pl, act, kv, r, n, max_query_len, max_seq_len, n_heads, heads, d_head, page,
        pages, block_table.shape[1], sq, d_head ** -0.5 if scale is None else scale, 1 if causal else 0, ws, ws_bytes,
        _stream_ptr(stream)))
    return out, lse
