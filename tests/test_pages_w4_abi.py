"""Refusals of the page calls and the 4-bit linear layers, on the CPU: everything here is caught on the host before any
HIP call."""
import ctypes

import pytest
import torch

import dfattn
from dfattn import kv8, ops, w4

NULL, MIS, SHAPE, OVER, WORK, FLAGS = -1, -2, -3, -5, -6, -8
STEP = 0x100000


def expect(status, fn, args):
    lib = ops.ops_lib()
    lib.dfattn_clear_error()
    assert getattr(lib, fn)(*args) == status
    assert lib.dfattn_last_error() == status
    if status:
        assert fn.encode() in lib.dfattn_last_error_message()
    lib.dfattn_clear_error()


def at(i, shift=0):
    return ctypes.c_void_p(STEP * (i + 1) + shift)


def pointers(n, changes):
    p = [at(i) for i in range(n)]
    for i, x in (changes or {}).items():
        p[i] = x
    return p


SIZES = [(dict(r=0), SHAPE), (dict(width=0), SHAPE), (dict(page=0), SHAPE), (dict(pages=0), SHAPE), (dict(r=8193), OVER),
         (dict(pages=(1 << 24) + 1), OVER), (dict(pages=1 << 20, page=4096), OVER), (dict(width=1 << 28), OVER),
         (dict(ws=None), WORK), (dict(ws_bytes=8), WORK), (dict(ws=ctypes.c_void_p(0x90000002)), MIS)]


def fork(ptrs=None, r=4, n=6, width=8, page=16, pages=100, ws=ctypes.c_void_p(0x90000000), ws_bytes=1 << 20):
    return pointers(12, ptrs) + [r, n, width, page, pages, ws, ws_bytes, None]


@pytest.mark.parametrize("kw,status", SIZES + [(dict(n=0), SHAPE), (dict(n=8193), OVER),
    *[(dict(ptrs={i: None}), NULL) for i in range(12) if i != 3], *[(dict(ptrs={i: at(i, 2)}), MIS) for i in range(12)],
    (dict(ptrs={4: at(0)}), SHAPE),            # new_table in place of block_table
    (dict(ptrs={5: at(1, 12)}), SHAPE),        # new_lens over the last seq_lens
    (dict(ptrs={9: at(2)}), SHAPE), (dict(ptrs={3: at(10)}), SHAPE), (dict(ptrs={6: at(7, 396)}), SHAPE),
    (dict(ptrs={8: at(11, 4)}), SHAPE),        # free_start inside counts
    (dict(ws=at(6, 4)), SHAPE)])
def test_fork(kw, status):
    expect(status, "dfattn_paged_fork", fork(**kw))


def free(ptrs=None, r=4, width=8, page=16, pages=100, ws=ctypes.c_void_p(0x90000000), ws_bytes=1 << 20):
    return pointers(6, ptrs) + [r, width, page, pages, ws, ws_bytes, None]


@pytest.mark.parametrize("kw,status", SIZES + [
    *[(dict(ptrs={i: None}), NULL) for i in range(6) if i != 2], *[(dict(ptrs={i: at(i, 2)}), MIS) for i in range(6)],
    (dict(ptrs={2: at(1)}), SHAPE), (dict(ptrs={3: at(0, 4)}), SHAPE), (dict(ptrs={5: at(4)}), SHAPE), (dict(ws=at(0)), SHAPE)])
def test_free(kw, status):
    expect(status, "dfattn_paged_free", free(**kw))


def compact(ptrs=None, r=4, width=8, page=16, pages=100, ws=ctypes.c_void_p(0x90000000), ws_bytes=1 << 20):
    return pointers(9, ptrs) + [r, width, page, pages, ws, ws_bytes, None]


@pytest.mark.parametrize("kw,status", SIZES + [
    *[(dict(ptrs={i: None}), NULL) for i in range(9)], *[(dict(ptrs={i: at(i, 2)}), MIS) for i in range(9)],
    (dict(ptrs={2: at(0, 4)}), SHAPE), (dict(ptrs={2: at(1)}), SHAPE), (dict(ptrs={6: at(7, 196)}), SHAPE),
    (dict(ptrs={8: at(1, 8)}), SHAPE), (dict(ws=at(1)), SHAPE)])
def test_compact(kw, status):
    expect(status, "dfattn_paged_compact", compact(**kw))


def copy(pools=((0x10000, 64),), ptrs=None, n=3, pages=10, n_pools=None, array="array"):
    a = (ctypes.c_size_t * (2 * len(pools) + 1))(*[x for p in pools for x in p], 0)
    return [ctypes.cast(a, ctypes.c_void_p) if array == "array" else array, len(pools) if n_pools is None else n_pools] + \
        pointers(3, ptrs) + [n, pages, None]


@pytest.mark.parametrize("kw,status", [
    (dict(pages=0), SHAPE), (dict(pages=(1 << 24) + 1), OVER), (dict(n=(1 << 24) + 1), OVER), (dict(n_pools=65536), OVER),
    (dict(n=0), 0), (dict(n_pools=0), 0), (dict(array=None), NULL), (dict(array=ctypes.c_void_p(0x1004)), MIS),
    (dict(ptrs={0: None}), NULL), (dict(ptrs={1: None}), NULL), (dict(ptrs={0: at(0, 2)}), MIS), (dict(ptrs={1: at(0, 1)}), MIS),
    (dict(ptrs={2: at(2, 2)}), MIS), (dict(pools=((0, 64),)), NULL), (dict(pools=((0x10000, 64), (0x20000, 0))), SHAPE),
    (dict(pools=((0x10000, (1 << 30) + 16),)), OVER)])
def test_copy(kw, status):
    expect(status, "dfattn_paged_copy", copy(**kw))


def test_workspace():
    f = dfattn.lib().dfattn_paged_workspace_bytes
    assert f(0, 5) == f(5, 0) == f(8193, 5) == f(5, (1 << 24) + 1) == 0
    assert 0 < f(1, 1) <= f(8192, 1 << 24) < 1 << 28


WEIGHTS = [(dict(dtype=2), FLAGS), (dict(fmt=3), FLAGS), (dict(group=16), SHAPE), (dict(group=256), SHAPE), (dict(group=0), SHAPE),
           (dict(n=0), SHAPE), (dict(k=0), SHAPE), (dict(n=(1 << 24) + 1), OVER)]


def quantize(ptrs=None, dtype=0, fmt=1, group=64, n=10, k=100, stride=None):
    return pointers(4, ptrs) + [dtype, fmt, group, n, k, k if stride is None else stride, None]


@pytest.mark.parametrize("kw,status", WEIGHTS + [
    *[(dict(ptrs={i: None}), NULL) for i in range(4)], (dict(ptrs={0: at(0, 2)}), MIS), (dict(ptrs={1: at(1, 8)}), MIS),
    (dict(ptrs={2: at(2, 1)}), MIS), (dict(ptrs={0: at(0, 1)}, dtype=1), MIS), (dict(stride=99), SHAPE), (dict(ptrs={1: at(0, 3984)}), SHAPE),
    (dict(ptrs={3: at(2, 39)}), SHAPE), (dict(ptrs={2: at(1, 638)}), SHAPE), (dict(k=(1 << 24) + 1), OVER)])
def test_quantize(kw, status):
    expect(status, "dfgpt2_w4_quantize", quantize(**kw))


def dequantize(ptrs=None, dtype=0, fmt=1, group=64, n=10, k=100):
    return pointers(4, ptrs) + [dtype, fmt, group, n, k, None]


@pytest.mark.parametrize("kw,status", WEIGHTS + [
    *[(dict(ptrs={i: None}), NULL) for i in range(4)], (dict(ptrs={3: at(3, 2)}), MIS), (dict(ptrs={0: at(0, 8)}), MIS),
    (dict(ptrs={3: at(0, 636)}), SHAPE), (dict(ptrs={3: at(1)}), SHAPE), (dict(ptrs={3: at(2, 16)}), SHAPE)])
def test_dequantize(kw, status):
    expect(status, "dfgpt2_w4_dequantize", dequantize(**kw))


def linear(ptrs=None, dtype=0, fmt=1, group=64, rows=3, k=100, n=10, stride=None, ws=None, ws_bytes=0):
    return pointers(7, ptrs) + [dtype, fmt, group, rows, k, n, k if stride is None else stride, 0, ws, ws_bytes, None]


@pytest.mark.parametrize("kw,status", WEIGHTS + [
    *[(dict(ptrs={i: None}), NULL) for i in (0, 1, 2, 3, 6)], (dict(ptrs={0: at(0, 2)}), MIS), (dict(ptrs={1: at(1, 4)}), MIS),
    (dict(ptrs={4: at(4, 2)}), MIS), (dict(ptrs={5: at(5, 2)}), MIS), (dict(ptrs={6: at(6, 2)}), MIS), (dict(stride=99), SHAPE),
    (dict(ptrs={6: at(6, 1)}, dtype=1), MIS), (dict(rows=(1 << 20) + 1), OVER), (dict(stride=(1 << 28) + 1), OVER), (dict(rows=0), 0),
    (dict(rows=1 << 20, n=1 << 24), OVER), (dict(rows=1030, k=250, n=64, ws=at(7), ws_bytes=64), WORK),
    (dict(rows=1030, k=250, n=64, ws=at(7, 2), ws_bytes=1 << 30), MIS), (dict(rows=1030, k=250, n=64, ws=at(6, 4), ws_bytes=1 << 30), SHAPE),
    (dict(ptrs={6: at(0, 1196)}), SHAPE), (dict(ptrs={6: at(1, 620)}), SHAPE), (dict(ptrs={6: at(4, 36)}), SHAPE),
    (dict(ptrs={6: at(5, 4)}), SHAPE), (dict(ptrs={6: at(3, 16)}), SHAPE),
    *[(dict(rows=1030, k=250, n=64, ws=at(i, 4), ws_bytes=1 << 30), SHAPE) for i in range(6)]])   # sums over what is read
def test_linear(kw, status):
    expect(status, "dfgpt2_w4_linear", linear(**kw))


def test_row_bytes():
    f = ops.ops_lib().dfgpt2_w4_row_bytes
    assert [f(k) for k in (0, 1, 32, 33, 768, 50257, (1 << 24) + 1)] == [0, 16, 16, 32, 384, 25136, 0]
    assert [w4.row_bytes(k) for k in (1, 32, 33, 768, 50257)] == [16, 16, 32, 384, 25136]


# ---------------------------------------------------------------- the wrappers, on tensors without a device
@pytest.fixture
def here(monkeypatch):
    """Tensors without a device of their own count as being on the current one; nothing may reach the library."""
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


@pytest.mark.parametrize("kw", [
    dict(table=meta(4)), dict(table=meta(5, 8)), dict(lens=meta(4, 1)), dict(lens=meta(4, dtype=torch.int64)),
    dict(parents=meta(6, dtype=torch.int64)), dict(keep_lens=meta(5)), dict(new_table=meta(6, 7)), dict(new_table=meta(5, 8)),
    dict(page_size=-1), dict(page_size=1 << 32), dict(n_pages=-1), dict(n_pages=1 << 32), dict(table=meta(8, 4).t())])
def test_fork_wrapper(here, kw):
    a = dict(table=meta(4, 8), lens=meta(4), parents=meta(6), page_size=16, n_pages=100)
    a.update(kw)
    with pytest.raises(ValueError):
        dfattn.paged_fork(a.pop("table"), a.pop("lens"), a.pop("parents"), **a)


@pytest.mark.parametrize("kw", [dict(ended=meta(3)), dict(ended=meta(4, dtype=torch.bool)), dict(page_size=1 << 32), dict(n_pages=-4)])
def test_free_wrapper(here, kw):
    a = dict(page_size=16, n_pages=100)
    a.update(kw)
    with pytest.raises(ValueError):
        dfattn.paged_free(meta(4, 8), meta(4), **a)


@pytest.mark.parametrize("kw", [dict(new_table=meta(4, 9)), dict(new_table=meta(4, 8, dtype=torch.int64)), dict(page_size=-16)])
def test_compact_wrapper(here, kw):
    a = dict(page_size=16, n_pages=100)
    a.update(kw)
    with pytest.raises(ValueError):
        dfattn.paged_compact(meta(4, 8), meta(4), **a)


@pytest.mark.parametrize("pools,src,dst,n", [
    ([], meta(3), meta(3), None), ([meta(4, 2), meta(5, 2)], meta(3), meta(3), None), ([meta(4, 0)], meta(3), meta(3), None),
    ([meta()], meta(3), meta(3), None), ([meta(4, 6)[:, ::2]], meta(3), meta(3), None), ([meta(4, 2)], meta(3), meta(2), None),
    ([meta(4, 2)], meta(3, dtype=torch.int64), meta(3), None), ([meta(4, 2)], meta(3), meta(3), meta(0)),
    ([meta(4, 2)], meta(3), meta(3), meta(1, dtype=torch.int64))])
def test_copy_wrapper(here, pools, src, dst, n):
    with pytest.raises(ValueError):
        dfattn.paged_copy(pools, src, dst, n)


def a_weight(**kw):
    w = w4.Weight(meta(10, 64, dtype=torch.uint8), meta(2, 10, dtype=torch.bfloat16), None, 100, 64, "i4")
    return w._replace(**kw)


@pytest.mark.parametrize("w,x,kw", [
    (a_weight(format="i8"), None, {}), (a_weight(group=16), None, {}), (a_weight(in_features=0), None, {}), (a_weight(in_features=129), None, {}),
    (a_weight(codes=meta(10, 64, dtype=torch.int8)), None, {}), (a_weight(scales=meta(2, 10, dtype=torch.float32)), None, {}),
    (a_weight(scales=meta(10, 2, dtype=torch.bfloat16)), None, {}), (a_weight(format="u4"), None, {}),
    (a_weight(format="u4", zeros=meta(2, 10, dtype=torch.int8)), None, {}), (a_weight(codes=meta(10, 128, dtype=torch.uint8)[:, ::2]), None, {}),
    (a_weight(), meta(3, 99, dtype=torch.float32), {}), (a_weight(), meta(3, 100, dtype=torch.float16), {}),
    (a_weight(), meta(100, dtype=torch.float32), {}), (a_weight(), meta(3, 200, dtype=torch.float32)[:, ::2], {}),
    (a_weight(), None, dict(bias=meta(9, dtype=torch.float32))), (a_weight(), None, dict(bias=meta(10, dtype=torch.bfloat16))),
    (a_weight(), None, dict(residual=meta(3, 11, dtype=torch.float32))), (a_weight(), None, dict(residual=meta(3, 10, dtype=torch.bfloat16))),
    (a_weight(), None, dict(out=meta(3, 11, dtype=torch.float32))), (a_weight(), None, dict(out=meta(3, 10, dtype=torch.bfloat16)))])
def test_linear_wrapper(here, w, x, kw):
    with pytest.raises(ValueError):
        w4.linear(meta(3, 100, dtype=torch.float32) if x is None else x, w, **kw)


@pytest.mark.parametrize("wants", ["x", "residual"])
def test_linear_has_no_gradient(here, wants):
    x, r = (torch.empty(3, n, device="meta", requires_grad=wants == name) for name, n in (("x", 100), ("residual", 10)))
    with pytest.raises(ValueError, match="gradient"):
        w4.linear(x, a_weight(), residual=r)
    with torch.no_grad(), pytest.raises(AssertionError, match="was called"):
        w4.linear(x, a_weight(), residual=r)


@pytest.mark.parametrize("w,group,fmt", [(meta(3, 4, dtype=torch.float32), 64, "i8"), (meta(3, 4, dtype=torch.float32), 48, "i4"),
                                         (meta(3, 0, dtype=torch.float32), 64, "i4"), (meta(12, dtype=torch.float32), 64, "i4"),
                                         (meta(3, 4, dtype=torch.float64), 64, "i4")])
def test_quantize_wrapper(here, w, group, fmt):
    with pytest.raises(ValueError):
        w4.quantize(w, group, fmt)


def test_dequantize_wrapper(here):
    with pytest.raises(ValueError):
        w4.dequantize(a_weight(), torch.float16)
    with pytest.raises(ValueError):
        w4.dequantize(a_weight(), out=meta(10, 99, dtype=torch.float32))
