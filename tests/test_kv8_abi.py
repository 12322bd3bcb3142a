"""The serving entry points' refusals, on the CPU: everything here is caught on the host before any HIP call."""
import ctypes

import pytest

import dfattn
from dfattn import ops

P, ODD, ODD2 = (ctypes.c_void_p(x) for x in (0x10000, 0x10002, 0x10001))
NULL, MIS, SHAPE, HEAD, OVER, WORK, FLAGS = -1, -2, -3, -4, -5, -6, -8


def expect(status, fn, args):
    lib = ops.ops_lib()
    lib.dfattn_clear_error()
    assert getattr(lib, fn)(*args) == status
    assert lib.dfattn_last_error() == status
    if status:
        assert fn.encode() in lib.dfattn_last_error_message()
    lib.dfattn_clear_error()


def plan(ptrs=None, n_free=9, r=4, width=8, cap=64, page=16, pages=100):
    p = [ctypes.c_void_p(0x10000 + 0x1000 * i) for i in range(9)]
    for i, x in (ptrs or {}).items():
        p[i] = x
    return p + [n_free, r, width, cap, page, pages, None]


@pytest.mark.parametrize("kw,status", [
    *[(dict(ptrs={i: None}), NULL) for i in range(9)], *[(dict(ptrs={i: ODD}), MIS) for i in range(9)],
    (dict(r=0), SHAPE), (dict(width=0), SHAPE), (dict(page=0), SHAPE), (dict(pages=0), SHAPE), (dict(r=8193), OVER),
    (dict(pages=1 << 28), OVER), (dict(width=1 << 28), OVER), (dict(cap=(1 << 31) + 1), OVER),
    (dict(ptrs={3: ctypes.c_void_p(0x10000 + 0x8000 + 8)}), SHAPE),  # free_start inside counts
    (dict(ptrs={5: ctypes.c_void_p(0x10000)}), SHAPE),               # seq_lens in place of cached_lens
    (dict(ptrs={7: ctypes.c_void_p(0x10000 + 0x8000 - 4 * 63)}), SHAPE),  # the slot map's end in counts
    (dict(ptrs={4: ctypes.c_void_p(0x10000 + 0x2000 + 32)}), SHAPE),      # the table in the free pages' last entry
])
def test_plan(kw, status):
    expect(status, "dfattn_paged_plan", plan(**kw))


def append(ptrs=None, act=0, kv=2, n=4, heads=2, d=64, page=16, pages=10, stride=None):
    p = [P] * 7
    for i, x in (ptrs or {}).items():
        p[i] = x
    return p + [act, kv, n, heads, d, page, pages, heads * d if stride is None else stride, None]


CACHE = [(dict(act=2), FLAGS), (dict(kv=0), FLAGS), (dict(kv=4), FLAGS), (dict(heads=0), SHAPE), (dict(pages=0), SHAPE),
         (dict(page=0), SHAPE), (dict(page=8), SHAPE), (dict(page=24), SHAPE), (dict(page=272), SHAPE), (dict(d=0), HEAD),
         (dict(d=129), HEAD), (dict(heads=65536), OVER), (dict(pages=1 << 28), OVER)]


@pytest.mark.parametrize("kw,status", CACHE + [
    *[(dict(ptrs={i: None}), NULL) for i in range(7)], (dict(ptrs={0: ODD}), MIS), (dict(ptrs={1: ODD2}, act=1), MIS),
    (dict(ptrs={2: ODD}), MIS), (dict(ptrs={3: ctypes.c_void_p(0x10008)}), MIS), (dict(ptrs={6: ODD}), MIS),
    (dict(stride=127), SHAPE), (dict(stride=(1 << 21) + 1), OVER), (dict(n=(1 << 31) + 1), OVER), (dict(n=0), 0),
])
def test_append(kw, status):
    expect(status, "dfattn_kv8_append", append(**kw))


def read(ptrs=None, act=0, kv=2, n=4, heads=2, d=64, page=16, pages=10):
    p = [P] * 7
    for i, x in (ptrs or {}).items():
        p[i] = x
    return p + [act, kv, n, heads, d, page, pages, None]


@pytest.mark.parametrize("kw,status", CACHE + [
    *[(dict(ptrs={i: None}), NULL) for i in range(7)], (dict(ptrs={5: ODD}), MIS), (dict(ptrs={6: ODD2}, act=1), MIS),
    (dict(ptrs={4: ODD}), MIS), (dict(ptrs={1: ctypes.c_void_p(0x10008)}), MIS), (dict(n=0), 0),
])
def test_read(kw, status):
    expect(status, "dfattn_kv8_read", read(**kw))


def attention(ptrs=None, act=0, kv=2, r=3, n=3, max_q=1, max_len=5000, heads=4, hk=2, d=64, page=16, pages=1000, width=400,
              stride=None, ws=None, ws_bytes=0):
    p = [P] * 10
    for i, x in (ptrs or {}).items():
        p[i] = x
    return p + [act, kv, r, n, max_q, max_len, heads, hk, d, page, pages, width,
                heads * d if stride is None else stride, 0.125, 1, ws, ws_bytes, None]


@pytest.mark.parametrize("kw,status", [({("hk" if k == "heads" else k): x for k, x in kw.items()}, s) for kw, s in CACHE] + [
    *[(dict(ptrs={i: None}), NULL) for i in range(9)], (dict(ptrs={0: ODD}), MIS), (dict(ptrs={8: ODD}), MIS),
    (dict(ptrs={9: ODD}), MIS), (dict(ptrs={1: ctypes.c_void_p(0x10008)}), MIS), (dict(ptrs={6: ODD}), MIS),
    (dict(heads=0), SHAPE), (dict(heads=3), SHAPE), (dict(width=0), SHAPE), (dict(stride=255), SHAPE),
    (dict(heads=65538, hk=2), OVER), (dict(r=65536), OVER), (dict(n=(1 << 30) + 1), OVER), (dict(width=1 << 28), OVER),
    (dict(r=60000, n=1 << 30, max_q=1 << 30), OVER), (dict(ws=P, ws_bytes=4), WORK), (dict(ws=ODD, ws_bytes=1 << 30), WORK),
    (dict(n=1 << 26, max_q=1 << 26, heads=34), OVER),  # 17 * 2^26 columns
    (dict(r=0), 0), (dict(n=0), 0), (dict(max_q=0), 0),
])
def test_attention(kw, status):
    expect(status, "dfattn_kv8_attention", attention(**kw))


def test_sizes():
    lib = dfattn.lib()
    assert lib.dfattn_kv8_pool_bytes(10, 2, 16, 64) == 10 * 2 * 16 * 64
    assert lib.dfattn_kv8_pool_bytes(10, 2, 32, 33) == 10 * 2 * 32 * 48
    for bad in ((0, 2, 16, 64), (10, 0, 16, 64), (10, 2, 17, 64), (10, 2, 0, 64), (10, 2, 16, 129), (10, 2, 16, 0)):
        assert lib.dfattn_kv8_pool_bytes(*bad) == 0
    size = lib.dfattn_kv8_attention_workspace_bytes
    assert size(1, 1, 1, 64, 12, 12, 64) == 0            # one short row: nothing to split
    assert size(1, 1, 1, 100000, 12, 12, 64) > 0
    assert size(0, 1, 1, 100000, 12, 12, 64) == 0 and size(1, 1, 1, 100000, 12, 5, 64) == 0
    assert size(1, 1 << 26, 1 << 26, 100000, 34, 2, 64) == 0
    with pytest.raises(ValueError):
        dfattn.kv8_cache(2, 2, 64, 17, device="cpu")
    with pytest.raises(ValueError):
        dfattn.kv8_cache(2, 2, 64, 16, "float32", device="cpu")


def logprobs(ptrs=None, dtype=0, rows=4, cols=100, stride=None, k=5):
    p = [P] * 7
    for i, x in (ptrs or {}).items():
        p[i] = x
    return p + [dtype, rows, cols, cols if stride is None else stride, k, None]


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=2), FLAGS), (dict(cols=0), SHAPE), (dict(stride=99), SHAPE), (dict(k=65), SHAPE), (dict(cols=3), SHAPE),
    (dict(rows=(1 << 21) + 1), OVER), (dict(cols=(1 << 27) + 1, stride=(1 << 30) + 1), OVER),
    *[(dict(ptrs={i: None}), NULL) for i in (0, 1, 2, 5, 6)], *[(dict(ptrs={i: ODD}), MIS) for i in range(7)],
    (dict(ptrs={0: ODD2}, dtype=1), MIS), (dict(rows=0), 0),
])
def test_token_logprobs(kw, status):
    expect(status, "dfgpt2_token_logprobs", logprobs(**kw))


def backward(ptrs=None, dtype=0, rows=4, cols=100, stride=None):
    p = [ctypes.c_void_p(0x10000 + 0x1000 * i) for i in range(7)]
    for i, x in (ptrs or {}).items():
        p[i] = x
    return p + [dtype, rows, cols, cols if stride is None else stride, None]


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=2), FLAGS), (dict(cols=0), SHAPE), (dict(stride=99), SHAPE), (dict(rows=(1 << 21) + 1), OVER),
    *[(dict(ptrs={i: None}), NULL) for i in (0, 1, 2, 3, 6)], *[(dict(ptrs={i: ODD}), MIS) for i in range(7)],
    (dict(ptrs={6: P}, stride=104), SHAPE), (dict(rows=0), 0), (dict(ptrs={6: ctypes.c_void_p(0x10004)}), SHAPE),
    (dict(ptrs={6: ctypes.c_void_p(0x10000 + 4 * (4 * 100 - 1))}), SHAPE),
])
def test_token_logprobs_backward(kw, status):
    expect(status, "dfgpt2_token_logprobs_backward", backward(**kw))
