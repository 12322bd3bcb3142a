"""The serving wrappers' refusals that need no GPU: sizes and strides that do not fit the entry points' 32 bits."""
import pytest
import torch

import dfattn
from dfattn import kv8

BIG = 1 << 32


@pytest.fixture
def here(monkeypatch):
    """Tensors without a device of their own count as being on the current one; nothing may reach the library."""
    names = (torch, torch.int32, torch.float32, torch.bfloat16, torch.int8, torch.float8_e4m3fn, -1)
    monkeypatch.setattr(kv8, "_names", lambda: names)
    monkeypatch.setattr(kv8, "_stream_ptr", lambda s: None)

    class Lib:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was called")

    monkeypatch.setattr(kv8, "lib", Lib)


def meta(*shape, dtype=torch.int32):
    return torch.empty(shape, dtype=dtype, device="meta")


def cache():
    codes = torch.int8
    return dfattn.KV8Cache(meta(4, 2, 16, 64, dtype=codes), meta(4, 2, 64, 16, dtype=codes),
                           meta(4, 2, dtype=torch.float32), meta(4, 2, dtype=torch.float32))


@pytest.mark.parametrize("kw", [dict(max_query_len=BIG), dict(max_query_len=-1), dict(max_seq_len=BIG + 64),
                                dict(max_seq_len=-1), dict(n_heads=0), dict(n_heads=-2)])
def test_attention(here, kw):
    a = dict(n_heads=2, max_query_len=1, max_seq_len=64, workspace=None)
    a.update(kw)
    with pytest.raises(ValueError):
        dfattn.kv8_attention(cache(), meta(3, 128, dtype=torch.float32), meta(3, 2), meta(4), meta(3), **a)


@pytest.mark.parametrize("kw", [dict(page_size=BIG + 16), dict(page_size=-16), dict(n_pages=BIG + 4), dict(n_pages=-1),
                                dict(token_capacity=BIG + 8), dict(token_capacity=-1)])
def test_plan(here, kw):
    a = dict(page_size=16, n_pages=4, token_capacity=8)
    a.update(kw)
    with pytest.raises(ValueError, match=next(iter(kw))):
        dfattn.paged_plan(meta(3), meta(3), meta(3, 2), meta(4), meta(1), **a)


@pytest.mark.parametrize("stride", [BIG, BIG + 4096, 3 * BIG + 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(here, stride, dtype):
    """Rows 2^32 elements apart and more: modulo 2^32 some of these are strides of a valid call, of other rows."""
    far = meta(2, 128, dtype=dtype).as_strided((2, 128), (stride, 1))
    with pytest.raises(ValueError, match="row stride"):
        dfattn.kv8_append(cache(), far, far, meta(2))
    with pytest.raises(ValueError, match="row stride"):
        dfattn.kv8_attention(cache(), far, meta(2, 2), meta(3), meta(2), 2, 1, 64, workspace=None)
