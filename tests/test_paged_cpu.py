"""Refusals of the paged-cache and packed-prompt operators that need no GPU: the
Python wrappers on CPU tensors, and the C ABI's checks, which come before any launch."""
import ctypes

import pytest
import torch

import joyomni_ops as jo
from joyomni_ops import _lib

L = _lib.lib
BF16, F32 = _lib.JO_DTYPE_BF16, _lib.JO_DTYPE_F32
S4, S6 = ctypes.c_int64 * 4, ctypes.c_int64 * 6


def test_wrappers_refuse_cpu_tensors():
    i = torch.zeros(1, dtype=torch.int32)
    q = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    c = torch.zeros(1, 16, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="cached_lens must be a CUDA tensor"):
        jo.paged_layout(i, i, i.view(1, 1), i, 16, 1)
    with pytest.raises(RuntimeError, match="key must be a CUDA tensor"):
        jo.paged_kv_write(q, q, c, c, i.long())
    with pytest.raises(RuntimeError, match="query must be a CUDA tensor"):
        jo.paged_attention(q, c, c, i.view(1, 1), torch.zeros(2, dtype=torch.int32), i)
    with pytest.raises(RuntimeError, match="query must be a CUDA tensor"):
        jo.prompt_attention(q, q, q, torch.zeros(2, dtype=torch.int32))


def layout(**kw):
    a = dict(cached=16, fresh=16, table=16, free=16, batch=2, width=4, stride=4, num_free=4, page=16, tokens=8, starts=16,
             lens=16, slots=16, pos=16, needed=16)
    a.update(kw)
    return L.jo_paged_layout(*a.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(batch=-1), "invalid shape"), (dict(tokens=-1), "invalid shape"), (dict(page=0), "page_size"),
    (dict(stride=3), "overlap"), (dict(starts=None), "null"), (dict(slots=None), "null"), (dict(cached=None), "null"),
    (dict(free=None), "null"), (dict(table=None), "null"),
])
def test_layout_refusals(kw, msg):
    assert layout(**kw) == _lib.JO_ERR_INVALID
    assert msg in _lib.last_error()


def write(**kw):
    a = dict(k=16, v=16, kc=16, vc=16, slots=16, tokens=2, heads=2, dim=64, blocks=4, page=16, rs=S4(128, 64, 128, 64),
             cs=S6(2048, 128, 64, 2048, 128, 64), dtype=BF16)
    a.update(kw)
    return L.jo_paged_kv_write(*a.values(), None)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(dtype=F32), _lib.JO_ERR_DTYPE, "bf16 and fp16"), (dict(dim=60), _lib.JO_ERR_INVALID, "multiple of 8"),
    (dict(page=0), _lib.JO_ERR_INVALID, "invalid shape"), (dict(tokens=-1), _lib.JO_ERR_INVALID, "invalid shape"),
    (dict(rs=S4(100, 64, 128, 64)), _lib.JO_ERR_ALIGN, "multiples of 8"), (dict(cs=S6(2048, 128, 64, -8, 128, 64)), _lib.JO_ERR_ALIGN, "non-negative"),
    (dict(v=24), _lib.JO_ERR_ALIGN, "16-byte"), (dict(slots=None), _lib.JO_ERR_INVALID, "null"),
])
def test_write_refusals(kw, code, msg):
    assert write(**kw) == code
    assert msg in _lib.last_error()


def paged(**kw):
    a = dict(q=16, kc=16, vc=16, table=16, starts=16, lens=16, out=16, tokens=4, batch=2, heads=4, kv_heads=2, dim=64,
             blocks=8, page=16, width=4, stride=4, rs=S4(256, 64, 256, 64),
             cs=S6(2048, 128, 64, 2048, 128, 64), causal=1, scale=0.1, most=4, dtype=BF16, ws=16, ws_bytes=1 << 40)
    a.update(kw)
    return L.jo_paged_attention(*a.values(), None)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(dtype=F32), _lib.JO_ERR_DTYPE, "bf16 and fp16"), (dict(dim=96), _lib.JO_ERR_INVALID, "head_dim"),
    (dict(page=24), _lib.JO_ERR_INVALID, "multiple of 16"), (dict(page=0), _lib.JO_ERR_INVALID, "multiple of 16"),
    (dict(heads=5), _lib.JO_ERR_INVALID, "multiple of kv_heads"), (dict(kv_heads=0), _lib.JO_ERR_INVALID, "kv_heads"),
    (dict(heads=512), _lib.JO_ERR_INVALID, "128 times"), (dict(batch=-1), _lib.JO_ERR_INVALID, "invalid shape"),
    (dict(width=1 << 28), _lib.JO_ERR_INVALID, "block table"), (dict(rs=S4(250, 64, 256, 64)), _lib.JO_ERR_ALIGN, "multiples of 8"),
    (dict(cs=S6(2048, -8, 64, 2048, 128, 64)), _lib.JO_ERR_ALIGN, "non-negative"), (dict(q=8), _lib.JO_ERR_ALIGN, "16-byte"),
    (dict(table=None), _lib.JO_ERR_INVALID, "null"), (dict(starts=None), _lib.JO_ERR_INVALID, "null"),
    (dict(rs=None), _lib.JO_ERR_INVALID, "null strides"),
])
def test_paged_attention_refusals(kw, code, msg):
    assert paged(**kw) == code
    assert msg in _lib.last_error()


def prompt(**kw):
    a = dict(q=16, k=16, v=16, starts=16, out=16, tokens=4, batch=2, heads=4, kv_heads=2, dim=64, rs=S4(256, 64, 256, 64),
             ks=S4(128, 64, 128, 64), causal=1, scale=0.1, dtype=BF16, ws=16, ws_bytes=1 << 40)
    a.update(kw)
    return L.jo_prompt_attention(*a.values(), None)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(dtype=F32), _lib.JO_ERR_DTYPE, "bf16 and fp16"), (dict(dim=256), _lib.JO_ERR_INVALID, "head_dim"),
    (dict(heads=3), _lib.JO_ERR_INVALID, "multiple of kv_heads"), (dict(ks=S4(128, 64, 128, 60)), _lib.JO_ERR_ALIGN, "multiples of 8"),
    (dict(out=24), _lib.JO_ERR_ALIGN, "16-byte"), (dict(k=None), _lib.JO_ERR_INVALID, "null"),
    (dict(starts=None), _lib.JO_ERR_INVALID, "null"),
])
def test_prompt_attention_refusals(kw, code, msg):
    assert prompt(**kw) == code
    assert msg in _lib.last_error()


def test_nothing_to_do_is_no_error():
    assert write(tokens=0) == _lib.JO_OK
    assert paged(tokens=0) == _lib.JO_OK
    assert paged(batch=0) == _lib.JO_OK
    assert prompt(tokens=0) == _lib.JO_OK
    assert prompt(heads=0) == _lib.JO_OK
