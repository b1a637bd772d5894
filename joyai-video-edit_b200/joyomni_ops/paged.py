"""Paged K/V cache and attention over requests of different lengths.

A cache is a pair of tensors [num_blocks, page_size, kv_heads, head_dim]; a
request's tokens lie in the blocks of its row of ``block_tables``: token position
``pos`` in slot ``block_tables[b, pos // page_size] * page_size + pos % page_size``.
One step of a server over such a cache is

    lay = paged_layout(cached_lens, new_lens, block_tables, free_blocks, page_size, num_tokens)
    paged_kv_write(k, v, key_cache, value_cache, lay.slots)            # every layer
    out = paged_attention(q, key_cache, value_cache, block_tables, lay.query_starts, lay.kv_lens)

with lengths, tables and slots on the GPU throughout; ``prompt_attention`` is the
form for whole packed prompts without a cache.  No call synchronises, and with
``out`` and ``workspace`` given none allocates, so a step can be captured in a
CUDA graph.  The reference keeps one dense K/V buffer per session instead
(deploy/xvideo/models/dit/dit.py:189-225) and has no counterpart.
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import check as _check, lib as _L

_DT16 = {torch.float16: _lib.JO_DTYPE_F16, torch.bfloat16: _lib.JO_DTYPE_BF16}
_I32, _I64 = torch.int32, torch.int64
_S4 = struct.Struct("4q").pack        # strides for the C ABI's const int64_t*
_S6 = struct.Struct("6q").pack
_stream = torch._C._cuda_getCurrentRawStream
_device = torch._C._cuda_getDevice
_layout, _write, _paged, _prompt = (_L.jo_paged_layout, _L.jo_paged_kv_write, _L.jo_paged_attention,
                                    _L.jo_prompt_attention)

# These calls take a few microseconds on the GPU, so what the host does for one
# counts: arguments are looked at in one expression each, and only a refusal
# walks through them again to say what is wrong (_refuse_*).


def _chk(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _on(idx: int, f, *args, **kw):
    """f(*args, **kw) with device `idx` current."""
    with torch.cuda.device(idx):
        return f(*args, **kw)


def _ints(t: torch.Tensor, name: str, dim: int, dtype: torch.dtype, idx: int) -> None:
    _chk(t.is_cuda, f"{name} must be a CUDA tensor")
    _chk(t.get_device() == idx, f"{name} must be on cuda:{idx}")
    _chk(t.dtype is dtype and t.dim() == dim, f"{name} must be a {dim}-D {dtype} tensor")
    _chk(t.numel() <= 1 or t.stride(-1) == 1, f"{name} last dim must be contiguous")


def _rows(t: torch.Tensor, name: str, dtype, idx: int) -> None:
    _chk(t.is_cuda, f"{name} must be a CUDA tensor")
    _chk(t.get_device() == idx, f"{name} must be on cuda:{idx}")
    _chk(t.dtype is dtype, f"{name} dtype is {t.dtype}, expected {dtype}")
    _chk(t.numel() == 0 or t.stride(-1) == 1, f"{name} last dim must be contiguous")


class PagedLayout(NamedTuple):
    """What a step's calls need about its requests; all on the GPU."""
    query_starts: torch.Tensor      # int32 [batch + 1]: first new token of every request, and their number
    kv_lens: torch.Tensor           # int32 [batch]: cached and new tokens together
    slots: torch.Tensor             # int64 [num_tokens]: cache slot of every new token, -1 for none
    positions: torch.Tensor         # int32 [num_tokens]: position of every new token in its request
    blocks_needed: torch.Tensor     # int32 [1]: free blocks that the step takes

    @classmethod
    def empty(cls, batch: int, num_tokens: int, device) -> "PagedLayout":
        i32 = dict(dtype=torch.int32, device=device)
        return cls(torch.empty(batch + 1, **i32), torch.empty(batch, **i32),
                   torch.empty(num_tokens, dtype=torch.int64, device=device), torch.empty(num_tokens, **i32),
                   torch.empty(1, **i32))


def paged_layout(cached_lens, new_lens, block_tables, free_blocks, page_size: int, num_tokens: int, *,
                 out: Optional[PagedLayout] = None) -> PagedLayout:
    """Block tables, slots and offsets of one step from its request lengths.

    cached_lens, new_lens: int32 [B], the tokens that request b has in the cache
    and its new ones (negative counts as 0).  block_tables: int32 [B, max_blocks],
    updated in place: the blocks a request newly needs are taken from the front of
    ``free_blocks`` (int32 [F]) in request order.  num_tokens: places of the
    token-wise results, at least the sum of new_lens; the places after the last
    request get slot -1 and position 0.  Where the free list or a table row is too
    short the slot is -1, and ``blocks_needed`` tells how many blocks the step
    wanted.  out: a PagedLayout to write into (its tensors contiguous)."""
    idx = cached_lens.get_device()
    B = cached_lens.numel()
    if not (idx >= 0 and cached_lens.dtype is _I32 and new_lens.dtype is _I32 and free_blocks.dtype is _I32
            and block_tables.dtype is _I32 and new_lens.get_device() == idx and free_blocks.get_device() == idx
            and block_tables.get_device() == idx and cached_lens.dim() == new_lens.dim() == free_blocks.dim() == 1
            and cached_lens.is_contiguous() and new_lens.is_contiguous() and free_blocks.is_contiguous()
            and block_tables.dim() == 2 and block_tables.is_contiguous() and block_tables.size(0) == B
            and new_lens.numel() == B and num_tokens >= 0):
        _refuse_layout(cached_lens, new_lens, block_tables, free_blocks, num_tokens)
    width = block_tables.size(1)
    if out is None:
        out = PagedLayout.empty(B, num_tokens, cached_lens.device)
    starts, lens, slots, pos, needed = out
    if not (starts.numel() == B + 1 and lens.numel() == B and slots.numel() == pos.numel() == num_tokens
            and needed.numel() == 1 and slots.dtype is _I64
            and starts.dtype is lens.dtype is pos.dtype is needed.dtype is _I32
            and starts.get_device() == lens.get_device() == slots.get_device() == pos.get_device() == idx
            and needed.get_device() == idx and starts.is_contiguous() and lens.is_contiguous()
            and slots.is_contiguous() and pos.is_contiguous()):
        raise RuntimeError(f"out must hold contiguous tensors on cuda:{idx} of PagedLayout.empty({B}, {num_tokens}, ...)'s "
                           "sizes and types")
    if _device() != idx:
        return _on(idx, paged_layout, cached_lens, new_lens, block_tables, free_blocks, page_size, num_tokens, out=out)
    status = _layout(cached_lens.data_ptr(), new_lens.data_ptr(), block_tables.data_ptr(), free_blocks.data_ptr(), B, width,
                     block_tables.stride(0) if B > 1 else width, free_blocks.numel(), page_size, num_tokens,
                     starts.data_ptr(), lens.data_ptr(), slots.data_ptr(), pos.data_ptr(), needed.data_ptr(), _stream(idx))
    if status:
        _check(status)
    return out


def _refuse_layout(cached_lens, new_lens, block_tables, free_blocks, num_tokens) -> None:
    _chk(cached_lens.is_cuda, "cached_lens must be a CUDA tensor")
    idx = cached_lens.get_device()
    for t, n in ((cached_lens, "cached_lens"), (new_lens, "new_lens"), (free_blocks, "free_blocks")):
        _ints(t, n, 1, _I32, idx)
    _ints(block_tables, "block_tables", 2, _I32, idx)       # rows may be apart: a slice of a wider table
    B = block_tables.size(0)
    _chk(cached_lens.numel() == B and new_lens.numel() == B,
         "cached_lens, new_lens and block_tables must have a row per request")
    _chk(num_tokens >= 0, "num_tokens must not be negative")


def paged_kv_write(key, value, key_cache, value_cache, slots) -> None:
    """Stores rows of key and value [T, kv_heads, head_dim] (bf16 or fp16; views
    with any token and head strides that are multiples of 8) into their slots of
    the caches [num_blocks, page_size, kv_heads, head_dim], in place.  Rows whose
    slot (int64 [T]) is negative or past the cache are left out.  Two rows must not
    have the same slot."""
    idx, dt = key.get_device(), key.dtype
    code = _DT16.get(dt)
    shape, cs = key.shape, key_cache.shape
    a, b, c, d = key.stride(), value.stride(), key_cache.stride(), value_cache.stride()
    if not (idx >= 0 and code is not None and len(shape) == 3 and value.shape == shape and len(cs) == 4
            and value_cache.shape == cs and cs[2:] == shape[1:] and value.dtype is dt
            and key_cache.dtype is dt and value_cache.dtype is dt and value.get_device() == idx
            and key_cache.get_device() == idx and value_cache.get_device() == idx and a[2] == b[2] == c[3] == d[3] == 1
            and slots.dtype is _I64 and slots.get_device() == idx and slots.is_contiguous() and slots.shape == shape[:1]):
        _refuse_write(key, value, key_cache, value_cache, slots)
    T, H, D = shape
    if _device() != idx:
        return _on(idx, paged_kv_write, key, value, key_cache, value_cache, slots)
    status = _write(key.data_ptr(), value.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), slots.data_ptr(), T, H, D,
                    cs[0], cs[1], _S4(a[0], a[1], b[0], b[1]), _S6(c[0], c[1], c[2], d[0], d[1], d[2]), code, _stream(idx))
    if status:
        _check(status)


def _refuse_write(key, value, key_cache, value_cache, slots) -> None:
    _chk(key.is_cuda, "key must be a CUDA tensor")
    idx, dt = key.get_device(), key.dtype
    _chk(dt in _DT16, "key must be bf16 or fp16")
    _chk(key.dim() == 3 and value.shape == key.shape, "key and value must be [tokens, kv_heads, head_dim]")
    _chk(key_cache.dim() == 4 and value_cache.shape == key_cache.shape and key_cache.shape[2:] == key.shape[1:],
         "caches must be [num_blocks, page_size, kv_heads, head_dim] with key's heads")
    for t, n in ((key, "key"), (value, "value"), (key_cache, "key_cache"), (value_cache, "value_cache")):
        _rows(t, n, dt, idx)
    _ints(slots, "slots", 1, _I64, idx)
    _chk(slots.numel() == key.size(0), "slots must have one entry per token")


_ws_bytes = {}


def varlen_attention_workspace(max_keys: int, head_dim: int) -> int:
    """Bytes of workspace that paged_attention and prompt_attention need on the
    current device for the partial results of work that is split along the keys.
    max_keys: the most keys that a request can have, block_tables' width times the
    page size, or the number of packed rows."""
    n = ctypes.c_int64()
    _check(_L.jo_varlen_attention_workspace(max_keys, head_dim, ctypes.byref(n)))
    return n.value


def _workspace(workspace, idx: int, max_keys: int, D: int):
    """(address, bytes, the tensor) of a call's workspace."""
    need = _ws_bytes.get((idx, max_keys, D))
    if need is None:
        if len(_ws_bytes) > 4096:
            _ws_bytes.clear()
        with torch.cuda.device(idx):
            need = _ws_bytes[(idx, max_keys, D)] = varlen_attention_workspace(max_keys, D)
    if workspace is None:
        if need == 0:
            return 0, 0, None
        workspace = torch.empty(need, dtype=torch.uint8, device=torch.device("cuda", idx))
        return workspace.data_ptr(), need, workspace
    have = workspace.numel() * workspace.element_size()
    _chk(workspace.get_device() == idx and workspace.is_contiguous() and have >= need,
         f"workspace must be a contiguous tensor of at least {need} bytes on cuda:{idx}")
    return workspace.data_ptr(), have, workspace


def _out(q, out):
    if out is None:
        return torch.empty_like(q) if q.is_contiguous() else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _chk(out.shape == q.shape, "out must have query's shape")
    _rows(out, "out", q.dtype, q.get_device())
    return out


def _refuse_query(query) -> None:
    _chk(query.is_cuda, "query must be a CUDA tensor")
    _chk(query.dim() == 3, "query must be [tokens, heads, head_dim]")
    _chk(query.dtype in _DT16, "query must be bf16 or fp16")
    _rows(query, "query", query.dtype, query.get_device())


def paged_attention(query, key_cache, value_cache, block_tables, query_starts, kv_lens, *, causal: bool = True,
                    scale: Optional[float] = None, max_query_len: Optional[int] = None, out=None, workspace=None):
    """softmax(scale * q k^T) v of new tokens over a paged cache.

    query [T, H, head_dim] (bf16 or fp16, head_dim 64 or 128) holds the requests'
    new tokens side by side: request b has rows query_starts[b] ..
    query_starts[b + 1] (int32 [B + 1]).  Its keys are tokens 0 .. kv_lens[b]
    (int32 [B]) of its blocks in key_cache and value_cache [num_blocks, page_size,
    kv_heads, head_dim], the new tokens' own among them (paged_kv_write first);
    page_size a multiple of 16.  Row i of n sees keys 0 .. kv_lens[b] - n + i
    (causal) or all; a row that sees none (or only scores of -infinity) is zero.  An
    infinity in a value that a row sees is infinity in its result, whatever its weight;
    values that it does not see have no influence.  H must be a multiple of
    kv_heads; query head h reads key head h // (H / kv_heads).  Rows of no request
    are not written.  max_query_len: the largest number of new tokens in a
    request, if the caller knows it (1 for a decoding step): it chooses the
    kernels, any value is right, and results differ by rounding: the kernel for
    requests of up to 32 rows (new tokens times H / kv_heads) keeps 16 bits and more of
    the weights before the product with V, the other one rounds them to query's type
    (1.1 to 1.4 times the error of rounding the result alone).  scale defaults to
    1 / sqrt(head_dim).  workspace: varlen_attention_workspace bytes, used by one
    call at a time; by default allocated per call."""
    idx, dt = query.get_device(), query.dtype
    code = _DT16.get(dt)
    shape, cs, ts = query.shape, key_cache.shape, block_tables.shape
    a, c, d = query.stride(), key_cache.stride(), value_cache.stride()
    if not (idx >= 0 and code is not None and len(shape) == 3 and len(cs) == 4 and len(ts) == 2
            and value_cache.shape == cs and a[2] == c[3] == d[3] == 1 and cs[3] == shape[2]
            and key_cache.dtype is dt and value_cache.dtype is dt and key_cache.get_device() == idx
            and value_cache.get_device() == idx and block_tables.dtype is _I32 and query_starts.dtype is _I32
            and kv_lens.dtype is _I32 and block_tables.get_device() == idx and query_starts.get_device() == idx
            and kv_lens.get_device() == idx and block_tables.is_contiguous() and query_starts.is_contiguous()
            and kv_lens.is_contiguous() and kv_lens.shape == ts[:1] and query_starts.shape == (ts[0] + 1,)):
        _refuse_paged(query, key_cache, value_cache, block_tables, query_starts, kv_lens)
    T, H, D = shape
    B, width = ts
    o = _out(query, out)
    ws, ws_bytes, _keep = _workspace(workspace, idx, width * cs[1], D)
    e = o.stride()
    if _device() != idx:
        return _on(idx, paged_attention, query, key_cache, value_cache, block_tables, query_starts, kv_lens, causal=causal,
                   scale=scale, max_query_len=max_query_len, out=o, workspace=_keep)
    status = _paged(query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), block_tables.data_ptr(),
                    query_starts.data_ptr(), kv_lens.data_ptr(), o.data_ptr(), T, B, H, cs[2], D, cs[0], cs[1], width,
                    block_tables.stride(0) if B > 1 else width, _S4(a[0], a[1], e[0], e[1]),
                    _S6(c[0], c[1], c[2], d[0], d[1], d[2]), 1 if causal else 0,
                    1.0 / math.sqrt(D) if scale is None else scale, T if max_query_len is None else max_query_len, code, ws,
                    ws_bytes, _stream(idx))
    if status:
        _check(status)
    return o


def _refuse_paged(query, key_cache, value_cache, block_tables, query_starts, kv_lens) -> None:
    _refuse_query(query)
    idx, dt = query.get_device(), query.dtype
    _chk(key_cache.dim() == 4 and value_cache.shape == key_cache.shape and key_cache.size(3) == query.size(2),
         "caches must be [num_blocks, page_size, kv_heads, head_dim] with query's head_dim")
    _rows(key_cache, "key_cache", dt, idx)
    _rows(value_cache, "value_cache", dt, idx)
    _ints(block_tables, "block_tables", 2, _I32, idx)       # rows may be apart: a slice of a wider table
    _ints(query_starts, "query_starts", 1, _I32, idx)
    _ints(kv_lens, "kv_lens", 1, _I32, idx)
    B = block_tables.size(0)
    _chk(query_starts.numel() == B + 1 and kv_lens.numel() == B,
         "query_starts must have batch + 1 entries and kv_lens batch")


def prompt_attention(query, key, value, seq_starts, *, causal: bool = True, scale: Optional[float] = None, out=None,
                     workspace=None):
    """softmax(scale * q k^T) v of whole packed prompts.

    query [T, H, head_dim], key and value [T, kv_heads, head_dim] (bf16 or fp16,
    head_dim 64 or 128; views with token and head strides that are multiples of 8
    are read in place); request b is rows seq_starts[b] .. seq_starts[b + 1]
    (int32 [B + 1]) of all three.  Row i sees keys 0 .. i of its own request
    (causal) or all of them.  H must be a multiple of kv_heads.  Rows of no
    request are not written.  What rows see, infinities, scale, out and workspace as in paged_attention."""
    idx, dt = query.get_device(), query.dtype
    code = _DT16.get(dt)
    shape, ks = query.shape, key.shape
    a, b, c = query.stride(), key.stride(), value.stride()
    if not (idx >= 0 and code is not None and len(shape) == 3 and len(ks) == 3 and value.shape == ks
            and ks[0] == shape[0] and ks[2] == shape[2] and a[2] == b[2] == c[2] == 1
            and key.dtype is dt and value.dtype is dt and key.get_device() == idx and value.get_device() == idx
            and seq_starts.dtype is _I32 and seq_starts.get_device() == idx and seq_starts.dim() == 1
            and seq_starts.is_contiguous() and seq_starts.numel() >= 1):
        _refuse_prompt(query, key, value, seq_starts)
    T, H, D = shape
    o = _out(query, out)
    ws, ws_bytes, _keep = _workspace(workspace, idx, T, D)
    e = o.stride()
    if _device() != idx:
        return _on(idx, prompt_attention, query, key, value, seq_starts, causal=causal, scale=scale, out=o, workspace=_keep)
    status = _prompt(query.data_ptr(), key.data_ptr(), value.data_ptr(), seq_starts.data_ptr(), o.data_ptr(), T,
                     seq_starts.numel() - 1, H, ks[1], D, _S4(a[0], a[1], e[0], e[1]), _S4(b[0], b[1], c[0], c[1]),
                     1 if causal else 0, 1.0 / math.sqrt(D) if scale is None else scale, code, ws, ws_bytes, _stream(idx))
    if status:
        _check(status)
    return o


def _refuse_prompt(query, key, value, seq_starts) -> None:
    _refuse_query(query)
    idx, dt = query.get_device(), query.dtype
    _chk(key.dim() == 3 and key.shape == value.shape and key.size(0) == query.size(0) and key.size(2) == query.size(2),
         "key and value must be [tokens, kv_heads, head_dim] with query's tokens and head_dim")
    _rows(key, "key", dt, idx)
    _rows(value, "value", dt, idx)
    _ints(seq_starts, "seq_starts", 1, _I32, idx)
    _chk(seq_starts.numel() >= 1, "seq_starts must have batch + 1 entries")
