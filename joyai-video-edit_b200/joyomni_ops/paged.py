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
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import check as _check, lib as _L

_DT16 = {torch.float16: _lib.JO_DTYPE_F16, torch.bfloat16: _lib.JO_DTYPE_BF16}
_S2 = ctypes.c_int64 * 2
_S3 = ctypes.c_int64 * 3


def _chk(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


class _On:
    """Makes the tensor's device current where it is not, and gives its current stream."""

    __slots__ = ("dev", "prev")

    def __init__(self, t: torch.Tensor):
        self.dev = t.device.index
        self.prev = None

    def __enter__(self) -> int:
        cur = torch.cuda.current_device()
        if cur != self.dev:
            self.prev = cur
            torch.cuda.set_device(self.dev)
        return torch.cuda.current_stream(self.dev).cuda_stream

    def __exit__(self, *exc):
        if self.prev is not None:
            torch.cuda.set_device(self.prev)
        return False


def _ints(t: torch.Tensor, name: str, dim: int, dtype: torch.dtype, dev) -> None:
    _chk(t.is_cuda and t.device == dev, f"{name} must be a CUDA tensor on {dev}")
    _chk(t.dtype == dtype and t.dim() == dim, f"{name} must be a {dim}-D {dtype} tensor")
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
    dev = cached_lens.device
    for t, n in ((cached_lens, "cached_lens"), (new_lens, "new_lens"), (free_blocks, "free_blocks")):
        _ints(t, n, 1, torch.int32, dev)
    _ints(block_tables, "block_tables", 2, torch.int32, dev)
    B, width = block_tables.shape
    _chk(cached_lens.size(0) == B and new_lens.size(0) == B, "cached_lens, new_lens and block_tables must have a row "
                                                             "per request")
    _chk(num_tokens >= 0, "num_tokens must not be negative")
    stride = block_tables.stride(0) if B > 1 else width
    if out is None:
        out = PagedLayout.empty(B, num_tokens, dev)
    else:
        want = ((B + 1, torch.int32), (B, torch.int32), (num_tokens, torch.int64), (num_tokens, torch.int32),
                (1, torch.int32))
        for t, (n, dt), name in zip(out, want, PagedLayout._fields):
            _chk(t.device == dev and t.dtype == dt and t.shape == (n,) and t.is_contiguous(),
                 f"out.{name} must be a contiguous {dt} tensor of {n} on {dev}")
    with _On(cached_lens) as st:
        _check(_L.jo_paged_layout(cached_lens.data_ptr(), new_lens.data_ptr(), block_tables.data_ptr(),
                                  free_blocks.data_ptr(), B, width, stride, free_blocks.size(0), page_size, num_tokens,
                                  out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), out[3].data_ptr(),
                                  out[4].data_ptr(), st))
    return out


def _rows(t: torch.Tensor, name: str, dev, dtype) -> None:
    _chk(t.is_cuda and t.device == dev, f"{name} must be a CUDA tensor on {dev}")
    _chk(t.dtype == dtype, f"{name} dtype is {t.dtype}, expected {dtype}")
    _chk(t.stride(-1) == 1 or t.numel() == 0, f"{name} last dim must be contiguous")


def paged_kv_write(key, value, key_cache, value_cache, slots) -> None:
    """Stores rows of key and value [T, kv_heads, head_dim] (bf16 or fp16; views
    with any token and head strides that are multiples of 8) into their slots of
    the caches [num_blocks, page_size, kv_heads, head_dim], in place.  Rows whose
    slot (int64 [T]) is negative or past the cache are left out.  Two rows must not
    have the same slot."""
    dev, dt = key.device, key.dtype
    _chk(dt in _DT16, "key must be bf16 or fp16")
    _chk(key.dim() == 3 and value.shape == key.shape, "key and value must be [tokens, kv_heads, head_dim]")
    _chk(key_cache.dim() == 4 and value_cache.shape == key_cache.shape and key_cache.shape[2:] == key.shape[1:],
         "caches must be [num_blocks, page_size, kv_heads, head_dim] with key's heads")
    for t, n in ((key, "key"), (value, "value"), (key_cache, "key_cache"), (value_cache, "value_cache")):
        _rows(t, n, dev, dt)
    _ints(slots, "slots", 1, torch.int64, dev)
    T, H, D = key.shape
    _chk(slots.size(0) == T, "slots must have one entry per token")
    nb, page = key_cache.shape[:2]
    a, b, c, d = key.stride(), value.stride(), key_cache.stride(), value_cache.stride()
    with _On(key) as st:
        _check(_L.jo_paged_kv_write(key.data_ptr(), value.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(),
                                    slots.data_ptr(), T, H, D, nb, page, _S2(a[0], a[1]), _S2(b[0], b[1]),
                                    _S3(c[0], c[1], c[2]), _S3(d[0], d[1], d[2]), _DT16[dt], st))


def varlen_attention_workspace(num_tokens: int, heads: int, head_dim: int) -> int:
    """Bytes of workspace that paged_attention and prompt_attention use for
    queries of these sizes (partial results of work that is split along the keys)."""
    n = ctypes.c_int64()
    _check(_L.jo_varlen_attention_workspace(num_tokens, heads, head_dim, ctypes.byref(n)))
    return n.value


def _workspace(workspace, T: int, H: int, D: int, dev):
    need = varlen_attention_workspace(T, H, D)
    if workspace is None:
        return torch.empty(need, dtype=torch.uint8, device=dev)
    _chk(workspace.is_cuda and workspace.device == dev and workspace.is_contiguous()
         and workspace.numel() * workspace.element_size() >= need,
         f"workspace must be a contiguous tensor of at least {need} bytes on {dev}")
    return workspace


def _queries(q, out, dev):
    _chk(q.is_cuda, "query must be a CUDA tensor")
    _chk(q.dim() == 3, "query must be [tokens, heads, head_dim]")
    _chk(q.dtype in _DT16, "query must be bf16 or fp16")
    _rows(q, "query", dev, q.dtype)
    if out is None:
        return torch.empty(q.shape, dtype=q.dtype, device=dev)
    _chk(out.shape == q.shape, "out must have query's shape")
    _rows(out, "out", dev, q.dtype)
    return out


def paged_attention(query, key_cache, value_cache, block_tables, query_starts, kv_lens, *, causal: bool = True,
                    scale: Optional[float] = None, max_query_len: Optional[int] = None, out=None, workspace=None):
    """softmax(scale * q k^T) v of new tokens over a paged cache.

    query [T, H, head_dim] (bf16 or fp16, head_dim 64 or 128) holds the requests'
    new tokens side by side: request b has rows query_starts[b] ..
    query_starts[b + 1] (int32 [B + 1]).  Its keys are tokens 0 .. kv_lens[b]
    (int32 [B]) of its blocks in key_cache and value_cache [num_blocks, page_size,
    kv_heads, head_dim], the new tokens' own among them (paged_kv_write first);
    page_size a multiple of 16.  Row i of n sees keys 0 .. kv_lens[b] - n + i
    (causal) or all; a row that sees none is zero.  H must be a multiple of
    kv_heads; query head h reads key head h // (H / kv_heads).  Rows of no request
    are not written.  max_query_len: the largest number of new tokens in a
    request, if the caller knows it (1 for a decoding step): it chooses the
    kernels and never changes what is computed.  scale defaults to
    1 / sqrt(head_dim).  workspace: varlen_attention_workspace bytes, used by one
    call at a time; by default allocated per call."""
    dev, dt = query.device, query.dtype
    o = _queries(query, out, dev)
    T, H, D = query.shape
    _chk(key_cache.dim() == 4 and value_cache.shape == key_cache.shape and key_cache.size(3) == D,
         "caches must be [num_blocks, page_size, kv_heads, head_dim] with query's head_dim")
    _rows(key_cache, "key_cache", dev, dt)
    _rows(value_cache, "value_cache", dev, dt)
    _ints(block_tables, "block_tables", 2, torch.int32, dev)
    _ints(query_starts, "query_starts", 1, torch.int32, dev)
    _ints(kv_lens, "kv_lens", 1, torch.int32, dev)
    B, width = block_tables.shape
    _chk(query_starts.size(0) == B + 1 and kv_lens.size(0) == B, "query_starts must have batch + 1 entries and kv_lens "
                                                                 "batch")
    nb, page, Hk, _ = key_cache.shape
    ws = _workspace(workspace, T, H, D, dev)
    a, c, d, e = query.stride(), key_cache.stride(), value_cache.stride(), o.stride()
    with _On(query) as st:
        _check(_L.jo_paged_attention(
            query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), block_tables.data_ptr(),
            query_starts.data_ptr(), kv_lens.data_ptr(), o.data_ptr(), T, B, H, Hk, D, nb, page, width,
            block_tables.stride(0) if B > 1 else width, _S2(a[0], a[1]), _S3(c[0], c[1], c[2]), _S3(d[0], d[1], d[2]),
            _S2(e[0], e[1]), bool(causal), 1.0 / math.sqrt(D) if scale is None else scale,
            T if max_query_len is None else max_query_len, _DT16[dt], ws.data_ptr(),
            ws.numel() * ws.element_size(), st))
    return o


def prompt_attention(query, key, value, seq_starts, *, causal: bool = True, scale: Optional[float] = None, out=None,
                     workspace=None):
    """softmax(scale * q k^T) v of whole packed prompts.

    query [T, H, head_dim], key and value [T, kv_heads, head_dim] (bf16 or fp16,
    head_dim 64 or 128; views with token and head strides that are multiples of 8
    are read in place); request b is rows seq_starts[b] .. seq_starts[b + 1]
    (int32 [B + 1]) of all three.  Row i sees keys 0 .. i of its own request
    (causal) or all of them.  H must be a multiple of kv_heads.  Rows of no
    request are not written.  scale, out and workspace as in paged_attention."""
    dev, dt = query.device, query.dtype
    o = _queries(query, out, dev)
    T, H, D = query.shape
    _chk(key.dim() == 3 and key.shape == value.shape and key.size(0) == T and key.size(2) == D,
         "key and value must be [tokens, kv_heads, head_dim] with query's tokens and head_dim")
    _rows(key, "key", dev, dt)
    _rows(value, "value", dev, dt)
    _ints(seq_starts, "seq_starts", 1, torch.int32, dev)
    _chk(seq_starts.size(0) >= 1, "seq_starts must have batch + 1 entries")
    ws = _workspace(workspace, T, H, D, dev)
    a, b, c, e = query.stride(), key.stride(), value.stride(), o.stride()
    with _On(query) as st:
        _check(_L.jo_prompt_attention(
            query.data_ptr(), key.data_ptr(), value.data_ptr(), seq_starts.data_ptr(), o.data_ptr(), T,
            seq_starts.size(0) - 1, H, key.size(1), D, _S2(a[0], a[1]), _S2(b[0], b[1]), _S2(c[0], c[1]),
            _S2(e[0], e[1]), bool(causal), 1.0 / math.sqrt(D) if scale is None else scale, _DT16[dt], ws.data_ptr(),
            ws.numel() * ws.element_size(), st))
    return o
