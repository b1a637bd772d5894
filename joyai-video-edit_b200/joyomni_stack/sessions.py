"""Many sessions over one paged K/V cache: prompts are encoded packed side by
side, later tokens (one or a chunk a session) attend to what their session has
in the cache.

``SessionCache`` owns the caches of every layer, the block tables and the list
of free blocks; ``SessionAttention`` is the attention half of a pre-norm block with
grouped heads on this package's operators:

    x_q = per_token_fp8(RMSNorm(x));  q, k, v = fp8_scaled_mm(x_q, W_qkv) + b
    q, k = RMSNorm_head + RoPE at the tokens' positions
    cache <- k, v;  o = attention over the session's cache, or over the packed prompts
    x + fp8_scaled_mm(per_token_fp8(o), W_proj) + b        residual in the GEMM epilogue

A step over both (begin() copies the step's lengths and free blocks to the GPU and
waits for that; what follows stays there):

    cache = SessionCache(layers, sessions=8, blocks=512, page_size=64, kv_heads=8, head_dim=128, device=dev)
    lay = cache.begin([77, 0, 12, 1, 1, 0, 0, 300])       # new tokens of every session
    for i, layer in enumerate(blocks):
        x = layer.forward(x, cache, i, lay)
    cache.end()

The reference serves one session from one dense window
(deploy/xvideo/serving/joyomni_streaming.py:959-1124) and encodes prompts with
an external library (deploy/xvideo/models/pipeline.py); this is new.
"""
from __future__ import annotations

from typing import List, Optional, Sequence

import torch

import joyomni_ops as jo

from .mmdit import NORM_EPS, Fp8Weight, quant


class SessionCache:
    """K and V of `sessions` sessions in pages of `page_size` tokens, for every layer.

    The host keeps lengths and block lists of its own (it decides who gets blocks);
    the GPU builds tables and slots from the lengths (``paged_layout``), taking
    blocks from the front of the free list in session order, as the host does.

    A step is what lies between ``begin`` and ``end``.  Its tokens and blocks become the
    sessions' in ``end``: one that is not ended (a layer raised, a retry) is dropped by
    the next ``begin``."""

    def __init__(self, layers: int, sessions: int, blocks: int, page_size: int, kv_heads: int, head_dim: int, device,
                 dtype=torch.bfloat16, max_tokens: Optional[int] = None):
        self.page = page_size
        self.device = device
        shape = (blocks, page_size, kv_heads, head_dim)
        self.caches = [(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device))
                       for _ in range(layers)]
        width = -(-(max_tokens or blocks * page_size) // page_size)
        self.tables = torch.full((sessions, width), -1, dtype=torch.int32, device=device)
        self.free: List[int] = list(range(blocks))
        self.held: List[List[int]] = [[] for _ in range(sessions)]
        self.lens = [0] * sessions
        # of the open step: new tokens of every session, and how many blocks it gets from the free list's front
        self.new = [0] * sessions
        self.taken = [0] * sessions
        self.longest = 0                             # positions that its tokens reach
        self.layout: Optional[jo.PagedLayout] = None

    def begin(self, new_lens: Sequence[int], num_tokens: Optional[int] = None) -> "jo.PagedLayout":
        """Makes room for new_lens[s] tokens of every session s, side by side in the
        step's rows; num_tokens (default: their sum) places of a padded step.  A step
        that is still open is dropped."""
        if len(new_lens) != len(self.lens) or min(new_lens, default=0) < 0:
            raise ValueError("new_lens must have a length of 0 or more for every session")
        total = sum(new_lens)
        if num_tokens is not None and num_tokens < total:
            raise ValueError(f"num_tokens ({num_tokens}) has no room for the step's {total} tokens")
        need = [self._pages(c + n) - self._pages(c) for c, n in zip(self.lens, new_lens)]
        if sum(need) > len(self.free):
            raise RuntimeError(f"{sum(need)} cache blocks are needed, {len(self.free)} are free")
        if max(self._pages(c + n) for c, n in zip(self.lens, new_lens)) > self.tables.size(1):
            raise RuntimeError("a session would be longer than max_tokens")
        lens = torch.tensor([self.lens, list(new_lens)], dtype=torch.int32).to(self.device)
        free = torch.tensor(self.free[:sum(need)], dtype=torch.int32).to(self.device)
        self.layout = jo.paged_layout(lens[0], lens[1], self.tables, free, self.page,
                                      total if num_tokens is None else num_tokens)
        self.new, self.taken = list(new_lens), need
        self.longest = max((c + n for c, n in zip(self.lens, new_lens) if n), default=0)
        return self.layout

    def end(self) -> None:
        """The step's tokens and blocks are part of the sessions now."""
        spare = []                                   # of sessions that ended within the step
        for s, k in enumerate(self.taken):
            if self.new[s] > 0:
                self.held[s] += self.free[:k]
            else:
                spare += self.free[:k]
            del self.free[:k]
        self.free += spare
        self.lens = [c + n for c, n in zip(self.lens, self.new)]
        self.new, self.taken = [0] * len(self.lens), [0] * len(self.lens)

    def _pages(self, tokens: int) -> int:
        return -(-tokens // self.page)

    def release(self, session: int) -> None:
        """Ends a session; its blocks are free for others.  Within a step, its tokens
        of the step go with it (their rows are computed all the same)."""
        self.free += self.held[session]
        self.held[session] = []
        self.lens[session] = 0
        self.new[session] = 0

    def write(self, layer: int, k, v) -> None:
        jo.paged_kv_write(k, v, *self.caches[layer], self.layout.slots)

    def attend(self, layer: int, q, causal: bool = True):
        lay = self.layout
        return jo.paged_attention(q, *self.caches[layer], self.tables, lay.query_starts, lay.kv_lens, causal=causal,
                                  max_query_len=max(self.new))


class SessionAttention:
    """Attention half of a pre-norm block: `heads` query heads, `kv_heads` key heads."""

    def __init__(self, hidden: int, heads: int, kv_heads: int, head_dim: int, device, seed: int = 0,
                 max_positions: int = 65536, rope_theta: float = 10000.0):
        g = torch.Generator(device=device).manual_seed(seed)
        self.heads, self.kv_heads, self.dim = heads, kv_heads, head_dim
        self.norm = (1 + 0.1 * torch.randn(hidden, generator=g, device=device)).to(torch.bfloat16)
        self.q_norm, self.k_norm = ((1 + 0.1 * torch.randn(head_dim, generator=g, device=device)).to(torch.bfloat16)
                                    for _ in "qk")
        self.qkv = Fp8Weight((heads + 2 * kv_heads) * head_dim, hidden, g, device)
        self.proj = Fp8Weight(hidden, heads * head_dim, g, device)
        self.one = torch.ones(hidden, dtype=torch.bfloat16, device=device)
        f = 1.0 / rope_theta ** (torch.arange(0, head_dim, 2, device=device).float() / head_dim)
        angle = torch.outer(torch.arange(max_positions, device=device).float(), f)
        self.cos, self.sin = angle.cos(), angle.sin()

    def project(self, x, positions):
        """q [T, heads, dim], k and v [T, kv_heads, dim] of the rows x at their positions."""
        T, H, Hk, D = x.size(0), self.heads, self.kv_heads, self.dim
        qkv = self.qkv(*quant(jo.rmsnorm(x, self.norm, NORM_EPS))).view(T, H + 2 * Hk, D)
        cos, sin = self.cos[positions], self.sin[positions]

        def turned(t, w):
            n = jo.rmsnorm(t.reshape(-1, D), w, NORM_EPS).view(t.shape)
            return jo.rope_apply(n, cos, sin, out=n)
        return turned(qkv[:, :H], self.q_norm), turned(qkv[:, H:H + Hk], self.k_norm), qkv[:, H + Hk:]

    def forward(self, x, cache: SessionCache, layer: int, layout: "jo.PagedLayout", prompts: bool = False):
        """x [T, hidden], the step's rows.  prompts: every session's tokens of this
        step are all that it has, so that they need not be read back from the cache.
        layout: what the cache's begin() returned for the step."""
        # on the host: on the GPU a position past the tables would be an access out of range
        if layout is not cache.layout:
            raise RuntimeError("layout is not that of the cache's last begin()")
        if cache.longest > self.cos.size(0):
            raise RuntimeError(f"a session reaches {cache.longest} positions, the layer has {self.cos.size(0)} (max_positions)")
        if prompts and any(c and n for c, n in zip(cache.lens, cache.new)):
            raise RuntimeError("prompts=True, but a session has tokens from earlier steps")
        q, k, v = self.project(x, layout.positions)
        cache.write(layer, k, v)
        o = jo.prompt_attention(q, k, v, layout.query_starts) if prompts else cache.attend(layer, q)
        return self.proj.residual(*quant(o.view(x.size(0), -1)), x, self.one)
