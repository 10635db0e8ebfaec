"""A serving step on the quantized modules: requests of any lengths, prompts and
single tokens mixed, over a paged key/value cache.

    cache = PagedKVCache(layers, pages, page_size, kv_heads, head_dim, requests, device=dev)
    step = cache.plan([17, 1, 0, 1])          # new tokens of each request this step
    for i, layer in enumerate(model):
        x = layer(x, cos, sin, cache, i, step)  # x [17 + 1 + 1, dims], requests in order
    cache.release(1)                          # its pages are free again

``PagedDecoderLayer`` strings the operators together: the quantized q|k|v
projection, ``kq.rope_kv_write`` into the cache, ``kq.paged_attention`` over it,
the output projection, then ``kq.moe_route`` and the quantized expert stacks.
Everything but the requests' lengths stays on the GPU and in stream order: a
step never waits for the device.
"""
from __future__ import annotations

from collections.abc import Sequence
from typing import NamedTuple

import torch
from torch import nn

from . import kq
from .nn import KQuantLinear, KQuantSwitchGLU


class Step(NamedTuple):
    """What the layers of one step share."""
    plan: kq.PagedPlan
    max_query_len: int


class PagedKVCache:
    """Key/value pages of all layers, with the requests' block tables and lengths.

    ``pages`` pages of ``page_size`` tokens serve up to ``requests`` requests, each
    of up to ``max_pages`` pages (default: all).  A page has the same number in
    every layer.  The lengths are known on the host; tables and the list of free
    pages live on the GPU."""

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, requests: int,
                 max_pages: int | None = None, dtype: torch.dtype = torch.bfloat16, device=None):
        shape = (layers, pages, page_size, kv_heads, head_dim)
        self.k, self.v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        self.page_size = page_size
        self.tables = torch.full((requests, pages if max_pages is None else max_pages), -1, dtype=torch.int32,
                                 device=device)
        self.free = torch.arange(pages, dtype=torch.int32, device=device)
        self.lens = [0] * requests

    def _pages(self, tokens: int) -> int:
        return -(-tokens // self.page_size)

    def plan(self, query_lens: Sequence[int]) -> Step:
        """Admits ``query_lens[b]`` new tokens of every request (0: it sits the step
        out) and says where they go.  Refuses, with nothing changed, what the pages
        do not hold."""
        if len(query_lens) != len(self.lens) or min(query_lens, default=0) < 0:
            raise ValueError(f"plan: {len(self.lens)} lengths of 0 or more expected, got {list(query_lens)}")
        total = [c + n for c, n in zip(self.lens, query_lens)]
        if max(map(self._pages, total), default=0) > self.tables.shape[1]:
            raise ValueError(f"plan: a request of {max(total)} tokens needs more than {self.tables.shape[1]} pages")
        need = sum(self._pages(t) - self._pages(c) for t, c in zip(total, self.lens))
        if need > self.free.shape[0]:
            raise ValueError(f"plan: {need} pages needed, {self.free.shape[0]} free")
        # (from pinned memory, which the allocator holds until the copy is done: from other
        # memory the copy would wait for all that is queued)
        ctx, new = torch.tensor([self.lens, list(query_lens)], dtype=torch.int32,
                                pin_memory=self.free.is_cuda).to(self.free.device, non_blocking=True)
        p = kq.paged_plan(ctx, new, self.tables, self.free, self.page_size, sum(query_lens))
        self.free, self.lens = self.free[need:], total
        return Step(p, max(query_lens, default=0))

    def release(self, request: int) -> None:
        """Ends a request: its pages go back to the free list."""
        held = self._pages(self.lens[request])
        self.free = torch.cat([self.free, self.tables[request, :held]])
        self.lens[request] = 0


def rope_tables(positions: int, rot: int, base: float = 10000.0, device=None) -> tuple[torch.Tensor, torch.Tensor]:
    """cos and sin ``[positions, rot / 2]`` of angle ``p * base^(-2i / rot)``, computed
    in 64 bits (an f32 product is off by 2^-8 radians at position 2^16) and held in f32."""
    f = base ** (torch.arange(0, rot, 2, dtype=torch.float64, device=device) / -max(rot, 1))
    a = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * f
    return a.cos().float(), a.sin().float()


def _rms_norm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    f = x.float()
    return (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + eps) * w.float()).to(x.dtype)


class PagedDecoderLayer(nn.Module):
    """Attention over the paged cache and a routed expert block, both pre-normed
    and with residuals, all projections quantized.  ``forward`` takes the step's
    tokens ``x [tokens, dims]`` (bf16 or fp16, the cache's type)."""

    def __init__(self, dims: int, heads: int, kv_heads: int, head_dim: int, experts: int, top_k: int,
                 expert_dims: int, codec: str = "q4_k", down_codec: str | None = None, interleaved: bool = False,
                 window: int = 0, softcap: float = 0.0, scoring: str = "softmax", n_groups: int = 1,
                 topk_groups: int = 1, route_scale: float = 1.0, eps: float = 1e-6, dtype=torch.bfloat16,
                 device=None):
        super().__init__()
        self.heads, self.kv_heads, self.head_dim, self.eps = heads, kv_heads, head_dim, eps
        self.interleaved, self.window, self.softcap = interleaved, window, softcap
        self.top_k, self.routing = top_k, dict(scoring=scoring, n_groups=n_groups, topk_groups=topk_groups,
                                               scale=route_scale)
        self.qkv = KQuantLinear(dims, (heads + 2 * kv_heads) * head_dim, False, codec, device)
        self.o = KQuantLinear(heads * head_dim, dims, False, codec, device)
        self.experts = KQuantSwitchGLU(dims, expert_dims, experts, codec, down_codec, device=device)
        self.gate = nn.Linear(dims, experts, bias=False, device=device, dtype=dtype).requires_grad_(False)
        self.register_buffer("attn_norm", torch.ones(dims, device=device))
        self.register_buffer("ffn_norm", torch.ones(dims, device=device))
        # the balance bias that sigmoid routers add to the choice
        self.register_buffer("route_bias", torch.zeros(experts, device=device) if scoring == "sigmoid" else None)

    def forward(self, x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, cache: PagedKVCache, layer: int,
                step: Step) -> torch.Tensor:
        p, t = step.plan, x.shape[0]
        if t == 0:
            return x
        kc, vc = cache.k[layer], cache.v[layer]
        qkv = self.qkv(_rms_norm(x, self.attn_norm, self.eps)).view(t, -1, self.head_dim)
        q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], 1)
        q = kq.rope_kv_write(q, k, v, cos, sin, p.positions, kc, vc, p.slots, self.interleaved)
        a = kq.paged_attention(q, kc, vc, cache.tables, p.seq_lens, p.cu_seqlens, step.max_query_len,
                               window=self.window, softcap=self.softcap)
        x = x + self.o(a.view(t, -1))
        h = _rms_norm(x, self.ffn_norm, self.eps)
        idx, w = kq.moe_route(self.gate(h), self.top_k, bias=self.route_bias, **self.routing)
        return x + self.experts(h, idx, w)
