"""Attention of a decoder layer over keys and values in 4 bits: what lies between its qkv and its o projection.

No counterpart in the reference, whose layers/attention.py hands the cache to backends that hold 16 or 8
bits. A layer owns one ``KV4Cache``; a forward pass appends the new tokens' keys and values and attends
over the cache (two launches, a third where the keys are split over workgroups). Rotary embeddings and
per-head norms of q and k are the caller's, before it. For a batch with low-rank adapters the projections
around it take ``lora=`` (quant/method.py).
"""
from __future__ import annotations

import importlib
from typing import NamedTuple

import torch

_pkg = __name__.rsplit(".", 2)[0]
_kv4 = importlib.import_module(f"{_pkg}.quant.kv4")


class KV4Batch(NamedTuple):
    """The sequences of one forward pass, the same for every layer (quant/kv4.py): ``page_table`` (B, width),
    ``cu_q`` (B + 1,) and ``seq_lens`` (B,) int32 on the device, the lengths with the new tokens; ``max_q`` and
    ``max_kv`` bound a sequence's new tokens and length, on the host: without ``max_q`` a decode step is planned as one
    prompt might be (64 users of up to 8192 tokens 336 us, with max_q=1 77)."""

    page_table: torch.Tensor
    cu_q: torch.Tensor
    seq_lens: torch.Tensor
    max_q: int | None = None
    max_kv: int | None = None


class KV4Attention:
    """``num_qo_heads`` query heads over the heads of ``cache``; ``sm_scale`` defaults to head_dim ** -0.5,
    ``window`` > 0 keeps the last so many keys in sight."""

    def __init__(self, num_qo_heads: int, cache: "_kv4.KV4Cache", *, sm_scale: float | None = None, window: int = 0) -> None:
        if num_qo_heads < cache.num_kv_heads or num_qo_heads % cache.num_kv_heads:
            raise ValueError(f"KV4Attention: {num_qo_heads} query heads for {cache.num_kv_heads} key/value heads")
        self.num_qo_heads, self.cache, self.sm_scale, self.window = num_qo_heads, cache, sm_scale, window

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, batch: KV4Batch) -> torch.Tensor:
        """q (T, num_qo_heads * head_dim), k and v (T, num_kv_heads * head_dim), of any row strides ->
        (T, num_qo_heads * head_dim)."""
        c = self.cache
        T, D = q.shape[0], c.head_dim
        q, k, v = (t.view(T, h, D) for t, h in ((q, self.num_qo_heads), (k, c.num_kv_heads), (v, c.num_kv_heads)))
        _kv4.kv4_append(c, k, v, batch.page_table, batch.cu_q, batch.seq_lens)
        out = _kv4.kv4_attention(q, c, batch.page_table, batch.cu_q, batch.seq_lens, max_q=batch.max_q,
                                 max_kv=batch.max_kv, sm_scale=self.sm_scale, window=self.window)
        return out.view(T, self.num_qo_heads * D)

    def forward_qkv(self, qkv: torch.Tensor, batch: KV4Batch) -> torch.Tensor:
        """The same on a merged projection's output (T, (num_qo_heads + 2 num_kv_heads) * head_dim)."""
        kv = self.cache.num_kv_heads * self.cache.head_dim
        return self.forward(*qkv.split([self.num_qo_heads * self.cache.head_dim, kv, kv], dim=1), batch)
