"""Attention of a decoder layer over keys and values in 4 bits: what lies between its qkv and its o projection.

No counterpart in the reference, whose layers/attention.py hands the cache to backends that hold 16 or 8
bits. A layer owns one ``KV4Cache``; a forward pass turns queries and keys by their positions (where the layer has a
``Rotary``), appends the new tokens' keys and values and attends over the cache (two launches, a third where the keys
are split over workgroups, one more for the rotary). Of whole prompts, which have their keys and values in hand
in 16 bits, ``prompt_attention`` attends over those. Per-head norms of q and k are the caller's, before it. For a batch
with low-rank adapters the projections around it take ``lora=`` (quant/method.py).
"""
from __future__ import annotations

import importlib
from typing import NamedTuple

import torch

_pkg = __name__.rsplit(".", 2)[0]
_kv4 = importlib.import_module(f"{_pkg}.quant.kv4")
_abi = importlib.import_module(f"{_pkg}._abi")
_host = importlib.import_module(f"{_pkg}._host")
engaged = importlib.import_module(f"{_pkg}._hip_engage").engaged


def _rows(t: torch.Tensor, like: torch.Tensor, name: str, heads: int | None, apart: bool) -> torch.Tensor:
    """(T, heads, D) rows as the kernel takes them: strided, each row of channels contiguous; apart: no row in another."""
    if t.dim() != 3 or t.dtype != like.dtype or t.shape[0] != like.shape[0] or t.shape[2] != like.shape[2] \
            or (heads is not None and t.shape[1] != heads):
        raise TypeError(f"prompt_attention: {name} must be ({like.shape[0]}, {heads or 'heads'}, {like.shape[2]}) {like.dtype}, "
                        f"got {t.dtype} {tuple(t.shape)}")
    if t.device != like.device:
        raise RuntimeError(f"prompt_attention: {name} is on {t.device}, q on {like.device}")
    if not _kv4._rows_ok(t) or (apart and t.shape[0] > 1 and not t.shape[2] <= t.stride(0) < 1 << 23):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def prompt_attention(
    q: torch.Tensor,  # (T, num_qo_heads, head_dim), any strides between rows
    k: torch.Tensor,  # (T, num_kv_heads, head_dim)
    v: torch.Tensor,
    cu_q: torch.Tensor,
    *,
    max_q: int | None = None,
    sm_scale: float | None = None,
    causal: bool = True,
    window: int = 0,
    out: torch.Tensor | None = None,
    return_lse: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Attention over whole prompts, packed: sequence b is the rows cu_q[b] .. cu_q[b+1] - 1 of q, k and v, in bf16 or fp16,
    heads of 64, 128 or 256 channels, num_qo_heads a multiple of num_kv_heads. (T, num_qo_heads, head_dim) in q's type; with
    return_lse also the natural logarithm of each softmax's sum, (T, num_qo_heads) f32.

    causal: a row sees its sequence's rows up to itself; window > 0: only the last ``window`` of those. sm_scale defaults to
    head_dim ** -0.5; it is positive and below 65536. cu_q (B + 1,) int32 is read on the device: a captured call replays with
    new ones, and padded sequences have no rows. A value of v that is not finite makes its channel not finite in the rows
    that see it, and leaves the others alone. Rows outside cu_q keep what they hold in an ``out`` that is given (strided or
    not; q itself, or no part of q, k and v), and are undefined in a fresh one.

    max_q, the most rows of a sequence, is what the host sizes the launch by (default: T). Too large a bound costs
    little time, too low a one more; neither changes what is read. One launch."""
    what = "prompt_attention"
    if sm_scale is None:
        sm_scale = q.shape[-1] ** -0.5
    r = _host.load().prompt_attention(q, k, v, cu_q, max_q, sm_scale, causal, window, out, return_lse)
    if r is not None:
        engaged("w4a8_mi355x.prompt_attention")
        return r if return_lse else r[0]
    if q.dim() != 3 or q.dtype not in (torch.bfloat16, torch.float16) or q.shape[2] not in (64, 128, 256):
        raise TypeError(f"{what}: q must be (T, heads, 64, 128 or 256) in bf16 or fp16, got {q.dtype} {tuple(q.shape)}")
    if not q.is_cuda:
        raise RuntimeError(f"{what}: q must be on the GPU")
    if cu_q.dtype != torch.int32 or cu_q.dim() != 1 or cu_q.shape[0] < 1:
        raise TypeError(f"{what}: cu_q must be a 1-D int32 tensor, got {cu_q.dtype} {tuple(cu_q.shape)}")
    if cu_q.device != q.device:
        raise RuntimeError(f"{what}: cu_q is on {cu_q.device}, q on {q.device}")
    T, Hq, D = q.shape
    q = _rows(q, q, "q", None, False)
    k = _rows(k, q, "k", None, True)
    v = _rows(v, q, "v", k.shape[1], True)
    H = k.shape[1]
    if H < 1 or Hq < H or Hq % H:
        raise ValueError(f"{what}: {Hq} query heads for {H} key/value heads")
    max_q = T if max_q is None else min(int(max_q), T)
    if window < 0 or max_q < 0:
        raise ValueError(f"{what}: window={window}, max_q={max_q}")
    if out is None:
        out = torch.empty((T, Hq, D), dtype=q.dtype, device=q.device)
    elif tuple(out.shape) != (T, Hq, D) or out.dtype != q.dtype or out.device != q.device or not _kv4._rows_ok(out):
        raise ValueError(f"{what}: out must be ({T}, {Hq}, {D}) {q.dtype} with 16-byte aligned rows, got {out.dtype} "
                         f"{tuple(out.shape)} {tuple(out.stride())}")
    cu_q = cu_q.contiguous()
    lse = torch.empty((T, Hq), dtype=torch.float32, device=q.device) if return_lse else None
    with torch.cuda.device(q.device):
        _abi.check(_abi.load().w4a8_prompt_attention(
            q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
            _abi.dtype_code(q.dtype), T, Hq, H, D, cu_q.data_ptr(), cu_q.shape[0] - 1, float(sm_scale), int(bool(causal)),
            int(window), max_q, out.data_ptr(), out.stride(0), out.stride(1), _abi.ptr(lse), _abi.stream_of(q)), what)
    engaged("w4a8_mi355x.prompt_attention")
    return (out, lse) if return_lse else out


class KV4Batch(NamedTuple):
    """The sequences of one forward pass, the same for every layer (quant/kv4.py): ``page_table`` (B, width),
    ``cu_q`` (B + 1,) and ``seq_lens`` (B,) int32 on the device, the lengths with the new tokens; ``max_q`` and
    ``max_kv`` bound a sequence's new tokens and length, on the host: without ``max_q`` a decode step is planned as one
    prompt might be (64 users of up to 8192 tokens 336 us, with max_q=1 77).

    ``positions`` (T,) or (axes, T) int32 or int64 on the device, for layers with a ``Rotary`` (a tree brings its own, for one
    axis). ``tree``: the new tokens are drafted ones (``kv4_tree``). ``whole``: every token of every sequence is new, so
    attention reads keys and values as they are given, and not their 4-bit form in the cache (which is written all the
    same): nearer to the model's own, and for prompts of 8192 the faster way."""

    page_table: torch.Tensor
    cu_q: torch.Tensor
    seq_lens: torch.Tensor
    max_q: int | None = None
    max_kv: int | None = None
    positions: torch.Tensor | None = None
    tree: "_kv4.KV4Tree | None" = None
    whole: bool = False


class KV4Attention:
    """``num_qo_heads`` query heads over the heads of ``cache``; ``sm_scale`` defaults to head_dim ** -0.5,
    ``window`` > 0 keeps the last so many keys in sight, ``rotary`` (layers/rotary.py) turns queries and keys."""

    def __init__(self, num_qo_heads: int, cache: "_kv4.KV4Cache", *, sm_scale: float | None = None, window: int = 0,
                 rotary=None) -> None:
        if num_qo_heads < cache.num_kv_heads or num_qo_heads % cache.num_kv_heads:
            raise ValueError(f"KV4Attention: {num_qo_heads} query heads for {cache.num_kv_heads} key/value heads")
        if rotary is not None and rotary.head_dim != cache.head_dim:
            raise ValueError(f"KV4Attention: a rotary for heads of {rotary.head_dim} channels, the cache has {cache.head_dim}")
        self.num_qo_heads, self.cache, self.sm_scale, self.window = num_qo_heads, cache, sm_scale, window
        self.rotary = rotary

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, batch: KV4Batch) -> torch.Tensor:
        """q (T, num_qo_heads * head_dim), k and v (T, num_kv_heads * head_dim), of any row strides ->
        (T, num_qo_heads * head_dim)."""
        c = self.cache
        T, D = q.shape[0], c.head_dim
        q, k, v = (t.view(T, h, D) for t, h in ((q, self.num_qo_heads), (k, c.num_kv_heads), (v, c.num_kv_heads)))
        if batch.whole and batch.tree is not None:
            raise ValueError("KV4Attention: whole prompts have no tree")
        if self.rotary is not None:
            positions = batch.positions if batch.positions is not None or batch.tree is None else batch.tree.positions
            if positions is None:
                raise ValueError("KV4Attention: a layer with a rotary needs the batch's positions")
            q, k = self.rotary.forward(q, k, positions)
        _kv4.kv4_append(c, k, v, batch.page_table, batch.cu_q, batch.seq_lens)
        if batch.whole:
            out = prompt_attention(q, k, v, batch.cu_q, max_q=batch.max_q, sm_scale=self.sm_scale, window=self.window)
        else:
            out = _kv4.kv4_attention(q, c, batch.page_table, batch.cu_q, batch.seq_lens, max_q=batch.max_q,
                                     max_kv=batch.max_kv, sm_scale=self.sm_scale, window=self.window, tree=batch.tree)
        return out.view(T, self.num_qo_heads * D)

    def forward_qkv(self, qkv: torch.Tensor, batch: KV4Batch) -> torch.Tensor:
        """The same on a merged projection's output (T, (num_qo_heads + 2 num_kv_heads) * head_dim)."""
        kv = self.cache.num_kv_heads * self.cache.head_dim
        return self.forward(*qkv.split([self.num_qo_heads * self.cache.head_dim, kv, kv], dim=1), batch)
