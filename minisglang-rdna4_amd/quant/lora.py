"""Low-rank adapters of many requests at once beside a shared projection.

No counterpart in the reference. Requests that share a quantized model each bring a low-rank pair (A, B)
per projection; a batch mixes them in any order, with requests that have none. ``adapters`` (M,) int32,
on the device, names each row's adapter (-1, or anything else outside 0 .. L-1: none):

    y[m] = base[m] + scaling[l] * (x[m] A_l^T) B_l^T,    l = adapters[m]

``w4a8_linear_lora`` is w4a8_linear with it, ``lora_add`` adds it to the output of any projection (an
unquantized lm_head, the W4A16 arm, an expert's). Both run on the current stream, allocate with torch and
synchronise nothing, and a captured call replays with other adapters.
"""
from __future__ import annotations

import ctypes
from typing import Sequence

import torch

from .. import _abi, _host
from .._hip_engage import engaged
from . import kernels

_DTYPES = (torch.bfloat16, torch.float16)
_MAX_RANK, _MAX_SLICES = 256, 8

_LEDGER = {False: "w4a8_mi355x.linear_lora(int4)", True: "w4a8_mi355x.linear_lora(e2m1)"}


class LoraAdapters:
    """L adapters of one projection, checked once.

    ``a`` (L, S * rank, K) and ``b`` (L, N, rank) in the model's type (bf16 or fp16), ``scaling`` (L,) f32
    (alpha / rank, as a rule). ``slices``: the output widths of the S projections that are merged in the
    weight (q, k and v; gate and up), multiples of 16; slice i uses the rank rows i * rank .. of ``a``. The
    rank is a multiple of 8 up to 256: adapters of lower rank are padded with zeros. The tensors are kept,
    not copied: an adapter is replaced by writing into its place."""

    def __init__(self, a: torch.Tensor, b: torch.Tensor, scaling: torch.Tensor, slices: Sequence[int] | None = None) -> None:
        if a.dim() != 3 or b.dim() != 3 or a.dtype not in _DTYPES or b.dtype != a.dtype:
            raise TypeError(f"LoraAdapters: a (L, slices * rank, K) and b (L, N, rank) in bf16 or fp16, got {a.dtype} "
                            f"{tuple(a.shape)} and {b.dtype} {tuple(b.shape)}")
        L, N, rank = b.shape
        slices = tuple(int(w) for w in slices) if slices is not None else (N,)
        if not 1 <= len(slices) <= _MAX_SLICES or sum(slices) != N or any(w <= 0 or w % 16 for w in slices):
            raise ValueError(f"LoraAdapters: slices must be 1 to {_MAX_SLICES} multiples of 16 that add up to N={N}, got "
                             f"{slices}")
        if rank < 8 or rank > _MAX_RANK or rank % 8:
            raise ValueError(f"LoraAdapters: the rank must be a multiple of 8 up to {_MAX_RANK}, got {rank} (pad a and b "
                             f"with zeros)")
        if L < 1 or a.shape[0] != L or a.shape[1] != len(slices) * rank or a.shape[2] < 8 or a.shape[2] % 8:
            raise ValueError(f"LoraAdapters: for b {tuple(b.shape)} and {len(slices)} slices, a must be ({L}, "
                             f"{len(slices) * rank}, K) with K a multiple of 8, got {tuple(a.shape)}")
        if scaling.dtype != torch.float32 or tuple(scaling.shape) != (L,):
            raise TypeError(f"LoraAdapters: scaling must be ({L},) float32, got {scaling.dtype} {tuple(scaling.shape)}")
        for name, t in (("a", a), ("b", b), ("scaling", scaling)):
            if t.device != a.device or not t.is_contiguous() or (name != "scaling" and t.data_ptr() % 16):
                raise ValueError(f"LoraAdapters: {name} must be contiguous, 16-byte aligned and on {a.device}")
        self.a, self.b, self.scaling, self.slices = a, b, scaling, slices
        self.rank, self.in_features, self.out_features = rank, a.shape[2], N
        self._cols = (ctypes.c_int64 * len(slices))(*slices)

    def __len__(self) -> int:
        return self.b.shape[0]


def _check(x: torch.Tensor, lora: LoraAdapters, adapters: torch.Tensor, what: str) -> None:
    if x.dim() != 2 or x.dtype != lora.a.dtype or x.shape[1] != lora.in_features:
        raise TypeError(f"{what}: x must be (M, {lora.in_features}) {lora.a.dtype} as the adapters are, got {x.dtype} "
                        f"{tuple(x.shape)}")
    if adapters.dtype != torch.int32 or tuple(adapters.shape) != (x.shape[0],):
        raise TypeError(f"{what}: adapters must be ({x.shape[0]},) int32, got {adapters.dtype} {tuple(adapters.shape)}")
    if not x.is_cuda or x.device != lora.a.device or adapters.device != x.device:
        raise RuntimeError(f"{what}: x, adapters and the adapters' weights must be on one GPU, got {x.device}, "
                           f"{adapters.device} and {lora.a.device}")


def _rows_ok(t: torch.Tensor) -> bool:
    return t.stride(1) == 1 and (t.shape[0] <= 1 or (t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1])) and t.data_ptr() % 16 == 0


def _add(base: torch.Tensor, x: torch.Tensor, lora: LoraAdapters, adapters: torch.Tensor, out: torch.Tensor, what: str):
    M, K = x.shape
    if not _rows_ok(x):
        x = x.clone(memory_format=torch.contiguous_format)  # contiguous() leaves what is, wherever it begins
    adapters = adapters.contiguous()
    lib = _abi.load()
    ws_bytes = int(lib.w4a8_lora_workspace_bytes(M, K, lora.rank, len(lora.slices)))
    ws = torch.empty((max(ws_bytes, 1),), dtype=torch.uint8, device=x.device)
    ld = lambda t: t.stride(0) if M > 1 else lora.out_features  # noqa: E731
    with torch.cuda.device(x.device):
        _abi.check(lib.w4a8_lora_add(
            x.data_ptr(), _abi.dtype_code(x.dtype), M, K, x.stride(0) if M > 1 else K, lora.a.data_ptr(), lora.b.data_ptr(),
            lora.scaling.data_ptr(), len(lora), lora.rank, ctypes.addressof(lora._cols), len(lora.slices),
            adapters.data_ptr(), base.data_ptr(), _abi.dtype_code(base.dtype), ld(base), out.data_ptr(), ld(out),
            ws.data_ptr(), ws_bytes, _abi.stream_of(x)), what)
    return out


def lora_add(y: torch.Tensor, x: torch.Tensor, lora: LoraAdapters, adapters: torch.Tensor,
             out: torch.Tensor | None = None) -> torch.Tensor:
    """y + scaling (x A^T) B^T per row, into y itself (returned) or into ``out``: y (M, N) is a projection's
    output for x (M, K), both in the adapters' type, their rows strided or not. ``out`` shares no memory
    with y, or is y. Rows without an adapter keep y's values. The sum is in f32 and rounded once; an
    infinity in x A^T makes NaN of that row's slice, and of nothing else."""
    what = "lora_add"
    if _host.load().lora_add(lora.a, lora.b, lora.scaling, lora.slices, adapters, y, x, y if out is None else out):
        engaged("w4a8_mi355x.lora_add")
        return y if out is None else out
    _check(x, lora, adapters, what)
    out = y if out is None else out
    for name, t in (("y", y), ("out", out)):
        if tuple(t.shape) != (x.shape[0], lora.out_features) or t.dtype != x.dtype or t.device != x.device or not _rows_ok(t):
            raise ValueError(f"{what}: {name} must be ({x.shape[0]}, {lora.out_features}) {x.dtype} on {x.device} with 16-byte "
                             f"aligned rows, got {t.dtype} {tuple(t.shape)} {tuple(t.stride())}")
    _add(y, x, lora, adapters, out, what)
    engaged("w4a8_mi355x.lora_add")
    return out


def w4a8_linear_lora(
    x: torch.Tensor,
    w_packed: torch.Tensor,  # as w4a8_linear takes them
    scales: torch.Tensor,
    w_zeros: torch.Tensor | None,
    group_size: int,
    lora: LoraAdapters,
    adapters: torch.Tensor,  # (M,) int32
    kernel: str | None = None,
    weight_is_e2m1: bool = False,
    x_fp8: torch.Tensor | None = None,
    act_scales: torch.Tensor | None = None,
) -> torch.Tensor:
    """``kernels.w4a8_linear`` plus each row's adapter: (M, N) in x's dtype. The adapters take x
    unquantized, also where the producer pair is given for the projection. The sum is in f32 and rounded
    once, so the call takes 4 bytes of workspace per output."""
    what = "w4a8_linear_lora"
    if x.is_cuda and (kernel is None or kernel == "decode_gemv"):
        r = _host.load().linear_lora(lora.a, lora.b, lora.scaling, lora.slices, adapters, x, w_packed, scales, w_zeros,
                                     group_size, weight_is_e2m1, x_fp8, act_scales,
                                     _abi.KERNEL_AUTO if kernel is None else _abi.KERNEL_DECODE)
        if r is not None:
            engaged(_LEDGER[bool(weight_is_e2m1)])
            return r
    _check(x, lora, adapters, what)
    if kernels._n_of(w_packed) != lora.out_features:
        raise ValueError(f"{what}: the weight has {kernels._n_of(w_packed)} output channels, the adapters "
                         f"{lora.out_features}")
    # in f32 until the adapters' part is added: rounding the projection's output to the type before would save a fifth
    # of its traffic (1777 x 2560 -> 19456 198 us where this takes 215, 2048 x 4096 -> 28672 305 and 365), and cost
    # 1.4 times the error of one rounding
    arm, _ = kernels._dense_arm(x, w_packed, group_size, kernel, weight_is_e2m1, x_fp8)
    with torch.cuda.device(x.device):  # _dense launches on the current one
        base, _ = kernels._dense(x, w_packed, scales, w_zeros, group_size, weight_is_e2m1, x_fp8, act_scales, False, arm,
                                 torch.float32)
    out = torch.empty((x.shape[0], lora.out_features), dtype=x.dtype, device=x.device)
    _add(base, x, lora, adapters, out, what)
    engaged(_LEDGER[bool(weight_is_e2m1)])
    return out
