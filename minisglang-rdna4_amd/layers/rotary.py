"""Rotary positions of queries and keys, with one position per token or several (time, height and width of images and
video).

Not a mirror of the reference's layers/rotary.py, which lies outside what this package restates. Pair i of a head's
first ``rotary_dim`` channels is turned by position[axis of i] * f_i, in f32 and rounded once. Angles are worked out in the
kernel from whole positions and frequencies as 64-bit fractions of a turn, with no table of sines and cosines to keep or to
outgrow: off by 2^-32 of a turn, and by 2^-65 for each position from 0 (at 2^31 2^-34, at 2^45 2^-20).
"""
from __future__ import annotations

import functools
import importlib
import math
from typing import Sequence

import torch

_pkg = __name__.rsplit(".", 2)[0]
_abi = importlib.import_module(f"{_pkg}._abi")
_host = importlib.import_module(f"{_pkg}._host")
engaged = importlib.import_module(f"{_pkg}._hip_engage").engaged

_MAX_AXES = 8


@functools.lru_cache(maxsize=None)
def _two_pi(bits: int) -> int:
    """2 pi in 2^-bits, to the last place or two: 8 (4 atan(1/5) - atan(1/239)), Machin's sum."""
    one = 1 << (bits + 16)

    def atan(n: int) -> int:
        term = one // n
        total, k = 0, 1
        while term:
            total += term // k if k % 4 == 1 else -(term // k)
            term //= n * n
            k += 2
        return total

    return (8 * (4 * atan(5) - atan(239))) >> 16


def _turns(freq: float) -> int:
    """freq / 2 pi modulo 1 in units of 2^-64, to the nearest."""
    bits = 96 + max(0, math.frexp(freq)[1])
    n, d = freq.as_integer_ratio()
    d *= _two_pi(bits)
    n <<= 64 + bits
    return ((2 * n + d) // (2 * d)) % (1 << 64)


def _rows_ok(t: torch.Tensor) -> bool:
    return t.stride(2) == 1 and all(t.shape[i] <= 1 or t.stride(i) % 8 == 0 for i in (0, 1)) and t.data_ptr() % 16 == 0


class Rotary:
    """Rotary positions for heads of ``head_dim`` channels (a multiple of 8, up to 1024), of which the first ``rotary_dim``
    (default: all; a multiple of 16) turn: pairs are channels i and i + rotary_dim/2, or with ``adjacent`` 2i and 2i + 1.

    Frequencies are base ** (-2i / rotary_dim) in f64, or ``inv_freq`` (rotary_dim/2 of them, f64 at best: scaled ones are given
    this way). ``scale`` multiplies the turned channels (attention factors of scaled frequencies). ``sections``: with several axes
    of positions, the pairs of each axis, which add up to rotary_dim/2; the first pairs are axis 0's, the next axis 1's, or
    with ``interleaved`` pair i is axis i % axes' while i < axes * sections[i % axes], and else axis 0's."""

    def __init__(self, head_dim: int, *, base: float = 10000.0, inv_freq: torch.Tensor | Sequence[float] | None = None,
                 rotary_dim: int | None = None, sections: Sequence[int] | None = None, interleaved: bool = False,
                 adjacent: bool = False, scale: float = 1.0, device: torch.device | str = "cuda") -> None:
        rotary_dim = head_dim if rotary_dim is None else int(rotary_dim)
        if head_dim < 16 or head_dim > 1024 or head_dim % 8 or rotary_dim < 16 or rotary_dim > head_dim or rotary_dim % 16:
            raise ValueError(f"Rotary: heads of 16 to 1024 channels (a multiple of 8), a multiple of 16 of which turn, got "
                             f"{rotary_dim} of {head_dim}")
        pairs = rotary_dim // 2
        if inv_freq is None:
            if not base > 0:
                raise ValueError(f"Rotary: base={base}")
            freq = [float(base) ** (-2.0 * i / rotary_dim) for i in range(pairs)]
        else:
            freq = [float(f) for f in (inv_freq.tolist() if isinstance(inv_freq, torch.Tensor) else inv_freq)]
        if len(freq) != pairs or not all(math.isfinite(f) for f in freq) or not math.isfinite(scale):
            raise ValueError(f"Rotary: {pairs} finite frequencies and a finite scale, got {len(freq)} and {scale}")
        sections = (pairs,) if sections is None else tuple(int(n) for n in sections)
        if not 1 <= len(sections) <= _MAX_AXES or any(n < 0 for n in sections) or sum(sections) != pairs:
            raise ValueError(f"Rotary: sections must be 1 to {_MAX_AXES} counts that add up to {pairs}, got {sections}")
        axes = len(sections)
        if interleaved and any(n and a and a + (n - 1) * axes >= pairs for a, n in enumerate(sections)):
            raise ValueError(f"Rotary: interleaved sections {sections} do not fit into {pairs} pairs")
        if interleaved:
            axis = [i % axes if i < axes * sections[i % axes] else 0 for i in range(pairs)]
        else:
            axis = [a for a, n in enumerate(sections) for _ in range(n)]
        # turns per position, whose product with the position wraps as it should; signed, as torch's integers are
        turns = [(_turns(f) + (1 << 63)) % (1 << 64) - (1 << 63) for f in freq]
        self.head_dim, self.rotary_dim, self.axes = head_dim, rotary_dim, axes
        self.sections, self.adjacent, self.scale = sections, bool(adjacent), float(scale)
        self.turns = torch.tensor(turns, dtype=torch.int64, device=device)
        self.axis = torch.tensor(axis, dtype=torch.int32, device=device)

    def forward(self, q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """q (T, heads, head_dim) and k (T, other heads, head_dim), of any strides between rows, in bf16 or fp16, turned by
        positions (T,) or (axes, T), int32 or int64: contiguous tensors of their shapes. One launch."""
        return self._run(q, k, positions, False)

    def forward_inplace(self, q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor) -> None:
        """The same in q's and k's own storage, whose rows must be 16-byte aligned (columns of a merged projection's
        output, as a rule)."""
        self._run(q, k, positions, True)

    def _run(self, q, k, positions, inplace: bool):
        r = _host.load().rotary(self.turns, self.axis, self.axes, self.head_dim, self.rotary_dim, self.adjacent, self.scale, q, k,
                                positions, inplace)
        if r is not None:
            engaged("w4a8_mi355x.rotary")
            return r
        what = "Rotary"
        if q.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"{what}: bf16 or fp16, got {q.dtype}")
        for name, t in (("q", q), ("k", k)):
            if t.dim() != 3 or t.dtype != q.dtype or t.shape[0] != q.shape[0] or t.shape[1] < 1 or t.shape[2] != self.head_dim:
                raise TypeError(f"{what}: {name} must be ({q.shape[0]}, heads, {self.head_dim}) {q.dtype}, got {t.dtype} "
                                f"{tuple(t.shape)}")
        T = q.shape[0]
        if positions.dtype not in (torch.int32, torch.int64) or tuple(positions.shape) not in (
                ((T,), (1, T)) if self.axes == 1 else ((self.axes, T),)):
            raise TypeError(f"{what}: positions must be {(T,) if self.axes == 1 else (self.axes, T)} int32 or int64, got "
                            f"{positions.dtype} {tuple(positions.shape)}")
        if not q.is_cuda or any(t.device != q.device for t in (k, positions, self.turns)):
            raise RuntimeError(f"{what}: q, k, positions and the rotary must be on one GPU, got {q.device}, {k.device}, "
                               f"{positions.device} and {self.turns.device}")
        if inplace:
            if not _rows_ok(q) or not _rows_ok(k):
                raise ValueError(f"{what}: in place, rows must be 16-byte aligned with strides that are multiples of 8, got "
                                 f"{tuple(q.stride())} and {tuple(k.stride())}")
            qo, ko = q, k
        else:
            q, k = (t if _rows_ok(t) else t.clone(memory_format=torch.contiguous_format) for t in (q, k))
            qo, ko = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))
        positions = positions.contiguous()
        with torch.cuda.device(q.device):
            _abi.check(_abi.load().w4a8_rotary(
                q.data_ptr(), q.stride(0), q.stride(1), q.shape[1], k.data_ptr(), k.stride(0), k.stride(1), k.shape[1],
                _abi.dtype_code(q.dtype), T, self.head_dim, self.rotary_dim, int(self.adjacent), positions.data_ptr(),
                int(positions.dtype == torch.int64), self.axes, T, self.turns.data_ptr(), self.axis.data_ptr(), self.scale,
                qo.data_ptr(), qo.stride(0), qo.stride(1), ko.data_ptr(), ko.stride(0), ko.stride(1), _abi.stream_of(q)), what)
        engaged("w4a8_mi355x.rotary")
        return qo, ko
