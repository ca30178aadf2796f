"""Keys and values in 4 bits: a paged cache, writing and reading it, and attention over it.

No counterpart in the reference, whose cache holds 16 or 8 bits (its python/minisgl/kvcache). A cached
vector of one token and key/value head is codes c in 0..15 with a step s and a least value m in the
model's type and stands for s c + m; the formulas and the memory layout, which is that of the matrix
units' operands, are in include/w4a8_mi355x.h. 4 + 32/D bits a value, about a quarter of bf16's.

Sequences are described as attention backends describe a ragged batch: ``page_table`` (B, width) int32,
``cu_q`` (B + 1,) int32, the first row of each sequence's new tokens and their total, and ``seq_lens``
(B,) int32, each length with the new tokens, which are the sequence's last. All three are read on the
device: a captured call replays with new ones. Decode passes one row per sequence, ``cu_q`` 0, 1, 2, ...
A padded sequence has length 0 (its rows are 0 in the output) or no rows.

Drafted tokens (speculative decoding) are appended like any others; ``kv4_tree`` turns their parents into what
``kv4_attention(tree=)`` masks by, and ``kv4_keep`` puts the accepted ones behind the context. A sequence is forked by
sharing its full pages and copying the last one (``kv4_copy_pages``); freeing a page takes nothing.

Every function runs on the current stream of its tensors' device and allocates with torch; nothing
synchronises.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Sequence

import torch

from .. import _abi, _host
from .._hip_engage import engaged

_DTYPES = (torch.bfloat16, torch.float16)
_HEAD_DIMS = (64, 128, 256)
_TREE_WORDS = 128


class KV4Cache:
    """The cache of one attention layer: ``num_pages`` pages of ``page_size`` tokens (a power of two from
    16) for ``num_kv_heads`` heads of ``head_dim`` (64, 128 or 256) channels of a model in ``dtype``
    (bf16 or fp16).

    ``k`` (pages, heads, page_size, head_dim/2) uint8, ``v`` (pages, heads, page_size/8, head_dim) int32,
    ``k_scale`` and ``v_scale`` (pages, heads, page_size, 2) dtype."""

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda") -> None:
        if dtype not in _DTYPES:
            raise TypeError(f"KV4Cache: bf16 or fp16, got {dtype}")
        if head_dim not in _HEAD_DIMS:
            raise ValueError(f"KV4Cache: heads of 64, 128 or 256 channels, got {head_dim}")
        if page_size < 16 or page_size > 65536 or page_size & (page_size - 1):
            raise ValueError(f"KV4Cache: pages of a power of two tokens from 16 to 65536, got {page_size}")
        if num_pages < 1 or num_kv_heads < 1:
            raise ValueError(f"KV4Cache: {num_pages} pages of {num_kv_heads} heads")
        # zeros: a slot that nobody wrote stands for a vector of zeros
        self._set(torch.zeros((num_pages, num_kv_heads, page_size, head_dim // 2), dtype=torch.uint8, device=device),
                  torch.zeros((num_pages, num_kv_heads, page_size // 8, head_dim), dtype=torch.int32, device=device),
                  torch.zeros((num_pages, num_kv_heads, page_size, 2), dtype=dtype, device=device),
                  torch.zeros((num_pages, num_kv_heads, page_size, 2), dtype=dtype, device=device))

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor) -> "KV4Cache":
        """A cache over existing storage, in the layout above: nothing is copied."""
        if k.dim() != 4 or k.dtype != torch.uint8 or v.dtype != torch.int32 or k_scale.dtype not in _DTYPES:
            raise TypeError(f"KV4Cache: k uint8 (pages, heads, page_size, head_dim/2), v int32 and bf16/fp16 scales, got "
                            f"{k.dtype} {tuple(k.shape)}, {v.dtype}, {k_scale.dtype}")
        pages, heads, page, half = k.shape
        if 2 * half not in _HEAD_DIMS or page < 16 or page > 65536 or page & (page - 1) or pages < 1 or heads < 1:
            raise ValueError(f"KV4Cache: heads of 64, 128 or 256 channels on pages of a power of two tokens from 16 to "
                             f"65536, got k {tuple(k.shape)}")
        scale = (pages, heads, page, 2)
        if tuple(v.shape) != (pages, heads, page // 8, 2 * half) or tuple(k_scale.shape) != scale \
                or tuple(v_scale.shape) != scale or v_scale.dtype != k_scale.dtype:
            raise ValueError(f"KV4Cache: for k {tuple(k.shape)}, v must be {(pages, heads, page // 8, 2 * half)} and the "
                             f"scales {scale} of one type, got {tuple(v.shape)}, {tuple(k_scale.shape)} "
                             f"{k_scale.dtype}, {tuple(v_scale.shape)} {v_scale.dtype}")
        ts = (k, v, k_scale, v_scale)
        if any(not t.is_contiguous() or t.device != k.device or t.data_ptr() % 16 for t in ts):
            raise ValueError("KV4Cache: the four tensors must be contiguous, 16-byte aligned and on one device")
        self = cls.__new__(cls)
        self._set(*ts)
        return self

    def _set(self, k, v, k_scale, v_scale) -> None:
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.num_pages, self.num_kv_heads, self.page_size = k.shape[:3]
        self.head_dim = 2 * k.shape[3]
        self.dtype, self.device = k_scale.dtype, k.device

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale))

    def _ptrs(self):
        return tuple(t.data_ptr() for t in (self.k, self.v, self.k_scale, self.v_scale))


def _batch(cache: KV4Cache, page_table: torch.Tensor, cu_q: torch.Tensor, seq_lens: torch.Tensor, what: str):
    """The ragged batch's checks; (table pointer, stride, width, cu pointer, lens pointer, sequences)."""
    if cache.device.type != "cuda":
        raise RuntimeError(f"{what}: the cache must be on the GPU")
    for name, t, dim in (("page_table", page_table, 2), ("cu_q", cu_q, 1), ("seq_lens", seq_lens, 1)):
        if t.dtype != torch.int32 or t.dim() != dim:
            raise TypeError(f"{what}: {name} must be a {dim}-D int32 tensor, got {t.dtype} {tuple(t.shape)}")
        if t.device != cache.device:
            raise RuntimeError(f"{what}: {name} is on {t.device}, the cache on {cache.device}")
    B = seq_lens.shape[0]
    if cu_q.shape[0] != B + 1 or page_table.shape[0] != B:
        raise ValueError(f"{what}: for {B} sequences cu_q must have {B + 1} entries and page_table {B} rows, got "
                         f"{tuple(cu_q.shape)} and {tuple(page_table.shape)}")
    if (B > 1 and (not seq_lens.is_contiguous())) or not cu_q.is_contiguous():
        raise ValueError(f"{what}: cu_q and seq_lens must be contiguous")
    width = page_table.shape[1]
    if width > 1 and page_table.stride(1) != 1 or (B > 1 and page_table.stride(0) < width):
        raise ValueError(f"{what}: page_table rows must be contiguous, got strides {tuple(page_table.stride())}")
    ldt = page_table.stride(0) if B > 1 else max(width, 1)
    return page_table.data_ptr(), ldt, width, cu_q.data_ptr(), seq_lens.data_ptr(), B


def _tensors(caches) -> tuple:
    """The caches' tensors as the host path takes them, four of each."""
    if isinstance(caches, KV4Cache):
        return caches.k, caches.v, caches.k_scale, caches.v_scale
    return tuple(t for c in caches for t in (c.k, c.v, c.k_scale, c.v_scale))


def _rows_ok(t: torch.Tensor) -> bool:
    return t.stride(2) == 1 and all(t.shape[i] <= 1 or t.stride(i) % 8 == 0 for i in (0, 1)) and t.data_ptr() % 16 == 0


def _rows(t: torch.Tensor, cache: KV4Cache, heads: int | None, name: str, what: str) -> torch.Tensor:
    """(T, heads, head_dim) rows as the kernels take them: strided, each row of channels contiguous."""
    if t.dim() != 3 or t.dtype != cache.dtype or t.shape[2] != cache.head_dim or (heads is not None and t.shape[1] != heads):
        raise TypeError(f"{what}: {name} must be (T, {heads or 'heads'}, {cache.head_dim}) "
                        f"{cache.dtype} as the cache is, got {t.dtype} {tuple(t.shape)}")
    if t.device != cache.device:
        raise RuntimeError(f"{what}: {name} is on {t.device}, the cache on {cache.device}")
    # a copy, not contiguous(): a contiguous tensor may begin anywhere
    return t if _rows_ok(t) else t.clone(memory_format=torch.contiguous_format)


def kv4_append(cache: KV4Cache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, cu_q: torch.Tensor,
               seq_lens: torch.Tensor) -> None:
    """Quantize the new tokens' keys and values (T, num_kv_heads, head_dim), of any strides, into the
    cache: the rows of sequence b are its tokens seq_lens[b] - n .. seq_lens[b] - 1. One launch.

    The 8 tokens of a block share words, so a page that still grows belongs to one sequence; full
    pages may be shared. Rows outside cu_q, before a sequence's first token or on a page that does not
    exist write nothing."""
    what = "kv4_append"
    if _host.load().kv4_append(cache.k, cache.v, cache.k_scale, cache.v_scale, page_table, cu_q, seq_lens, k, v):
        engaged("w4a8_mi355x.kv4_append")
        return
    k = _rows(k, cache, cache.num_kv_heads, "k", what)
    v = _rows(v, cache, cache.num_kv_heads, "v", what)
    if v.shape[0] != k.shape[0]:
        raise ValueError(f"{what}: k has {k.shape[0]} rows, v {v.shape[0]}")
    table, ldt, width, cu, lens, B = _batch(cache, page_table, cu_q, seq_lens, what)
    with torch.cuda.device(cache.device):
        _abi.check(_abi.load().w4a8_kv4_append(
            k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), _abi.dtype_code(k.dtype),
            k.shape[0], cache.num_kv_heads, cache.head_dim, *cache._ptrs(), cache.num_pages, cache.page_size, table, ldt,
            width, cu, lens, B, _abi.stream_of(k)), what)
    engaged("w4a8_mi355x.kv4_append")


def kv4_read(cache: KV4Cache, page_table: torch.Tensor, cu_q: torch.Tensor, seq_lens: torch.Tensor,
             num_rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """The cached values of each sequence's last cu_q[b+1] - cu_q[b] tokens, as (k, v), (num_rows,
    num_kv_heads, head_dim) in the cache's type: what an unquantized attention, an offload or a check
    reads. With cu_q the running sum of seq_lens, whole sequences. Rows outside cu_q are not written; a
    row without a place in the cache is NaN. One launch."""
    what = "kv4_read"
    r = _host.load().kv4_read(cache.k, cache.v, cache.k_scale, cache.v_scale, page_table, cu_q, seq_lens, num_rows)
    if r is not None:
        engaged("w4a8_mi355x.kv4_read")
        return r
    table, ldt, width, cu, lens, B = _batch(cache, page_table, cu_q, seq_lens, what)
    if num_rows < 0:
        raise ValueError(f"{what}: num_rows={num_rows}")
    k = torch.empty((num_rows, cache.num_kv_heads, cache.head_dim), dtype=cache.dtype, device=cache.device)
    v = torch.empty_like(k)
    with torch.cuda.device(cache.device):
        _abi.check(_abi.load().w4a8_kv4_read(
            *cache._ptrs(), _abi.dtype_code(cache.dtype), cache.num_pages, cache.page_size, cache.num_kv_heads,
            cache.head_dim, table, ldt, width, cu, lens, B, num_rows, k.data_ptr(), v.data_ptr(), _abi.stream_of(k)), what)
    engaged("w4a8_mi355x.kv4_read")
    return k, v


class KV4Tree(NamedTuple):
    """What the new tokens of a call see of each other: ``mask`` (T, words) int32, bit j % 32 of word j / 32 for the
    sequence's new token j, and ``positions`` (T,) int32, as rotary embeddings and windows count them. ``kv4_tree`` makes
    it from parents; any other bits may stand there."""

    mask: torch.Tensor
    positions: torch.Tensor


def kv4_tree(parents: torch.Tensor, cu_q: torch.Tensor, seq_lens: torch.Tensor, *, max_q: int, window: int = 0) -> KV4Tree:
    """The tree of drafted tokens whose parents these are: (T,) int32, each the index among its sequence's new tokens of
    the one that it follows, or -1 for the context's last token; a parent stands before its children, and what does not
    is taken as -1. A token sees its ancestors and itself, window > 0: the last ``window`` of them.

    max_q: the most new tokens of a sequence, up to 4096; a token from there on is seen by none. Rows outside cu_q are not
    written. One launch."""
    what = "kv4_tree"
    r = _host.load().kv4_tree(parents, cu_q, seq_lens, max_q, window)
    if r is not None:
        engaged("w4a8_mi355x.kv4_tree")
        return KV4Tree(*r)
    for name, t in (("parents", parents), ("cu_q", cu_q), ("seq_lens", seq_lens)):
        if t.dtype != torch.int32 or t.dim() != 1:
            raise TypeError(f"{what}: {name} must be a 1-D int32 tensor, got {t.dtype} {tuple(t.shape)}")
        if not t.is_cuda or t.device != parents.device:
            raise RuntimeError(f"{what}: parents, cu_q and seq_lens must be on one GPU, got {name} on {t.device}")
    B, T = seq_lens.shape[0], parents.shape[0]
    if cu_q.shape[0] != B + 1:
        raise ValueError(f"{what}: for {B} sequences cu_q must have {B + 1} entries, got {tuple(cu_q.shape)}")
    if not 1 <= max_q <= 32 * _TREE_WORDS or window < 0:
        raise ValueError(f"{what}: max_q={max_q} (1 to {32 * _TREE_WORDS}), window={window}")
    parents, cu_q, seq_lens = (t.contiguous() for t in (parents, cu_q, seq_lens))
    words = (int(max_q) + 31) // 32
    mask = torch.empty((T, words), dtype=torch.int32, device=parents.device)
    pos = torch.empty((T,), dtype=torch.int32, device=parents.device)
    with torch.cuda.device(parents.device):
        _abi.check(_abi.load().w4a8_kv4_tree(parents.data_ptr(), T, cu_q.data_ptr(), seq_lens.data_ptr(), B, words, int(window),
                                             mask.data_ptr(), pos.data_ptr(), _abi.stream_of(parents)), what)
    engaged("w4a8_mi355x.kv4_tree")
    return KV4Tree(mask, pos)


def _layers(caches: KV4Cache | Sequence[KV4Cache], what: str) -> Sequence[KV4Cache]:
    caches = (caches,) if isinstance(caches, KV4Cache) else tuple(caches)
    if not caches:
        raise ValueError(f"{what}: no cache")
    c = caches[0]
    if c.device.type != "cuda":
        raise RuntimeError(f"{what}: the cache must be on the GPU")
    for o in caches[1:]:
        if (o.k.shape, o.dtype, o.device) != (c.k.shape, c.dtype, c.device):
            raise ValueError(f"{what}: the caches must be alike, got {tuple(c.k.shape)} {c.dtype} on {c.device} and "
                             f"{tuple(o.k.shape)} {o.dtype} on {o.device}")
    if len({o.k.data_ptr() for o in caches}) != len(caches):
        raise ValueError(f"{what}: a cache is given twice")
    return caches


def _arrays(caches: Sequence[KV4Cache]):
    return (ctypes.c_void_p * (4 * len(caches)))(*(p for c in caches for p in c._ptrs()))


def kv4_copy_pages(caches: KV4Cache | Sequence[KV4Cache], src: torch.Tensor, dst: torch.Tensor) -> None:
    """Copy page src[i] to page dst[i] in each of the caches (layers of one shape), src and dst (n,) int32 on the device:
    the partial last page of a sequence that is forked, or pages that move to make a cache compact. One launch per 64 caches.

    The destinations are distinct and none of them is another pair's source: such a page would hold parts of either. A
    pair with a page that does not exist, or with twice the same, copies nothing."""
    what = "kv4_copy_pages"
    if _host.load().kv4_copy_pages(_tensors(caches), src, dst):
        engaged("w4a8_mi355x.kv4_copy_pages")
        return
    caches = _layers(caches, what)
    c = caches[0]
    for name, t in (("src", src), ("dst", dst)):
        if t.dtype != torch.int32 or t.dim() != 1:
            raise TypeError(f"{what}: {name} must be a 1-D int32 tensor, got {t.dtype} {tuple(t.shape)}")
        if t.device != c.device:
            raise RuntimeError(f"{what}: {name} is on {t.device}, the caches on {c.device}")
    if src.shape != dst.shape:
        raise ValueError(f"{what}: {src.shape[0]} sources, {dst.shape[0]} destinations")
    src, dst = src.contiguous(), dst.contiguous()
    arrays = _arrays(caches)
    with torch.cuda.device(c.device):
        _abi.check(_abi.load().w4a8_kv4_copy_pages(
            ctypes.addressof(arrays), len(caches), c.num_pages, c.page_size, c.num_kv_heads, c.head_dim, src.data_ptr(),
            dst.data_ptr(), src.shape[0], _abi.stream_of(src)), what)
    engaged("w4a8_mi355x.kv4_copy_pages")


def kv4_keep(caches: KV4Cache | Sequence[KV4Cache], page_table: torch.Tensor, cu_q: torch.Tensor, seq_lens: torch.Tensor,
             keep: torch.Tensor, kept: torch.Tensor) -> torch.Tensor:
    """Put the accepted ones of the new tokens behind the context, in each of the caches (layers of one shape), and return
    the sequences' lengths with them alone, (B,) int32. ``keep`` (B, width) int32: of sequence b's new tokens, in ascending
    order, the indices of its ``kept[b]`` accepted ones ((B,) int32, between 0 and what is there). page_table, cu_q and
    seq_lens are those that the tokens were appended with.

    An entry below its own place, or not of a new token, leaves its slot as it is. Slots behind the new length keep what
    they hold, and the next tokens are appended over them. One launch per 64 caches."""
    what = "kv4_keep"
    r = _host.load().kv4_keep(_tensors(caches), page_table, cu_q, seq_lens, keep, kept)
    if r is not None:
        engaged("w4a8_mi355x.kv4_keep")
        return r
    caches = _layers(caches, what)
    c = caches[0]
    table, ldt, width, cu, lens, B = _batch(c, page_table, cu_q, seq_lens, what)
    for name, t, dim in (("keep", keep, 2), ("kept", kept, 1)):
        if t.dtype != torch.int32 or t.dim() != dim or t.shape[0] != B:
            raise TypeError(f"{what}: {name} must be a {dim}-D int32 tensor of {B} rows, got {t.dtype} {tuple(t.shape)}")
        if t.device != c.device:
            raise RuntimeError(f"{what}: {name} is on {t.device}, the caches on {c.device}")
    keep, kept = keep.contiguous(), kept.contiguous()
    now = torch.empty((B,), dtype=torch.int32, device=c.device)
    arrays = _arrays(caches)
    with torch.cuda.device(c.device):
        _abi.check(_abi.load().w4a8_kv4_keep(
            ctypes.addressof(arrays), len(caches), c.num_pages, c.page_size, c.num_kv_heads, c.head_dim, table, ldt, width, cu,
            lens, B, keep.data_ptr(), keep.shape[1], keep.shape[1], kept.data_ptr(), now.data_ptr(), _abi.stream_of(now)), what)
    engaged("w4a8_mi355x.kv4_keep")
    return now


def kv4_attention(
    q: torch.Tensor,  # (T, num_qo_heads, head_dim), any strides between rows
    cache: KV4Cache,
    page_table: torch.Tensor,
    cu_q: torch.Tensor,
    seq_lens: torch.Tensor,
    *,
    max_q: int | None = None,
    max_kv: int | None = None,
    sm_scale: float | None = None,
    causal: bool = True,
    window: int = 0,
    out: torch.Tensor | None = None,
    return_lse: bool = False,
    tree: KV4Tree | None = None,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Attention of the new tokens over their sequences' cached keys and values (the new tokens' own
    among them: append first). (T, num_qo_heads, head_dim) in q's type; with return_lse also the natural
    logarithm of each softmax's sum, (T, num_qo_heads) f32.

    num_qo_heads is a multiple of the cache's heads. sm_scale defaults to head_dim ** -0.5; it is positive
    and below 65536, and scores are within f32's range, bf16 queries below 2^96, steps of cached keys below 2^100, of cached values
    below 2^64 (below 2^100 where none of the sequence's is below 2^-4: the small ones would weigh less). causal: a
    token sees the keys up to its own position; window > 0: only the last ``window`` of those. A row
    that sees no key is 0 (lse -inf). out, where given, may be strided; rows outside cu_q keep what they
    hold there, and are undefined in a fresh output. Rows of out that overlap are refused, and so is an out that
    overlaps q without being q.

    tree: the new tokens are drafted ones; a token sees the cached context before them and, of them, those that its
    row of ``tree.mask`` names (``causal`` says nothing then). window > 0 counts from ``tree.positions``, among cached
    tokens: of the new ones the mask alone decides. More than 64 queries that share a key (max_q times the heads of a
    group) have a kernel of their own where there is no window, heads have up to 128 channels and max_kv is 512 or more: products
    there are in fp16, errors before the output's rounding are up to four times as large, and bf16 models' values below 2^-29 of
    their sequence's largest count as 0.

    max_q and max_kv, the most new tokens and the greatest length of a sequence, are what the host
    plans the launch by (default: T rows, and the table's capacity): how it is split, and for trees the kernel, whose
    roundings differ. Too large a bound costs time, too low a one as well; neither changes which keys are read. One launch, and a second that joins the
    parts where the keys are split over workgroups."""
    what = "kv4_attention"
    if sm_scale is None:
        sm_scale = cache.head_dim ** -0.5
    if tree is None:
        r = _host.load().kv4_attention(cache.k, cache.v, cache.k_scale, cache.v_scale, page_table, cu_q, seq_lens, q, max_q,
                                       max_kv, sm_scale, causal, window, out, return_lse)
    else:
        r = _host.load().kv4_tree_attention(cache.k, cache.v, cache.k_scale, cache.v_scale, page_table, cu_q, seq_lens, q,
                                            max_q, max_kv, sm_scale, window, out, return_lse, tree.mask, tree.positions)
    if r is not None:
        engaged("w4a8_mi355x.kv4_attention")
        return r if return_lse else r[0]
    q = _rows(q, cache, None, "q", what)
    T, Hq, D = q.shape
    if Hq < cache.num_kv_heads or Hq % cache.num_kv_heads:
        raise ValueError(f"{what}: {Hq} query heads for {cache.num_kv_heads} key/value heads")
    table, ldt, width, cu, lens, B = _batch(cache, page_table, cu_q, seq_lens, what)
    if window < 0:
        raise ValueError(f"{what}: window={window}")
    mask = None
    if tree is not None:
        mask, pos = tree
        if mask.dtype != torch.int32 or mask.dim() != 2 or mask.shape[0] != T or not 1 <= mask.shape[1] <= _TREE_WORDS \
                or pos.dtype != torch.int32 or tuple(pos.shape) != (T,):
            raise TypeError(f"{what}: tree must be ({T}, 1 to {_TREE_WORDS}) int32 words and ({T},) int32 positions, got "
                            f"{mask.dtype} {tuple(mask.shape)} and {pos.dtype} {tuple(pos.shape)}")
        if mask.device != cache.device or pos.device != cache.device:
            raise RuntimeError(f"{what}: tree is on {mask.device} and {pos.device}, the cache on {cache.device}")
        mask, pos = mask.contiguous(), pos.contiguous()
    cap = width * cache.page_size
    max_q = T if max_q is None else min(int(max_q), T)
    max_kv = cap if max_kv is None else min(int(max_kv), cap)
    if max_q < 0 or max_kv < 0:
        raise ValueError(f"{what}: max_q={max_q}, max_kv={max_kv}")
    if out is None:
        out = torch.empty((T, Hq, D), dtype=q.dtype, device=q.device)
    elif tuple(out.shape) != (T, Hq, D) or out.dtype != q.dtype or out.device != q.device or not _rows_ok(out):
        raise ValueError(f"{what}: out must be ({T}, {Hq}, {D}) {q.dtype} with 16-byte aligned rows, got {out.dtype} "
                         f"{tuple(out.shape)} {tuple(out.stride())}")
    if window:  # a block of queries sees no more than this
        max_kv = min(max_kv, window + max_q)
    lse = torch.empty((T, Hq), dtype=torch.float32, device=q.device) if return_lse else None
    lib = _abi.load()
    if mask is None:
        ws_bytes = int(lib.w4a8_kv4_attention_workspace_bytes(T, Hq, cache.num_kv_heads, D, B, max_q, max_kv))
    else:
        ws_bytes = int(lib.w4a8_kv4_tree_attention_workspace_bytes(T, Hq, cache.num_kv_heads, D, B, window, max_q, max_kv))
    ws = torch.empty((ws_bytes,), dtype=torch.uint8, device=q.device) if ws_bytes > 0 else None
    before = (q.data_ptr(), _abi.dtype_code(q.dtype), q.stride(0), q.stride(1), T, Hq, cache.num_kv_heads, D, *cache._ptrs(),
              cache.num_pages, cache.page_size, table, ldt, width, cu, lens, B, float(sm_scale))
    after = (out.data_ptr(), out.stride(0), out.stride(1), _abi.ptr(lse), _abi.ptr(ws), max(ws_bytes, 0), _abi.stream_of(q))
    with torch.cuda.device(cache.device):
        if mask is None:
            rc = lib.w4a8_kv4_attention(*before, int(bool(causal)), int(window), max_q, max_kv, *after)
        else:
            rc = lib.w4a8_kv4_tree_attention(*before, int(window), max_q, max_kv, mask.data_ptr(), mask.shape[1], mask.shape[1],
                                             pos.data_ptr(), *after)
        _abi.check(rc, what)
    engaged("w4a8_mi355x.kv4_attention")
    return (out, lse) if return_lse else out
