"""Pages copied and accepted tokens moved in the 4-bit cache (quant/kv4.py kv4_copy_pages, kv4_keep): refusals on the CPU,
and on the GPU every byte of the caches against the documented layout."""
import random

import pytest
import torch

from conftest import pkg

DTYPES = [torch.bfloat16, torch.float16]
ARRAYS = ("k", "v", "k_scale", "v_scale")


def _kv4():
    return pkg("quant.kv4")


def filled(dev, pages, page, H, D, dtype, seed):
    """A cache of arbitrary bytes (scales any 16 bits, NaN among them)."""
    g = torch.Generator().manual_seed(seed)
    c = _kv4().KV4Cache(pages, page, H, D, dtype, dev)
    for n in ARRAYS:
        t = getattr(c, n)
        raw = torch.randint(0, 256, (t.numel() * t.element_size(),), generator=g, dtype=torch.uint8)
        t.copy_(raw.view(t.dtype).view(t.shape))
    return c


def raw(c):
    return [getattr(c, n).cpu().contiguous().view(torch.uint8).clone() for n in ARRAYS]


def tokens(c):
    """Each slot's codes and scales: K (pages, H, page, D/2), V (pages, H, page, D), scales as 32-bit words."""
    j = torch.arange(8, dtype=torch.int32) * 4
    v = ((c.v.cpu().unsqueeze(3) >> j.view(1, 1, 1, 8, 1)) & 15).flatten(2, 3)
    return [c.k.cpu().clone(), v, c.k_scale.cpu().view(torch.int32).squeeze(-1).clone(), c.v_scale.cpu().view(torch.int32).squeeze(-1).clone()]


# ------------------------------------------------------------------------------------------------
# CPU
# ------------------------------------------------------------------------------------------------
def test_refusals():
    kv4 = _kv4()
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32)  # noqa: E731
    c = kv4.KV4Cache(4, 16, 1, 64, device="cpu")
    for f in (lambda: kv4.kv4_copy_pages(c, i32(0), i32(1)), lambda: kv4.kv4_copy_pages([c], i32(0), i32(1)),
              lambda: kv4.kv4_keep(c, i32([0]).view(1, 1), i32(0, 1), i32(1), i32([0]).view(1, 1), i32(1))):
        with pytest.raises(RuntimeError, match="on the GPU"):
            f()
    with pytest.raises(ValueError, match="no cache"):
        kv4.kv4_copy_pages([], i32(0), i32(1))


def test_abi_refusals():
    if torch.cuda.is_available():
        pytest.skip("the pointers are not real")
    import ctypes

    lib = pkg("_abi").load()
    P = 1 << 20

    def arrays(*ptrs):
        a = (ctypes.c_void_p * len(ptrs))(*ptrs)
        return a, ctypes.addressof(a)

    good, at = arrays(P, P, P, P)
    twice, at2 = arrays(P, P, P, P, P, P, P, P)
    odd, at3 = arrays(P, P + 8, P, P)
    for a, code, what in (((at, -1, 4, 16, 1, 64, P, P, 1), 1, "caches"), ((at, 1, 4, 24, 1, 64, P, P, 1), 2, "power of two"),
                          ((at, 1, 4, 16, 1, 96, P, P, 1), 2, "64, 128 or 256"), ((at, 1, 4, 16, 1, 64, None, P, 1), 1, "src and dst"),
                          ((None, 1, 4, 16, 1, 64, P, P, 1), 1, "src and dst"), ((at2, 2, 4, 16, 1, 64, P, P, 1), 1, "twice"),
                          ((at3, 1, 4, 16, 1, 64, P, P, 1), 1, "16-byte"), ((at, 1, 4, 16, 1, 64, P, P, -1), 1, "pairs"),
                          ((at, 1, 4, 65536, 256, 256, P, P, 1 << 20), 2, "index ranges")):
        rc = lib.w4a8_kv4_copy_pages(*a, None)
        assert rc == code and what in lib.w4a8_last_error().decode(), (a, rc, lib.w4a8_last_error())
    assert lib.w4a8_kv4_copy_pages(at, 1, 4, 16, 1, 64, P, P, 0, None) == 0 and lib.w4a8_kv4_copy_pages(at, 0, 4, 16, 1, 64, P, P, 1, None) == 0

    def keep(at=at, caches=1, D=64, width=4, ldt=4, B=2, keep=P, ldk=3, most=3, kept=P, now=4 * P):
        rc = lib.w4a8_kv4_keep(at, caches, 4, 16, 1, D, P, ldt, width, P, 2 * P, B, keep, ldk, most, kept, now, None)
        return rc, lib.w4a8_last_error().decode()

    for kw, code, what in ((dict(caches=0), 1, "caches"), (dict(D=32), 2, "64, 128 or 256"), (dict(kept=None), 1, "kept"),
                           (dict(keep=None), 1, "keep"), (dict(ldk=2), 1, "keep"), (dict(ldt=3), 1, "stride"), (dict(at=at2, caches=2), 1, "twice"),
                           (dict(now=2 * P + 4), 1, "overlaps seq_lens"), (dict(B=65536), 2, "index ranges")):
        rc, msg = keep(**kw)
        assert rc == code and what in msg, (kw, rc, msg)
    assert keep(B=0)[0] == 0
    del good, twice, odd


# ------------------------------------------------------------------------------------------------
# GPU: pages
# ------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page,H,D,layers", [(16, 8, 128, 3), (64, 1, 64, 1), (16, 1, 256, 2), (512, 2, 128, 1), (16, 1, 64, 70)])
def test_copy_pages(dev, dtype, page, H, D, layers):
    pages = 23
    caches = [filled(dev, pages, page, H, D, dtype, seed) for seed in range(layers)]
    before = [raw(c) for c in caches]
    src = torch.tensor([3, 3, 9, -1, 4, 22, 7, 23, 5, 2 ** 31 - 1, 8], dtype=torch.int32)
    dst = torch.tensor([0, 1, 21, 2, 23, 20, 7, 6, -2 ** 31, 10, 11], dtype=torch.int32)
    _kv4().kv4_copy_pages(caches[0] if layers == 1 else caches, src.to(dev), dst.to(dev))
    for c, was in zip(caches, before):
        for got, t in zip(raw(c), was):
            for a, b in ((3, 0), (3, 1), (9, 21), (22, 20), (8, 11)):
                t[b] = t[a]
            assert torch.equal(got, t)


@pytest.mark.gpu
def test_copy_pages_refusals_and_capture(dev):
    kv4 = _kv4()
    c, o = filled(dev, 8, 16, 2, 64, torch.bfloat16, 1), filled(dev, 8, 16, 2, 64, torch.bfloat16, 2)
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    for args, e in ((([c, c], i32(0), i32(1)), ValueError), (([c, filled(dev, 9, 16, 2, 64, torch.bfloat16, 1)], i32(0), i32(1)), ValueError),
                    (([c, filled(dev, 8, 16, 2, 64, torch.float16, 1)], i32(0), i32(1)), ValueError), ((c, i32(0).long(), i32(1)), TypeError),
                    ((c, i32(0, 1), i32(1)), ValueError), ((c, i32(0).cpu(), i32(1)), RuntimeError), (([], i32(0), i32(1)), ValueError),
                    ((c, i32([0], [1]), i32(1, 2)), TypeError)):
        with pytest.raises(e):
            kv4.kv4_copy_pages(*args)
    was = raw(c)
    kv4.kv4_copy_pages(c, i32()[:0], i32()[:0])
    assert all(torch.equal(a, b) for a, b in zip(raw(c), was))
    both = i32(0, 5, 1, 6, 2, 7)
    kv4.kv4_copy_pages([c, o], both[::2], both[1::2])  # strided lists
    assert torch.equal(c.k[5:], c.k[:3]) and torch.equal(o.v[5:], o.v[:3])
    src, dst = i32(0, 0), i32(6, 7)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kv4.kv4_copy_pages([c, o], src, dst)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv4.kv4_copy_pages([c, o], src, dst)
    for rep, (a, b) in enumerate((((1, 2), (7, 6)), ((3, 3), (4, 5)), ((-1, 2), (0, 1)))):
        src.copy_(i32(*a))
        dst.copy_(i32(*b))
        want = [raw(x) for x in (c, o)]
        graph.replay()
        torch.cuda.synchronize()
        for x, ts in zip((c, o), want):
            for t, got in zip(ts, raw(x)):
                for p, r in zip(a, b):
                    if p >= 0:
                        t[r] = t[p]
                assert torch.equal(got, t), rep


@pytest.mark.gpu
def test_pages_past_4_gib(dev):
    """Pages of 256 KB of codes, numbers up to 17000: bytes past 2^32."""
    c = _kv4().KV4Cache(17000, 4096, 1, 128, torch.bfloat16, dev)
    c.k[16998], c.v[16998], c.k_scale[16998], c.v_scale[16998] = 7, 9, 2.0, 3.0
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    _kv4().kv4_copy_pages(c, i32(16998, 16998), i32(16999, 0))
    for t, x in ((c.k, 7), (c.v, 9), (c.k_scale, 2.0), (c.v_scale, 3.0)):
        assert (t[16999] == x).all() and (t[0] == x).all() and not t[1:16998:500].any()
    # one token accepted there
    table = i32(16999).view(1, 1)
    c.k[16999, :, 5], c.k_scale[16999, :, 5] = 3, 5.0
    now = _kv4().kv4_keep(c, table, i32(0, 4), i32(6), i32([3]).view(1, 1), i32(1))
    assert now.tolist() == [3] and (c.k[16999, :, 2] == 3).all() and (c.k_scale[16999, :, 2] == 5).all()
    assert (c.k[16999, :, 3] == 7).all() and not c.k[1:16998:500].any()


# ------------------------------------------------------------------------------------------------
# GPU: accepted tokens
# ------------------------------------------------------------------------------------------------
def emulate(parts, table, page, lens, news, keep, kept):
    """The moves on each slot's codes and scales, as if all were read before the first is written."""
    was = [t.clone() for t in parts]

    def place(b, pos):
        if pos < 0 or pos // page >= table.shape[1]:
            return None
        p = table[b, pos // page].item()
        return (p, pos % page) if 0 <= p < parts[0].shape[0] else None

    for b, (n, new) in enumerate(zip(lens, news)):
        m = min(max(kept[b], 0), new, len(keep[b]))
        for j in range(m):
            i = keep[b][j]
            if not j < i < new:
                continue
            src, dst = place(b, n - new + i), place(b, n - new + j)
            if src and dst:
                for t, w in zip(parts, was):
                    t[dst[0], :, dst[1]] = w[src[0], :, src[1]]
    return parts


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page,H,D,layers", [(16, 8, 128, 2), (32, 1, 64, 1), (16, 2, 256, 1), (16, 1, 64, 67)])
@pytest.mark.parametrize("news", [[5, 1, 0, 13, 8], [64, 17, 33, 3, 100]])
def test_keep(dev, dtype, page, H, D, layers, news):
    rng = random.Random(layers + sum(news))
    lens = [n + rng.randrange(0, 40) for n in news]
    lens[0], lens[1] = news[0] + 19, news[1]  # a block that begins among old tokens, and no context
    count = [-(-max(n, 1) // page) for n in lens]
    pages = sum(count) + 2
    perm = random.Random(1).sample(range(pages), pages)
    table = torch.full((len(lens), max(count)), -1, dtype=torch.int32)
    at = 0
    for b, k in enumerate(count):
        table[b, :k] = torch.tensor(perm[at:at + k])
        at += k
    width = 24
    keep = [sorted(rng.sample(range(n), min(n, rng.randrange(0, width + 1)))) for n in news]
    kept = [len(k) for k in keep]
    keep = [k + [2 ** 30] * (width - len(k)) for k in keep]  # nothing is read there
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    cu = [2 + sum(news[:i]) for i in range(len(news) + 1)]
    for variant in range(3):
        if variant == 1:  # not ascending, twice the same, below its place, negative, past the tokens; more and fewer than there are
            keep = [[rng.randrange(-2, n + 4) for _ in range(width)] for n in news]
            kept = [width + 5, -3, 9, width, 2]
        elif variant == 2:  # a page that does not exist, a table that ends too early
            table = table[:, :max(1, table.shape[1] - 1)].contiguous()
            table[3, 0] = pages
        caches = [filled(dev, pages, page, H, D, dtype, seed) for seed in range(layers)]
        parts = [tokens(c) for c in caches]
        now = _kv4().kv4_keep(caches if layers > 1 else caches[0], table.to(dev), i32(cu), i32(lens), i32(keep), i32(kept))
        assert now.tolist() == [n - w + min(max(m, 0), w, width) for n, w, m in zip(lens, news, kept)]
        for c, was in zip(caches, parts):
            for got, want in zip(tokens(c), emulate(was, table, page, lens, news, keep, kept)):
                assert torch.equal(got, want), variant


@pytest.mark.gpu
def test_keep_refusals_empty_and_capture(dev):
    kv4 = _kv4()
    c = filled(dev, 8, 16, 2, 64, torch.bfloat16, 1)
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    table, cu, lens, keep, kept = i32([0, 1], [2, 3]), i32(0, 3, 6), i32(20, 10), i32([0, 2], [1, 2]), i32(2, 2)
    for kw, e in ((dict(keep=keep.long()), TypeError), (dict(keep=keep[:1]), TypeError), (dict(kept=kept[:1]), TypeError),
                  (dict(kept=kept.cpu()), RuntimeError), (dict(cu=cu[:2]), ValueError), (dict(table=table.long()), TypeError),
                  (dict(caches=[c, c]), ValueError)):
        a = dict(caches=c, table=table, cu=cu, lens=lens, keep=keep, kept=kept)
        a.update(kw)
        with pytest.raises(e):
            kv4.kv4_keep(*a.values())
    was = tokens(c)
    assert kv4.kv4_keep(c, table[:0], cu[:1], lens[:0], keep[:0], kept[:0]).shape == (0,)
    assert kv4.kv4_keep(c, table, cu, lens, keep[:, :0], kept).tolist() == [17, 7]
    assert all(torch.equal(a, b) for a, b in zip(tokens(c), was))
    strided = torch.stack([keep, keep], -1)[..., 0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kv4.kv4_keep(c, table, cu, lens, strided, kept * 0)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        now = kv4.kv4_keep(c, table, cu, lens, keep, kept)
    for rep, (n, k, m) in enumerate((((20, 10), ([0, 2], [1, 2]), (2, 2)), ((19, 3), ([1, 2], [2, 0]), (2, 1)), ((32, 32), ([2, 2], [0, 1]), (0, 2)))):
        lens.copy_(i32(*n))
        keep.copy_(i32(*k))
        kept.copy_(i32(*m))
        want = emulate(tokens(c), table.cpu(), 16, n, (3, 3), k, m)
        graph.replay()
        torch.cuda.synchronize()
        assert now.tolist() == [a - 3 + b for a, b in zip(n, m)]
        assert all(torch.equal(a, b) for a, b in zip(tokens(c), want)), rep
