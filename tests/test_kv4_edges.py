"""The 4-bit cache and its attention (quant/kv4.py) at the edges of what a call may hold: windows past the table, scales
that reach f32's end, one row of any stride, outputs on top of inputs, lengths near 2^31, and errors that keep their text."""
import math

import pytest
import torch

from conftest import pkg
from test_kv4 import DTYPES, Setup, _kv4


# ------------------------------------------------------------------------------------------------
# GPU
# ------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_window_past_the_table_is_nan(dev, dtype, causal):
    """A sequence longer than its table: a row whose window begins past the table's end sees missing tokens alone, and is
    NaN as a row is that sees some of them. In decode, over several rows, with the tokens split and not."""
    page = 16
    for width, past, news, window, kw in ((1, 24, 1, 8, {"max_q": 1}), (1, 24, 30, 8, {}), (1, 24, 39, 1, {}), (3, 1, 20, 8, {}),
                                          (256, 4000, 1, 3000, {"max_q": 1}), (256, 4000, 1, 3000, {"max_q": 1, "max_kv": 1}),
                                          (256, 4000, 40, 3000, {"max_q": 40}), (256, 600, 1200, 500, {})):
        cap = width * page
        s = Setup(dev, dtype, 64, 1, page, [cap], [1], seed=width)
        n = cap + past
        seq = torch.tensor([n], dtype=torch.int32, device=dev)
        cu = torch.tensor([0, news], dtype=torch.int32, device=dev)
        q = torch.randn(news, 2, 64, generator=torch.Generator().manual_seed(1)).to(dtype).to(dev)
        out, lse = _kv4().kv4_attention(q, s.cache, s.d_table, cu, seq, window=window, causal=causal, return_lse=True, **kw)
        # row i is at position n - news + i; not causal, it sees up to the sequence's end
        missing = torch.arange(n - news, n) >= cap if causal else torch.ones(news, dtype=torch.bool)
        where = (width, past, news, window, kw)
        assert torch.equal(torch.isnan(out).all(-1).all(-1).cpu(), missing), where
        assert torch.equal(torch.isnan(out).any(-1).any(-1).cpu(), missing), where
        assert torch.equal(torch.isnan(lse).all(-1).cpu(), missing) and torch.isfinite(lse.cpu()[~missing]).all(), where


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sm_scale", [1e-3, 1e-12, 1e-30])
def test_small_queries_and_scales(dev, dtype, sm_scale):
    """Queries of zeros (padding) and of the type's smallest numbers with scales far below 1: all scores are zero, or as
    good as zero, and the output is the mean of the values that a row sees."""
    s = Setup(dev, dtype, 64, 1, 16, [70, 300], [1, 66], seed=31)
    fi = torch.finfo(dtype)
    for q in (torch.zeros(67, 2, 64), torch.full((67, 2, 64), fi.smallest_normal), torch.full((67, 2, 64), fi.smallest_normal * fi.eps)):
        for kw in ({}, {"max_q": 66}, {"max_q": 1, "max_kv": 300}):
            s.check(q.to(dtype), f"queries of {q[0, 0, 0]}, {kw}", sm_scale=sm_scale, **kw)
            s.check(q.to(dtype), f"queries of {q[0, 0, 0]}, window, {kw}", window=3, sm_scale=sm_scale, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("sm_scale", [1e-3, 0.125])
def test_slots_nobody_wrote_count_as_keys(dev, sm_scale):
    """A fresh cache holds vectors of zeros with steps of zero: the output is 0, and a row's sum is its keys' number."""
    kv4 = _kv4()
    cache = kv4.KV4Cache(8, 16, 1, 64, device=dev)
    table = torch.arange(7, dtype=torch.int32, device=dev).view(1, 7)
    n, new = 100, 66
    cu, seq = torch.tensor([0, new], dtype=torch.int32, device=dev), torch.tensor([n], dtype=torch.int32, device=dev)
    seen = torch.arange(n - new + 1, n + 1).double()
    for q in (torch.zeros(new, 1, 64, dtype=torch.bfloat16, device=dev), torch.ones(new, 1, 64, dtype=torch.bfloat16, device=dev)):
        for window in (0, 1, 5):
            for kw in ({}, {"max_q": 1}):
                out, lse = kv4.kv4_attention(q, cache, table, cu, seq, sm_scale=sm_scale, window=window, return_lse=True, **kw)
                want = torch.log(seen.clamp_max(window) if window else seen)
                assert (out == 0).all()
                # The sum is held as 2^46 of it, a power that follows from the steps: lse is log(2^46 n) - 46 log 2 in f32, terms
                # below 37 and 32, the logarithm off by up to a last place (2^-23), the product by half of one, the
                # difference of numbers below 5 by half of one again: 37 / 2^23 + 32 / 2^24 + 5 / 2^24 = 6.7e-6.
                assert ((lse.flatten().cpu().double() - want).abs() <= 6.7e-6).all(), (window, kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_any_strides_and_alignment(dev, dtype):
    """k, v and q whose rows the kernels do not take as they are: contiguous but not 16-byte aligned, and one row of a
    wider buffer whose stride is no multiple of 8."""
    kv4 = _kv4()
    H, G, D, page, n = 2, 4, 64, 16, 21
    want = Setup(dev, dtype, D, H, page, [n], [n], seed=41)
    q = want.q(H * G)
    ref = want.attend(q)

    def shifted(t):
        buf = torch.empty(t.numel() + 8, dtype=dtype, device=dev)
        view = buf[1:1 + t.numel()].view(t.shape)
        view.copy_(t)
        assert view.is_contiguous() and view.data_ptr() % 16
        return view

    cu_all = torch.tensor([0, n], dtype=torch.int32, device=dev)

    def same(cache):
        for a, b in zip((cache.k, cache.v, cache.k_scale, cache.v_scale),
                        (want.cache.k, want.cache.v, want.cache.k_scale, want.cache.v_scale)):
            ids = want.table[0].long().to(dev)
            tokens = 2 if a.dtype == torch.int32 else n  # whole blocks of V; the last one's other tokens hold anything
            assert torch.equal(a[ids].transpose(1, 2).flatten(0, 1)[:tokens].contiguous().view(torch.uint8),
                               b[ids].transpose(1, 2).flatten(0, 1)[:tokens].contiguous().view(torch.uint8))

    cache = kv4.KV4Cache(want.cache.num_pages, page, H, D, dtype, dev)
    kv4.kv4_append(cache, shifted(want.k), shifted(want.v), want.d_table, cu_all, want.d_seq)
    same(cache)
    assert torch.equal(kv4.kv4_attention(shifted(q), want.cache, want.d_table, want.d_cu, want.d_seq), ref)
    # a decode step of one row at a time, out of a buffer of odd width
    cache = kv4.KV4Cache(want.cache.num_pages, page, H, D, dtype, dev)
    wide = torch.zeros(1, H * D + 4, dtype=dtype, device=dev)
    qwide = torch.zeros(1, H * G * D + 4, dtype=dtype, device=dev)
    cu = torch.tensor([0, 1], dtype=torch.int32, device=dev)
    for i in range(n):
        wide[:, :H * D].copy_(want.k[i].view(1, -1))
        row = wide.as_strided((1, H, D), (H * D + 4, D, 1))
        assert row.stride(0) % 8
        v = want.v[i:i + 1].to(dev)
        seq = torch.tensor([i + 1], dtype=torch.int32, device=dev)
        kv4.kv4_append(cache, row, v, want.d_table, cu, seq)
        qwide[:, :H * G * D].copy_(q[i].view(1, -1))
        out = torch.full_like(qwide, 3.0)
        view, qrow = (t.as_strided((1, H * G, D), (H * G * D + 4, D, 1)) for t in (out, qwide))
        got = kv4.kv4_attention(qrow, cache, want.d_table, cu, seq, max_q=1, out=view)
        assert got.data_ptr() == view.data_ptr() and (out[:, H * G * D:] == 3).all()
        plain = kv4.kv4_attention(q[i:i + 1].to(dev), want.cache, want.d_table, cu, seq, max_q=1)
        assert torch.equal(got, plain)
    same(cache)
    # one head: the stride between heads does not matter
    one = Setup(dev, dtype, D, 1, page, [n], [n], seed=42)
    qd = one.q(1).to(dev)
    odd = torch.as_strided(qd, (n, 1, D), (D, 3, 1))
    assert torch.equal(one.attend(odd), one.attend(qd))


def test_one_row_of_any_stride_passes_the_abi():
    """Host checks of the C entry points, with pointers that are never read: a stride between rows or heads that there is
    only one of is not looked at; what passes them ends at the workspace."""
    lib = pkg("_abi").load()
    P = 1 << 20

    def attend(T, Hq, ldq, hq, ldo, ho):
        rc = lib.w4a8_kv4_attention(P, 0, ldq, hq, T, Hq, 1, 128, P, P, P, P, 16, 16, P, 1 << 12, 1 << 12, P, P, 1, 1.0, 1, 0, 1,
                                    1 << 16, P, ldo, ho, None, None, 0, None)
        assert rc == 1
        return lib.w4a8_last_error()

    assert b"workspace" in attend(1, 4, 516, 128, 516, 128) and b"workspace" in attend(4, 1, 128, 3, 128, 5)
    assert b"multiples of 8" in attend(2, 4, 516, 128, 512, 128) and b"multiples of 8" in attend(1, 4, 512, 124, 512, 128)
    assert b"multiples of 8" in attend(2, 4, 512, 128, 516, 128)


def test_abi_refuses_an_output_on_top_of_its_queries():
    """Host checks of the C entry point: what passes them ends at the launch, for which there is no GPU."""
    if torch.cuda.is_available():
        pytest.skip("the pointers are not real")
    lib = pkg("_abi").load()
    P = 1 << 24

    def attend(q, out, T=4, Hq=4, ld=512, h=128, ldo=None, ho=None):
        rc = lib.w4a8_kv4_attention(P + 2 * q, 0, ld, h, T, Hq, 1, 128, P, P, P, P, 16, 16, P, 1 << 12, 1 << 12, P, P, 1, 1.0, 1, 0, 1,
                                    64, P + 2 * out, ldo or ld, ho or h, None, P, 1 << 30, None)
        return rc, lib.w4a8_last_error()

    for kw in (dict(q=0, out=512), dict(q=512, out=0), dict(q=0, out=128), dict(q=0, out=8), dict(q=0, out=0, ldo=1024), dict(q=0, out=0, ho=256, ldo=1024),
               dict(q=0, out=256, ld=1024, h=128), dict(q=0, out=64, ld=2048, h=256), dict(q=0, out=128, ld=128, h=512),
               dict(q=0, out=8, T=1), dict(q=0, out=8, Hq=1), dict(q=0, out=0, ld=128, h=512, ldo=512, ho=128)):
        rc, text = attend(**kw)
        assert rc == 1 and b"overlaps q" in text, kw
    for kw in (dict(q=0, out=0), dict(q=0, out=2048), dict(q=2048, out=0), dict(q=0, out=512, ld=1024), dict(q=512, out=0, ld=1024),
               dict(q=0, out=128, ld=2048, h=256), dict(q=128, out=0, ld=1024, h=256), dict(q=0, out=512, ld=128, h=1024), dict(q=0, out=512, T=1),
               dict(q=0, out=128, Hq=1, ld=256), dict(q=0, out=0, ld=128, h=512), dict(q=0, out=0, T=1, ldo=4096)):
        rc, text = attend(**kw)
        assert rc == 3 and b"launch failed" in text, kw


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_outputs_beside_and_on_top_of_q(dev, dtype):
    """In place of the queries, and in other columns of their buffer: the bits of a fresh output. Shifted: refused."""
    kv4 = _kv4()
    for lens, news, kw in (([40, 333, 5], [1, 1, 1], {"max_q": 1}), ([40, 333], [33, 70], {}), ([3000], [1], {"max_q": 1}), ([3000], [300], {})):
        s = Setup(dev, dtype, 128, 2, 16, lens, news, seed=51)
        T = sum(news)
        wide = torch.randn(T + 1, 32, 128, generator=torch.Generator().manual_seed(1)).to(dtype).to(dev)
        args = s.cache, s.d_table, s.d_cu, s.d_seq
        for cut in ((slice(0, 8), slice(8, 16)), (slice(0, 16, 2), slice(1, 16, 2))):
            buf = wide.clone()
            q = buf[:T, cut[0]]
            want = kv4.kv4_attention(q, *args, **kw)
            kv4.kv4_attention(q, *args, out=buf[:T, cut[1]], **kw)
            assert torch.equal(buf[:T, cut[1]], want) and torch.equal(q, wide[:T, cut[0]]) and torch.equal(buf[:, 16:], wide[:, 16:])
            assert kv4.kv4_attention(q, *args, out=q, **kw).data_ptr() == q.data_ptr() and torch.equal(q, want)
        q = buf[:T, :8]
        for out in (buf[:T, 4:12], buf[1:, :8]) if T > 1 else (buf[:T, 4:12],):
            with pytest.raises(RuntimeError, match="overlaps q"):
                kv4.kv4_attention(q, *args, out=out, **kw)


@pytest.mark.gpu
def test_lengths_below_zero_see_nothing(dev):
    """Lengths of a padded batch that hold anything below zero: rows of 0, lse -inf, nothing appended."""
    kv4 = _kv4()
    s = Setup(dev, torch.bfloat16, 64, 1, 16, [40], [1], seed=61)
    news = [3, 1, 40, 2]
    seq = torch.tensor([-2 ** 31, -2 ** 31 + 2, -1, -2 ** 31 + 1], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 3, 4, 44, 46], dtype=torch.int32, device=dev)
    table = s.d_table.expand(4, -1).contiguous()
    q = torch.randn(sum(news), 2, 64, device=dev).bfloat16()
    before = [t.clone() for t in (s.cache.k, s.cache.v)]
    kv4.kv4_append(s.cache, q[:, :1], q[:, :1], table, cu, seq)
    torch.cuda.synchronize()
    assert torch.equal(before[0], s.cache.k) and torch.equal(before[1], s.cache.v)
    for kw in (dict(window=2), dict(), dict(max_q=1, window=5), dict(max_q=1), dict(causal=False, window=1), dict(causal=False)):
        out, lse = kv4.kv4_attention(q, s.cache, table, cu, seq, return_lse=True, **kw)
        torch.cuda.synchronize()
        assert (out == 0).all() and (lse == -math.inf).all(), kw


def test_tables_that_reach_2_31_tokens_are_refused():
    """A sequence's last tile has to end below 2^31 tokens."""
    if torch.cuda.is_available():
        pytest.skip("the pointers are not real")
    lib = pkg("_abi").load()
    P = 1 << 24

    def attend(page, width):
        rc = lib.w4a8_kv4_attention(P, 0, 128, 128, 1, 1, 1, 128, P, P, P, P, 16, page, P, width, width, P, P, 1, 1.0, 1, 0, 1, 64,
                                    P + 4096, 128, 128, None, P, 1 << 30, None)
        return rc, lib.w4a8_last_error()

    for page in (16, 32, 65536):
        most = (2 ** 31 - 1 - 32) // page
        rc, text = attend(page, most + 1)
        assert rc == 2 and b"past its index ranges" in text, (page, text)
        rc, text = attend(page, most)
        assert rc == 3 and b"launch failed" in text, (page, text)


@pytest.mark.gpu
def test_pages_past_4_gib(dev):
    """A cache whose codes pass 4 GiB, its first, middle and last pages in use: every bit of a small cache's results."""
    kv4 = _kv4()
    D, page, lens, news = 64, 16, [150, 33, 16], [20, 33, 1]
    s = Setup(dev, torch.bfloat16, D, 1, page, lens, news, seed=71)
    pages = (1 << 32) // (page * D // 2) + 50
    big = kv4.KV4Cache(pages, page, 1, D, device=dev)
    assert big.k.numel() > 1 << 32
    used = sum(-(-n // page) for n in lens)
    g = torch.Generator().manual_seed(3)
    ids = torch.cat([torch.arange(5), pages // 2 + torch.arange(4), torch.arange(pages - 11, pages)])
    ids = ids[torch.randperm(len(ids), generator=g)][:used].int()
    table, at = torch.full_like(s.table, -1), 0
    for b, n in enumerate(lens):
        c = -(-n // page)
        table[b, :c] = ids[at:at + c]
        at += c
    args = table.to(dev), s.cu_all.to(dev), s.d_seq
    kv4.kv4_append(big, s.k.to(dev), s.v.to(dev), *args)
    for got, want in zip(kv4.kv4_read(big, *args, sum(lens)), kv4.kv4_read(s.cache, s.d_table, *args[1:], sum(lens))):
        assert torch.equal(got, want)
    q = s.q(4)
    for kw in ({}, {"max_q": 1}, {"window": 9}):
        assert torch.equal(kv4.kv4_attention(q.to(dev), big, table.to(dev), s.d_cu, s.d_seq, **kw), s.attend(q, **kw))
    # nothing beside the pages in use was written
    for t in (big.k, big.v, big.k_scale, big.v_scale):
        t.index_fill_(0, ids.long().to(dev), 0)
        assert t.view(-1).view(torch.int64).max() == 0 and t.view(-1).view(torch.int64).min() == 0
