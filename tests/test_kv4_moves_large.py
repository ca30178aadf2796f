"""What moves in the 4-bit cache (kv4_read, kv4_copy_pages, kv4_keep) at the sizes that take another way: several heads a wave,
writes past the caches, more than 64 accepted tokens."""
import random

import pytest
import torch

from test_kv4_moves import ARRAYS, DTYPES, _kv4, emulate, filled, tokens


def scaled(dev, pages, page, H, D, dtype, seed):
    """A cache of arbitrary codes and finite scales."""
    g = torch.Generator(device=dev).manual_seed(seed)
    c = _kv4().KV4Cache(pages, page, H, D, dtype, dev)
    c.k.random_(0, 256, generator=g)
    c.v.random_(-2 ** 31, 2 ** 31 - 1, generator=g)
    c.k_scale.normal_(generator=g)
    c.v_scale.normal_(generator=g)
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,H,page,T", [(128, 5, 64, 66003), (64, 7, 16, 80003), (256, 3, 32, 90005), (128, 1, 16, 70001), (64, 5, 128, 1700),
                                          (128, 5, 64, 140003), (64, 7, 32, 190001), (256, 3, 16, 120005)])
def test_many_rows_are_read_as_few(dev, dtype, D, H, page, T):
    """The bits of the same rows read a few hundred at a time, each head's own; rows without a page are NaN."""
    lens = [T * 3 // 5, 1, T - T * 3 // 5 - 1]
    count = [-(-n // page) for n in lens]
    c = scaled(dev, sum(count) + 2, page, H, D, dtype, H)
    perm = torch.randperm(c.num_pages, generator=torch.Generator().manual_seed(1)).int()
    table = torch.full((3, max(count)), -1, dtype=torch.int32)
    at = 0
    for b, k in enumerate(count):
        table[b, :k] = perm[at:at + k]
        at += k
    table[0, 3] = -1
    table = table.to(dev)
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    cu, seq = i32(0, lens[0], lens[0] + 1, T), i32(*lens)
    got = _kv4().kv4_read(c, table, cu, seq, T)
    few = 8192 // H - 5
    row = 0
    for b, n in enumerate(lens):
        for i in range(0, n, few):
            m = min(few, n - i)
            want = _kv4().kv4_read(c, table[b:b + 1], i32(0, m), i32(i + m), m)
            for a, w in zip(got, want):
                assert torch.equal(a[row + i:row + i + m].view(torch.int16), w.view(torch.int16)), (b, i)
        row += n
    assert torch.isnan(got[0][3 * page:4 * page]).all() and torch.isfinite(got[1][4 * page:4 * page + 100].float()).all()
    # against the layout, a row here and there
    j = torch.arange(8, device=dev, dtype=torch.int32) * 4
    for r in range(5, lens[0], max(1, lens[0] // 97)):
        p, slot = int(table[0, r // page]), r % page
        if p < 0:
            continue
        codes = torch.stack([c.k[p, :, slot] & 15, c.k[p, :, slot] >> 4], -1).flatten(-2).double()
        ks, vs = c.k_scale[p, :, slot].double(), c.v_scale[p, :, slot].double()
        assert torch.equal(got[0][r], (codes * ks[:, :1] + ks[:, 1:]).float().to(dtype))
        codes = ((c.v[p, :, slot // 8] >> j[slot % 8]) & 15).double()
        assert torch.equal(got[1][r], (codes * vs[:, :1] + vs[:, 1:]).float().to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("D,H,most", [(128, 1, 3), (64, 3, 2), (256, 2, 12), (128, 20, 5)])
def test_rows_of_many_sequences(dev, D, H, most):
    """Rows next to each other of different sequences, with more than 64 empty ones between two, rows before and behind all; the
    bits of each sequence read alone."""
    rng = random.Random(most)
    news = [0] * 3 + [rng.choice((0, 1, rng.randrange(0, most))) for _ in range(900)] + [1] + [0] * 64 + [2] + [0] * 150 + [1, 1] + [0] * 70
    page, B = 16, len(news)
    lens = [n + rng.randrange(0, 20) if n else 5 for n in news]
    width = -(-max(lens) // page)
    c = scaled(dev, 300, page, H, D, torch.bfloat16, H)
    table = torch.randint(0, 300, (B, width), generator=torch.Generator().manual_seed(1), dtype=torch.int32).to(dev)
    cu = [3 + sum(news[:i]) for i in range(B + 1)]
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    T = cu[-1] + 4
    got = _kv4().kv4_read(c, table, i32(*cu), i32(*lens), T)
    for b, n in enumerate(news):
        if n:
            want = _kv4().kv4_read(c, table[b:b + 1], i32(0, n), i32(lens[b]), n)
            for a, w in zip(got, want):
                assert torch.equal(a[cu[b]:cu[b + 1]].view(torch.int16), w.view(torch.int16)), b


@pytest.mark.gpu
@pytest.mark.parametrize("page,H,D,layers,n", [(64, 8, 128, 3, 230), (16, 5, 64, 70, 161), (128, 3, 256, 1, 400), (64, 8, 128, 3, 701), (16, 5, 64, 70, 461),
                                                    (128, 3, 256, 1, 1501)])
def test_many_pages(dev, page, H, D, layers, n):
    """More bytes than the caches hold, to the last of them."""
    pages = 2 * n + 3
    caches = [scaled(dev, pages, page, H, D, torch.bfloat16, i) for i in range(layers)]
    assert 2 * n * layers * H * page * (D + 8) > 32 << 20
    before = [[getattr(c, a).clone() for a in ARRAYS] for c in caches]
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(2)).int()
    src, dst = perm[:n].clone(), perm[n:2 * n].clone()
    src[5], dst[7], src[9] = -1, pages, dst[9]
    _kv4().kv4_copy_pages(caches if layers > 1 else caches[0], src.to(dev), dst.to(dev))
    ok = [i for i in range(n) if i not in (5, 7, 9)]
    for c, was in zip(caches, before):
        for a, t in zip(ARRAYS, was):
            t[dst[ok].long().to(dev)] = t[src[ok].long().to(dev)]
            assert torch.equal(getattr(c, a).view(torch.uint8), t.view(torch.uint8)), a


@pytest.mark.gpu
@pytest.mark.parametrize("page,H,D", [(16, 3, 128), (64, 1, 64), (32, 2, 256)])
@pytest.mark.parametrize("off", [0, 5])
def test_many_accepted_tokens(dev, page, H, D, off):
    """More than the 64 slots that are looked up at once, from the first slot of a block and from a later one."""
    rng = random.Random(page + off)
    news, most = [400, 400, 77, 130], [65, 300, 64, 130]
    lens = [n + 24 + off for n in news]
    count = [-(-n // page) for n in lens]
    pages = sum(count) + 1
    perm = rng.sample(range(pages), pages)
    table = torch.full((4, max(count)), -1, dtype=torch.int32)
    at = 0
    for b, k in enumerate(count):
        table[b, :k] = torch.tensor(perm[at:at + k])
        at += k
    width = 310
    keep = [sorted(rng.sample(range(n), m)) + [0] * (width - m) for n, m in zip(news, most)]
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    cu = [sum(news[:i]) for i in range(5)]
    c = filled(dev, pages, page, H, D, torch.bfloat16, 5)
    was = tokens(c)
    now = _kv4().kv4_keep(c, table.to(dev), i32(cu), i32(lens), i32(keep), i32(most))
    assert now.tolist() == [n - w + m for n, w, m in zip(lens, news, most)]
    for got, want in zip(tokens(c), emulate(was, table, page, lens, news, keep, most)):
        assert torch.equal(got, want)
