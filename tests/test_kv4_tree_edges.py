"""Trees of drafted tokens over the 4-bit cache at the edges of what a call may hold: queries, keys and steps whose powers of
two leave f32's range, keys of all sizes side by side, maxima that one tile's units cannot hold, sequences longer than their
table under a window, values at fp16's ends. References and tolerances are test_kv4_tree's."""
import math
import random

import pytest
import torch

from test_kv4_tree import DTYPES, Setup, _kv4, cache_values, check, lines, pack, random_tree, ref


def again(s):
    """The cache of s's keys and values as they are now."""
    _kv4().kv4_append(s.cache, s.k.to(s.dev), s.v.to(s.dev), s.d_table, s.cu_all.to(s.dev), s.d_seq)


def mask_tree(see, positions, dev, words=4):
    return _kv4().KV4Tree(pack(see, words).to(dev), torch.tensor(positions, dtype=torch.int32, device=dev))


# ------------------------------------------------------------------------------------------------
# GPU: more than 64 columns
# ------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,G", [(128, 4), (64, 2)])
def test_small_queries_over_small_keys(dev, dtype, D, G):
    """Queries and keys of zeros (a warm-up) and of the smallest numbers: all scores are zero, or as good as zero, and the
    output is the mean of the values that a row sees, masked ones not among them."""
    rng = random.Random(D)
    lens, news = [700, 90], [40, 33]
    trees = [random_tree(n, rng) for n in news]
    see = [x for t in trees for x in lines(t)]
    parents = torch.tensor([p for t in trees for p in t], dtype=torch.int32, device=dev)
    least = torch.finfo(dtype).smallest_normal
    s = Setup(dev, dtype, D, 1, 64, lens, news, seed=7)
    tree = _kv4().kv4_tree(parents, s.d_cu, s.d_seq, max_q=40)
    keys, q = s.k, s.q(G)
    for k in (0.0, least, 2.0 ** -10, 1.0):
        s.k = (keys.float() * k).to(dtype)
        again(s)
        for x in (0.0, least, 2.0 ** -10):
            for sm in (D ** -0.5, 1e-30):
                out = check(s, (q.float() * x).to(dtype), tree, see, max_q=40, max_kv=700, sm_scale=sm)
                assert torch.isfinite(out.float()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("D,G", [(128, 4), (64, 2)])
def test_large_queries_beside_large_keys(dev, D, G):
    """Queries near 2^96 in a channel that the keys have as 0, keys near 2^99 in the others: every score is 0, without a
    rounding. The steps are a power of two, so that c - 7.5 times one has 4 bits. The output is the mean, off by p's, its sum's
    and V's roundings to fp16 (2^-11 each of A, of A and of the output) and f32's sums (2^-12 A)."""
    rng = random.Random(D)
    lens, news = [700, 90], [40, 33]
    see = [x for n in news for x in lines(random_tree(n, rng))]
    s = Setup(dev, torch.bfloat16, D, 1, 64, lens, news, seed=9)
    s.k = (torch.randint(0, 16, s.k.shape, generator=torch.Generator().manual_seed(1)) * 2.0 ** 95).to(torch.bfloat16)
    s.k[:, :, 0], s.k[:, :, 1] = 0, 15 * 2.0 ** 95
    again(s)
    q = torch.zeros(sum(news), G, D, dtype=torch.bfloat16)
    q[:, :, 0] = 2.0 ** 95
    q[::3, :, 0] = -(2.0 ** 93)
    tree = mask_tree(see, [0] * len(see), dev, 2)
    out, lse = s.attend(q, tree=tree, max_q=40, max_kv=700, return_lse=True)
    want, rl, A, _, _ = ref(q, cache_values(s.cache), s.table, s.page, lens, news, see, [0] * len(see), D ** -0.5, bounds=True)
    assert ((out.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -11 * (2.5 * A + want.abs()) + 2.0 ** -25).all()
    assert (lse.cpu().double() - rl).abs().max().item() < 2e-4 + 2.0 ** -11


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_a_far_maximum_beside_keys_of_zeros(dev, dtype, sign):
    """Scores of 2^24 and more (in size) over the context, drafted tokens with keys of zeros that some rows do not see: those rows
    are the mean of the context, the others the one end of the softmax."""
    lens, news = [544, 500], [32, 20]
    s = Setup(dev, dtype, 128, 1, 64, lens, news, seed=11)
    for b, (n, new) in enumerate(zip(lens, news)):
        at = sum(lens[:b])
        s.k[at:at + n - new] = 2.0 ** 20 if dtype == torch.bfloat16 else 2.0 ** 15
        s.k[at + n - new:at + n] = 0
    again(s)
    q = torch.full((sum(news), 4, 128), sign * (8.0 if dtype == torch.bfloat16 else 1024.0), dtype=dtype)
    see = [x if i % 3 else [] for n in news for i, x in enumerate([[i] for i in range(n)])]
    out = check(s, q, mask_tree(see, [0] * len(see), dev, 1), see, max_q=32, max_kv=544)
    assert torch.isfinite(out.float()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("D,G", [(128, 4), (64, 2)])
@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** 25, 2.0 ** 45, 2.0 ** 90])
@pytest.mark.parametrize("equal", [True, False])
def test_keys_of_all_sizes_in_one_tile(dev, D, G, size, equal):
    """Context tokens with keys many times as large as their neighbours', whose scores are so far below those that they weigh
    nothing, and drafted tokens with such keys that some rows do not see: what the rest weighs is as without them. (All
    channels alike, a step of 2^-14 of the vector, or not.)"""
    rng = random.Random(D)
    lens, news = [700, 130], [40, 33]
    s = Setup(dev, torch.bfloat16, D, 1, 64, lens, news, seed=13)
    g = torch.Generator().manual_seed(5)
    big = torch.zeros(sum(lens), dtype=torch.bool)
    for b, (n, new) in enumerate(zip(lens, news)):
        at = sum(lens[:b])
        big[at:at + n - new:5] = True
        big[at + n - new:at + n:7] = True
    s.k[big] = (size * (torch.ones(1) if equal else torch.rand(int(big.sum()), 1, D, generator=g) * 0.5 + 0.75)).to(torch.bfloat16)
    again(s)
    q = (s.q(G).float() * 0.5 - 1.0).to(torch.bfloat16)  # the sum of a row's channels is below zero
    see = [[j for j in x if j % 7] or [1] for n in news for x in lines(random_tree(n, rng))]
    out = s.attend(q, tree=mask_tree(see, [0] * len(see), dev, 2), max_q=40, max_kv=700).cpu().double()
    # test_kv4_tree's tolerance, d over the keys that weigh something
    k, v = cache_values(s.cache)
    args = (s.table, s.page, lens, news, see, [0] * len(see), D ** -0.5)
    want, _, A, _, _ = ref(q, (k, v), *args, bounds=True)
    _, _, _, _, d = ref(q, (torch.where(k.abs().amax(-1, keepdim=True) > size / 2, 0.0, k), v), *args, bounds=True)
    rest = 2.0 ** -11 * (2.5 * A + want.abs()) + d * (A + want.abs())
    vmax = s.v.float().abs().max().item()
    assert ((out - want).abs() <= 2.0 ** -8 * want.abs() + torch.maximum(rest, torch.full_like(rest, 3.5e-4 * vmax)) + 2.0 ** -25).all()


@pytest.mark.gpu
@pytest.mark.parametrize("end", [65504.0, -65504.0])
@pytest.mark.parametrize("max_kv", [512, 2000])
def test_vectors_of_fp16s_last_number(dev, end, max_kv):
    """Values that are 65504 in all channels, whose range's middle is past fp16's end: in the context, alone or among others, and
    in a drafted token that some rows do not see, beside which nothing may change."""
    lens, news = [2000], [40]
    s = Setup(dev, torch.float16, 128, 1, 64, lens, news, seed=3)
    s.k[:] = 0
    s.k[700, 0, 0] = 16
    s.v[700], s.v[900], s.v[1970] = end, end, end  # 1970: new token 10
    again(s)
    q = torch.zeros(40, 4, 128, dtype=torch.float16)
    q[:, :2, 0] = 64  # a score of 102: token 700 takes all; the other heads weigh all the same
    see = [[i] if i % 2 else [i, 10] for i in range(40)]
    see[10] = [10]
    tree = mask_tree(see, [0] * 40, dev, 2)
    out, lse = s.attend(q, tree=tree, max_q=40, max_kv=max_kv, sm_scale=0.1, return_lse=True)
    want, rl, A, C, _ = ref(q, cache_values(s.cache), s.table, s.page, lens, news, see, [0] * 40, 0.1, bounds=True)
    assert (out[:, :2].cpu() == end).all()  # one key: its value
    # as test_kv4_tree has it: p s and the sum rounded to fp16, the output's rounding, f32's sums
    assert ((out.cpu().double() - want).abs() <= 2.0 ** -11 * (C + 0.5 * A + 2 * want.abs()) + 2.0 ** -24).all()
    assert (lse.cpu().double() - rl).abs().max().item() < 2e-4 + 2.0 ** -11
    # what no row sees weighs nothing
    none = [[i] if i != 10 else [] for i in range(40)]
    a = s.attend(q, tree=mask_tree(none, [0] * 40, dev, 2), max_q=40, max_kv=max_kv, sm_scale=0.1)
    s.v[1970] = 0
    again(s)
    assert torch.equal(a, s.attend(q, tree=mask_tree(none, [0] * 40, dev, 2), max_q=40, max_kv=max_kv, sm_scale=0.1))


# ------------------------------------------------------------------------------------------------
# GPU: windows
# ------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,width,new", [(64, 1, 1), (64, 2, 3), (128, 2, 30), (256, 3, 20), (128, 40, 70)])
def test_windows_past_the_table_are_nan(dev, dtype, D, width, new):
    """A sequence longer than its table: a row of a tree that sees a token past the table is NaN, whatever its window, as a row
    of a chain is; one that sees none is 0. Beside it a sequence that its table holds."""
    page = 16
    cap = width * page
    rng = random.Random(width)
    trees = [random_tree(new, rng), random_tree(2, rng)]
    parents = torch.tensor([p for t in trees for p in t], dtype=torch.int32, device=dev)
    for past in (0, 1, new, new + 1, new + 2, new + 7, 24, 4000, 2 ** 31 - 1 - cap):
        s = Setup(dev, dtype, D, 1, page, [cap, min(cap, 13)], [new, 2], seed=width)
        n = cap + past
        if n < new:
            continue
        s.lens = [n, s.lens[1]]
        s.d_seq = torch.tensor(s.lens, dtype=torch.int32, device=dev)
        q = s.q(2)
        for window in (1, 5, 8, cap + new):
            for kw in ({}, dict(max_q=new), dict(max_q=1, max_kv=1)):
                tree = _kv4().kv4_tree(parents, s.d_cu, s.d_seq, max_q=new, window=window)
                see = [x[-window:] for t in trees for x in lines(t)]
                check(s, q, tree, see, window, **kw)
                # rows that see nothing of the new tokens, from positions all over the window
                see = [x if i % 3 else [] for i, x in enumerate(see)]
                at = [min(p + rng.randrange(0, 2 * window), 2 ** 31 - 1) for p in tree.positions.tolist()]
                check(s, q, mask_tree(see, at, dev, tree.mask.shape[1]), see, window, **kw)


@pytest.mark.gpu
def test_tree_sizes_past_64_bits_are_refused(dev):
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    for max_q in (2 ** 63 - 1, 2 ** 62, 4097, 0, -2 ** 63):
        with pytest.raises(ValueError, match="max_q"):
            _kv4().kv4_tree(i32(-1, 0), i32(0, 2), i32(5), max_q=max_q)
