"""Attention over the 4-bit cache where a sequence's values are of sizes as far apart as is documented (steps below 2^64, or below
2^100 beside none below 2^-4): a token weighs what its score tells, whatever its value. References and tolerances are test_kv4's and test_kv4_tree's, relative to the largest value."""
import random

import pytest
import torch

import test_kv4_tree
from test_kv4 import Setup, _kv4


@pytest.mark.gpu
@pytest.mark.parametrize("small,large", [(0.0, 2.0 ** 66), (2.0 ** -60, 2.0 ** 66), (2.0 ** -120, 2.0 ** 66), (4.0, 2.0 ** 99)])
@pytest.mark.parametrize("D,G,news,lens", [(64, 4, [1, 1], [700, 3000]), (128, 2, [7, 20], [300, 900]), (64, 8, [30, 66], [300, 2000]),
                                           (256, 2, [1, 40], [500, 90])])
def test_weights_do_not_follow_values(dev, small, large, D, G, news, lens):
    """Zeros and small values before, among and behind large ones: over a wave's tiles, waves of a workgroup and splits."""
    rng = random.Random(D)
    s = Setup(dev, torch.bfloat16, D, 1, 16, lens, news, seed=21)
    base = s.v.float() / s.v.float().abs().max()
    at = torch.cat([torch.arange(n) for n in lens])
    size = torch.tensor([n for n in lens for _ in range(n)])
    trees = [test_kv4_tree.random_tree(n, rng) for n in news]
    see = [x for t in trees for x in test_kv4_tree.lines(t)]
    parents = torch.tensor([p for t in trees for p in t], dtype=torch.int32, device=dev)
    tree = _kv4().kv4_tree(parents, s.d_cu, s.d_seq, max_q=max(news))
    for big in (at >= size // 2, at < size // 2, at % 97 == 5, at % 64 < 32):
        s.v = torch.where(big.view(-1, 1, 1), base * large, base * small).to(torch.bfloat16)
        _kv4().kv4_append(s.cache, s.k.to(dev), s.v.to(dev), s.d_table, s.cu_all.to(dev), s.d_seq)
        for kw in ({}, {"max_q": max(news)}, {"max_q": max(news), "max_kv": max(lens)}):
            s.check(s.q(G), f"{small} {large} {kw}", **kw)
            # the narrow form of a tree: windows, heads of 256, few columns; and the one for many
            test_kv4_tree.check(s, s.q(G), tree, see, **kw)
            s.check(s.q(G), f"window, {small} {large} {kw}", window=200, **kw)
