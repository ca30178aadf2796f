"""The attention half of a layer as speculative decoding runs it: whole prompts, then drafted trees that are verified, their
accepted tokens kept, and the next step on top, with rotary positions throughout; steps captured and replayed; and a
sequence that is forked. Every step's attention is held against 64 bits over what the cache holds, and the cache against
the tokens that were accepted."""
import random

import pytest
import torch

from conftest import pkg
from test_kv4 import cache_values, ref_values
from test_kv4_tree import lines, random_tree, ref as tree_ref
from test_prompt_attention import compare, ref as prompt_ref
from test_rotary import check as rotary_check, freqs

HQ, H, D, PAGE, BASE = 8, 2, 64, 16, 1e4


def _qkv(T, g, dtype):
    return (torch.randn(T, (HQ + 2 * H) * D, generator=g) * 0.8).to(dtype)


def _split(qkv):
    return tuple(t.reshape(qkv.shape[0], -1, D) for t in qkv.split([HQ * D, H * D, H * D], 1))


def _close(out, want, v, dtype):
    eps = 2.0 ** (-8 if dtype == torch.bfloat16 else -11)
    err = (out.cpu().double().view(want.shape) - want).abs() - eps * want.abs() - (3.5e-4 if dtype == torch.bfloat16 else 2e-4) * v - 2.0 ** -25
    assert err.max().item() <= 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompts_trees_and_kept_tokens(dev, dtype):
    kv4, att, rotary = pkg("quant.kv4"), pkg("layers.attention"), pkg("layers.rotary")
    g, rng = torch.Generator().manual_seed(3), random.Random(3)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    rot = rotary.Rotary(D, base=BASE, device=dev)
    layers = [att.KV4Attention(HQ, kv4.KV4Cache(40, PAGE, H, D, dtype, dev), rotary=rot) for _ in range(2)]
    caches = [x.cache for x in layers]
    table = torch.randperm(40, generator=g).int()[:24].view(3, 8)
    d_table = table.to(dev)
    lens = [37, 1, 64]
    cu = [0, 37, 38, 102]
    axis = torch.zeros(D // 2, dtype=torch.long)
    kept_k, kept_v = [[[] for _ in lens] for _ in layers], [[[] for _ in lens] for _ in layers]

    # whole prompts: attention over their own keys, in the model's type
    positions = torch.cat([torch.arange(n) for n in lens]).int()
    batch = att.KV4Batch(d_table, i32(cu), i32(lens), max(lens), max(lens), positions=positions.to(dev), whole=True)
    for l, layer in enumerate(layers):
        qkv = _qkv(cu[-1], g, dtype).to(dev)
        out = layer.forward_qkv(qkv, batch)
        q, k, v = _split(qkv)
        qr, kr = rot.forward(q, k, positions.to(dev))
        rotary_check(qr, q, positions.view(1, -1), freqs(BASE, D), axis, D, False, 1.0)
        compare(out.view(-1, HQ, D), None, prompt_ref(qr, kr, v, cu, D ** -0.5), dtype, D, max(lens))
        for b in range(3):
            kept_k[l][b].append(kr[cu[b]:cu[b + 1]].cpu())
            kept_v[l][b].append(v[cu[b]:cu[b + 1]].cpu())

    # drafted trees; the step of both layers is captured once per shape and replayed with what changes
    news = [6, 4, 9]
    T, cu_t = sum(news), [0, 6, 10, 19]
    s_qkv = [torch.zeros(T, (HQ + 2 * H) * D, dtype=dtype, device=dev) for _ in layers]
    s_parents, s_lens, s_cu = i32([0] * T), i32([0, 0, 0]), i32(cu_t)
    s_keep, s_kept = i32([[0] * 9] * 3), i32([0, 0, 0])

    def step():
        tree = kv4.kv4_tree(s_parents, s_cu, s_lens, max_q=max(news))
        b = att.KV4Batch(d_table, s_cu, s_lens, max(news), 8 * PAGE, tree=tree)
        return tree, [layer.forward_qkv(x, b) for layer, x in zip(layers, s_qkv)]

    def accept():
        return kv4.kv4_keep(caches, d_table, s_cu, s_lens, s_keep, s_kept)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), accept()  # lengths of 0: nothing is written
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    verify, finish = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(verify):
        tree, outs = step()
    with torch.cuda.graph(finish):
        now = accept()
    for rep in range(4):
        trees = [random_tree(n, rng, near=3) for n in news]
        full = [n + w for n, w in zip(lens, news)]
        s_parents.copy_(i32([p for t in trees for p in t]))
        s_lens.copy_(i32(full))
        qkvs = [_qkv(T, g, dtype) for _ in layers]
        for a, b in zip(s_qkv, qkvs):
            a.copy_(b)
        verify.replay()
        torch.cuda.synchronize()
        see = [x for t in trees for x in lines(t)]
        positions = [n + len(x) - 1 for n, t in zip(lens, trees) for x in lines(t)]
        assert tree.positions.tolist() == positions
        turned = []
        for l, (layer, x, out) in enumerate(zip(layers, s_qkv, outs)):
            q, k, v = _split(x)
            qr, kr = rot.forward(q, k, tree.positions)
            turned.append((kr.cpu(), v.cpu()))
            kv = cache_values(layer.cache)
            want, _ = tree_ref(qr.cpu(), kv, table, PAGE, full, news, see, positions, D ** -0.5)
            _close(out, want, 4.0, dtype)
            eager = kv4.kv4_attention(qr, layer.cache, d_table, s_cu, s_lens, tree=kv4.KV4Tree(*(t.clone() for t in tree)), max_q=max(news),
                                      max_kv=8 * PAGE)
            assert torch.equal(eager.view(T, -1), out), rep
        # a path of each tree is accepted, of one sequence nothing
        path = [lines(t)[rng.randrange(len(t))] for t in trees]
        path[rep % 3] = []
        s_keep.copy_(i32([p + [-5] * (9 - len(p)) for p in path]))
        s_kept.copy_(i32([len(p) for p in path]))
        finish.replay()
        torch.cuda.synchronize()
        lens = [n + len(p) for n, p in zip(lens, path)]
        assert now.tolist() == lens
        for l, layer in enumerate(layers):
            ck, cv = cache_values(layer.cache)
            for b in range(3):
                rows = [cu_t[b] + i for i in path[b]]
                kept_k[l][b].append(turned[l][0][rows])
                kept_v[l][b].append(turned[l][1][rows])
                pos = torch.arange(lens[b])
                at = table[b, pos // PAGE].long(), pos % PAGE
                assert torch.equal(ck[at[0], :, at[1]], ref_values(torch.cat(kept_k[l][b])))
                assert torch.equal(cv[at[0], :, at[1]], ref_values(torch.cat(kept_v[l][b])))

    # a fork of the last sequence: full pages shared, the last one copied; both go on with tokens of their own
    last = (lens[2] - 1) // PAGE
    free = [p for p in range(40) if p not in table.flatten().tolist()]
    kv4.kv4_copy_pages(caches, i32([table[2, last].item()]), i32([free[0]]))
    fork = torch.stack([table[2], table[2]])
    fork[1, last] = free[0]
    if lens[2] % PAGE == 0:
        fork[0, last + 1], fork[1, last + 1] = free[1], free[2]
    for l, layer in enumerate(layers):
        qkv = _qkv(2, g, dtype).to(dev)
        positions = i32([lens[2], lens[2]])
        b = att.KV4Batch(fork.to(dev), i32([0, 1, 2]), i32([lens[2] + 1] * 2), 1, 8 * PAGE, positions=positions)
        out = layer.forward_qkv(qkv, b)
        q, k, v = _split(qkv)
        qr, kr = rot.forward(q, k, positions)
        kv = cache_values(layer.cache)
        want, _ = tree_ref(qr.cpu(), kv, fork, PAGE, [lens[2] + 1] * 2, [1, 1], [[0], [0]], [lens[2]] * 2, D ** -0.5)
        _close(out, want, 4.0, dtype)
        pos = torch.arange(lens[2] + 1)
        for i in range(2):
            at = fork[i, pos // PAGE].long(), pos % PAGE
            assert torch.equal(kv[0][at[0], :, at[1]], ref_values(torch.cat(kept_k[l][2] + [kr[i:i + 1].cpu()])))
            assert torch.equal(kv[1][at[0], :, at[1]], ref_values(torch.cat(kept_v[l][2] + [v[i:i + 1].cpu()])))


def test_layer_refusals():
    kv4, att, rotary = pkg("quant.kv4"), pkg("layers.attention"), pkg("layers.rotary")
    cache = kv4.KV4Cache(2, 16, 2, 64, device="cpu")
    with pytest.raises(ValueError, match="rotary for heads"):
        att.KV4Attention(4, cache, rotary=rotary.Rotary(128, device="cpu"))
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32)  # noqa: E731
    t = lambda n: torch.zeros(1, n, dtype=torch.bfloat16)  # noqa: E731
    b = att.KV4Batch(i32([0]).view(1, 1), i32(0, 1), i32(1))
    with pytest.raises(ValueError, match="positions"):
        att.KV4Attention(4, cache, rotary=rotary.Rotary(64, device="cpu")).forward(t(256), t(128), t(128), b)
    with pytest.raises(ValueError, match="no tree"):
        att.KV4Attention(4, cache).forward(t(256), t(128), t(128), b._replace(whole=True, tree=kv4.KV4Tree(i32([1]), i32(1))))
