"""Trees of drafted tokens over the 4-bit cache (quant/kv4.py kv4_tree, kv4_attention(tree=)): refusals on the CPU, and on
the GPU bits and positions against a walk up the tree, and attention against 64 bits over the cached values.

Tolerances. Up to 64 columns (queries times heads that share a key), and with a window, the ones that attention over the
cache is tested with. More columns: with A = sum p |v| / sum p, the output o is off by
  - p rounded to fp16, and its sum, 2^-11 (A + |o|);
  - bf16 models: V' = s c + m rounded to fp16, 2^-11 A;
  - fp16 models instead: p s rounded to fp16, 2^-11 of sum p |v - mid| / sum p, mid the middle of the value's range;
    mid rounded to fp16, and summed with p as it is but divided by the rounded ones' sum: 2^-11 2 sum p |mid| / sum p;
  - bf16 models: s (c - 7.5), 8 bits by 4, rounded to fp16's 11, 2^-11 of it: a score is off by d = 2^-11 scale sum |q| |k - mid|,
    mid the middle of the key's range, p by d of itself and o by d (A + |o|);
  - 2^-25 of the largest cached value's power of two where V' is subnormal, and f32's sums and exponentials, 2^-12 A here,
and by the rounding of the output. d moves lse as well."""
import math
import random

import pytest
import torch

from conftest import pkg
from test_kv4 import Setup, cache_values

DTYPES = [torch.bfloat16, torch.float16]


def _kv4():
    return pkg("quant.kv4")


def lines(parents):
    """Each node's ancestors and itself, the root first."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if 0 <= p < i else []) + [i])
    return out


def random_tree(n, rng, near=6):
    return [-1 if i == 0 or rng.random() < 0.15 else rng.randrange(max(0, i - near), i) for i in range(n)]


def pack(see, words):
    """(rows, words) int32 of lists of seen tokens."""
    out = []
    for s in see:
        bits = sum(1 << j for j in s if j < 32 * words)
        part = [(bits >> (32 * w)) & 0xffffffff for w in range(words)]
        out.append([w - (1 << 32) if w >> 31 else w for w in part])
    return torch.tensor(out, dtype=torch.int32).view(len(see), words)


def ref(q, kv, table, page, lens, news, see, positions, scale, window=0, bounds=False):
    """see: per row the new tokens that it sees. out and lse in f64, NaN where a page is missing."""
    k, v = kv
    H = k.shape[1]
    T, Hq, D = q.shape
    G = Hq // H
    out, A, C = (torch.zeros(T, Hq, D, dtype=torch.float64) for _ in range(3))
    lse, d = torch.full((T, Hq), -math.inf, dtype=torch.float64), torch.zeros(T, Hq, 1, dtype=torch.float64)
    row = 0
    for b, (n, new) in enumerate(zip(lens, news)):
        for i in range(new):
            r = row + i
            lo = max(0, positions[r] - window + 1) if window else 0
            keys = list(range(lo, max(n - new, 0))) + [n - new + j for j in see[r] if j < new and n - new + j >= 0]
            if not keys:
                continue
            pos = torch.tensor(keys)
            missing = pos // page >= table.shape[1]
            pages = table[b, (pos // page).clamp_max(table.shape[1] - 1)].long()
            missing |= (pages < 0) | (pages >= k.shape[0])
            if missing.any():
                out[r], lse[r] = math.nan, math.nan
                continue
            kk = k[pages, :, pos % page].repeat_interleave(G, 1).transpose(0, 1)  # (Hq, keys, D)
            vv = v[pages, :, pos % page].repeat_interleave(G, 1).transpose(0, 1)
            x = (kk * q[r].double().unsqueeze(1)).sum(-1) * scale
            pr = torch.softmax(x, 1).unsqueeze(-1)
            out[r], A[r] = (pr * vv).sum(1), (pr * vv.abs()).sum(1)
            half = (vv.amax(-1, keepdim=True) + vv.amin(-1, keepdim=True)) / 2
            C[r] = (pr * ((vv - half).abs() + 2 * half.abs())).sum(1)
            lse[r] = torch.logsumexp(x, 1)
            mid = (kk.amax(-1, keepdim=True) + kk.amin(-1, keepdim=True)) / 2
            d[r, :, 0] = ((kk - mid).abs() * q[r].double().abs().unsqueeze(1)).sum(-1).amax(1) * scale * 2.0 ** -11
        row += new
    return (out, lse, A, C, d) if bounds else (out, lse)


def check(s, q, tree, see, window=0, lse_of_nan=True, **kw):
    out, lse = s.attend(q, tree=tree, window=window, return_lse=True, **kw)
    D = s.cache.head_dim
    scale = kw.get("sm_scale", D ** -0.5)
    want, rl, A, C, d = ref(q, cache_values(s.cache), s.table, s.page, s.lens, s.news, see, tree.positions.tolist(), scale, window, True)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(out.cpu()), nan)
    eps = 2.0 ** (-8 if q.dtype == torch.bfloat16 else -11)
    vmax = s.v.float().abs().max().item()
    rest = torch.full_like(want, (3.5e-4 if q.dtype == torch.bfloat16 else 2e-4) * vmax)
    rows = min(max(kw.get("max_q", q.shape[0]), -(-q.shape[0] // len(s.lens))), q.shape[0])
    wide = not window and D <= 128 and rows * (q.shape[1] // s.cache.num_kv_heads) > 64
    if wide:
        d = d if q.dtype == torch.bfloat16 else torch.zeros_like(d)
        rounded = 2 * A if q.dtype == torch.bfloat16 else C
        rest = torch.maximum(rest, 2.0 ** -11 * (rounded + 0.5 * A + want.abs()) + d * (A + want.abs()) + 2.0 ** -25 * max(vmax, 2.0 ** -24))
    err = (out.cpu().double() - want).abs() - eps * want.abs() - rest - 2.0 ** -25
    assert err[~nan].numel() == 0 or err[~nan].max().item() <= 0, f"off by {err[~nan].max().item():.3e} past the tolerance"
    lf = torch.isfinite(rl)
    if not lse_of_nan:  # a row that sees a value that is NaN: its lse is not specified
        lf &= ~nan.any(-1)
    assert torch.equal(torch.isfinite(lse.cpu()) & lf, lf) and (not lse_of_nan or torch.equal(torch.isfinite(lse.cpu()), lf))
    most = 2 * s.k.double().abs().max().item() * q.double().abs().sum(-1).max().item() * scale
    tol = 2e-4 + 2.0 ** -21 * most + (d.squeeze(-1) + 2.0 ** -11 if wide else 0.0 * d.squeeze(-1))
    assert not lf.any() or ((lse.cpu().double() - rl).abs() - tol)[lf].max().item() < 0
    return out


# ------------------------------------------------------------------------------------------------
# CPU
# ------------------------------------------------------------------------------------------------
def test_refusals():
    kv4 = _kv4()
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32)  # noqa: E731
    with pytest.raises(RuntimeError, match="one GPU"):
        kv4.kv4_tree(i32(-1, 0), i32(0, 2), i32(5), max_q=2)
    with pytest.raises(TypeError, match="parents"):
        kv4.kv4_tree(i32(-1, 0).long(), i32(0, 2), i32(5), max_q=2)
    c = kv4.KV4Cache(4, 32, 2, 128, device="cpu")
    x = torch.zeros(2, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="on the GPU"):
        kv4.kv4_attention(x, c, i32([0]).view(1, 1), i32(0, 2), i32(5), tree=kv4.KV4Tree(i32([1], [3]), i32(3, 4)))


def test_abi_refusals():
    if torch.cuda.is_available():
        pytest.skip("the pointers are not real")
    lib = pkg("_abi").load()
    P = 1 << 20
    for a, code in (((P, 4, P, P, 1, 0, 0, P, P), 1), ((P, 4, P, P, 1, 129, 0, P, P), 1), ((P, 4, P, P, 1, 1, -1, P, P), 1),
                    ((P, -1, P, P, 1, 1, 0, P, P), 1), ((None, 4, P, P, 1, 1, 0, P, P), 1), ((P, 4, P, P, 1, 1, 0, P, None), 1),
                    ((P, 1 << 31, P, P, 1, 1, 0, P, P), 2), ((P, 0, P, P, 1, 1, 0, P, P), 0), ((P, 4, P, P, 0, 1, 0, P, P), 0)):
        assert lib.w4a8_kv4_tree(*a, None) == code, a

    def attend(bits=P, ldb=1, words=1, pos=P, window=0, width=4, T=2):
        rc = lib.w4a8_kv4_tree_attention(P, 0, 512, 128, T, 4, 1, 128, P, P, P, P, 16, 16, P, width, width, P, P, 1, 1.0, window, 2, 64, bits,
                                         ldb, words, pos, P, 256, 64, None, None, 0, None)
        return rc, lib.w4a8_last_error().decode()

    for kw in (dict(bits=None), dict(words=0), dict(words=129, ldb=129), dict(ldb=1, words=2), dict(window=4, pos=None)):
        rc, msg = attend(**kw)
        assert rc == 1 and "bits" in msg, (kw, rc, msg)
    rc, msg = attend(width=(1 << 27) - 4)
    assert rc == 2 and "index ranges" in msg
    assert attend()[1].startswith("w4a8_kv4_tree_attention: out's rows overlap")


# ------------------------------------------------------------------------------------------------
# GPU
# ------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 1, 3])
def test_bits_and_positions(dev, window):
    rng = random.Random(window)
    news = [1, 0, 33, 64, 5, 150, 700]
    trees = [random_tree(n, rng) for n in news]
    trees[3] = list(range(-1, 63))   # a chain
    trees[4] = [3, -7, 2, 0, 4]      # entries that do not stand before their node
    lens = [n + rng.randrange(0, 50) for n in news]
    cu = [3 + sum(news[:i]) for i in range(len(news) + 1)]
    parents = torch.full((cu[-1] + 4,), 77, dtype=torch.int32)
    parents[3:cu[-1]] = torch.tensor([p for t in trees for p in t], dtype=torch.int32)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    for max_q in (700, 1024, 90):
        tree = _kv4().kv4_tree(parents.to(dev), i32(cu), i32(lens), max_q=max_q, window=window)
        assert tree.mask.shape == (len(parents), -(-max_q // 32))
        at = 3
        for t, n in zip(trees, lens):
            line = lines(t)
            see = [x[-window:] if window else x for x in line]
            assert torch.equal(tree.mask[at:at + len(t)].cpu(), pack(see, tree.mask.shape[1]))
            assert tree.positions[at:at + len(t)].tolist() == [n - len(t) + len(x) - 1 for x in line]
            at += len(t)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,H,G,page", [(128, 2, 4, 16), (64, 1, 3, 32), (256, 1, 2, 16), (128, 1, 8, 64), (64, 2, 1, 16)])
@pytest.mark.parametrize("lens,news", [([40, 9, 200], [7, 9, 3]), ([500, 0, 1, 90], [33, 0, 1, 70]), ([1100], [13]), ([2000, 77], [64, 2])])
def test_trees(dev, dtype, D, H, G, page, lens, news):
    s = Setup(dev, dtype, D, H, page, lens, news, seed=D + G)
    q = s.q(H * G, scale=1.5)
    rng = random.Random(sum(news))
    trees = [random_tree(n, rng) for n in news]
    parents = torch.tensor([p for t in trees for p in t], dtype=torch.int32, device=dev)
    for window, kw in ((0, dict(max_q=max(news), max_kv=max(lens))), (5, {}), (64, dict(max_q=max(news))), (0, dict(max_q=1, sm_scale=0.3))):
        tree = _kv4().kv4_tree(parents, s.d_cu, s.d_seq, max_q=max(news), window=window)
        see = [x[-window:] if window else x for t in trees for x in lines(t)]
        check(s, q, tree, see, window, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_chain_is_causal_attention(dev, dtype):
    """Where every drafted token follows the one before it: the same bits where the launch is planned alike, with a window and
    for few columns; else nearly."""
    for D, G, lens, news in ((128, 4, [300, 40, 9000], [20, 40, 4]), (64, 3, [64, 100], [1, 3]), (128, 4, [300, 40, 2000], [20, 32, 4])):
        s = Setup(dev, dtype, D, 2, 16, lens, news, seed=1)
        q = s.q(2 * G)
        parents = torch.tensor([i - 1 for n in news for i in range(n)], dtype=torch.int32, device=dev)
        for window in (0, 17):
            tree = _kv4().kv4_tree(parents, s.d_cu, s.d_seq, max_q=max(news), window=window)
            for kw in ({}, dict(max_q=max(news), max_kv=max(lens))):
                a, al = s.attend(q, tree=tree, window=window, return_lse=True, **kw)
                b, bl = s.attend(q, window=window, return_lse=True, **kw)
                if window or max(news) * G <= 16:
                    assert torch.equal(a, b) and torch.equal(al, bl)
                else:
                    check(s, q, tree, [list(range(i + 1)) for n in news for i in range(n)], **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("news,context,D", [([3, 2], 60, 64), ([40, 100], 60, 64), ([40, 100], 600, 64), ([70, 90], 530, 128)])
def test_any_mask(dev, dtype, news, context, D):
    """Rows that see nothing, everything, only others, bits past the tokens, and too few words."""
    lens = [context, context + 40]
    s = Setup(dev, dtype, D, 2, 16, lens, news, seed=4)
    q = s.q(4)
    T = sum(news)
    rng = random.Random(5)
    see = [sorted(rng.sample(range(n), rng.randrange(0, n + 1))) for n in news for _ in range(n)]
    see[0], see[1] = [], list(range(news[0]))
    positions = [n - w + rng.randrange(0, w) for n, w in zip(lens, news) for _ in range(w)]
    for words in (1, 4, 7):
        mask = pack(see, words)
        if words > 4:
            mask[:, -1] = -1  # tokens 192 .. 223: there are none
        seen = [[j for j in x if j < 32 * words] for x in see]
        tree = _kv4().KV4Tree(mask.to(dev), torch.tensor(positions, dtype=torch.int32, device=dev))
        for window in (0, 30, 1):
            check(s, q, tree, seen, window)
    # no context at all: what sees nothing is 0
    s = Setup(dev, dtype, D, 2, 16, news, news, seed=4)
    tree = _kv4().KV4Tree(pack(see, 4).to(dev), torch.zeros(T, dtype=torch.int32, device=dev))
    out = check(s, q, tree, see, **(dict(max_q=max(news)) if context > 500 else {}))
    assert not out[0].any()
    # a window from a position far behind: none of the context
    tree = _kv4().KV4Tree(pack(see, 4).to(dev), torch.full((T,), 2 ** 31 - 1, dtype=torch.int32, device=dev))
    check(s, q, tree, see, 5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("news,lens", [([5, 3], [70, 90]), ([64, 40], [70, 90]), ([64, 40], [700, 590]), ([70, 600], [700, 600])])
def test_missing_pages_and_unseen_values(dev, dtype, news, lens):
    """Tokens on pages that do not exist, or past the table: NaN in who sees them and in nobody else; so are tokens whose
    vectors are not finite."""
    s = Setup(dev, dtype, 128, 1, 16, lens, news, seed=2)
    q = s.q(4)
    rng = random.Random(1)
    trees = [random_tree(n, rng) for n in news]
    see = [x for t in trees for x in lines(t)]
    parents = torch.tensor([p for t in trees for p in t], dtype=torch.int32, device=dev)
    tree = _kv4().kv4_tree(parents, s.d_cu, s.d_seq, max_q=max(news))
    s.table[0, (lens[0] - 1) // 16] = -1     # the last tokens of the first sequence
    s.d_table = s.table.to(dev)
    check(s, q, tree, see)
    # lengths past the table: the last nodes have no place
    s.table = s.table[:, :s.table.shape[1] - (1 if lens[0] < 100 else 3)].contiguous()
    s.d_table = s.table.to(dev)
    check(s, q, tree, see)
    wide = torch.full((2, s.table.shape[1]), 2 ** 30, dtype=torch.int32)
    s.table = wide
    s.d_table = wide.to(dev)
    check(s, q, tree, see)
    # a node that holds NaN
    s = Setup(dev, dtype, 128, 1, 16, lens, news, seed=2)
    at = lens[1] - news[1] + 1
    page, slot = s.table[1, at // 16].item(), at % 16
    s.cache.v_scale[page, :, slot] = math.nan
    tree = _kv4().kv4_tree(parents, s.d_cu, s.d_seq, max_q=max(news))
    out = check(s, q, tree, see, lse_of_nan=False)
    sees = torch.tensor([r >= news[0] and 1 in see[r] for r in range(sum(news))])
    assert torch.equal(torch.isnan(out.cpu()).flatten(1).all(1), sees)
    # a token of the context that holds an infinity: every row of its sequence is NaN, and no other
    if lens[1] > news[1] + 40:
        start = sum(lens[:1])
        for x, at in (("k", 33), ("v", 18)):
            s = Setup(dev, dtype, 128, 1, 16, lens, news, seed=2)
            getattr(s, x)[start + at, 0, 7] = -math.inf
            _kv4().kv4_append(s.cache, s.k.to(dev), s.v.to(dev), s.d_table, s.cu_all.to(dev), s.d_seq)
            out = s.attend(q, tree=tree)
            assert not torch.isfinite(out[news[0]:].float()).any() and torch.isfinite(out[:news[0]].float()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,G", [(64, 8), (128, 8), (64, 2), (128, 2)])
def test_wide_trees_of_any_size(dev, dtype, D, G):
    """More than 64 columns: keys, values and queries of sizes far from 1, scores that raise the maximum in every tile and
    scores past 2^24, one split and many."""
    rng = random.Random(D)
    lens, news = [1500, 64, 900], [50, 64, 31]
    trees = [random_tree(n, rng) for n in news]
    see = [x for t in trees for x in lines(t)]
    parents = torch.tensor([p for t in trees for p in t], dtype=torch.int32, device=dev)
    big, small = (2.0 ** 40, 2.0 ** -40) if dtype == torch.bfloat16 else (2.0 ** 9, 2.0 ** -9)
    cases = [(1.0, 1.0, 1.0), (big, small, small), (small, big, big), (big, big, small), (small, small, big)]
    if dtype == torch.bfloat16:  # up to the steps that may be cached, 2^100, and the queries' 2^96
        cases += [(1.0, 2.0 ** 100, 1.0), (2.0 ** 100, 1.0, 2.0 ** -101), (2.0 ** -90, 2.0 ** -90, 2.0 ** 92)]
    for ks, vs, qs in cases:
        s = Setup(dev, dtype, D, 1, 64, lens, news, seed=3)
        ramp = torch.cat([torch.arange(n) for n in lens]).view(-1, 1, 1) / 200 if ks == 1.0 else 1.0
        s.k, s.v = (s.k.float() * ramp * ks).to(dtype), (s.v.float() * vs).to(dtype)
        _kv4().kv4_append(s.cache, s.k.to(dev), s.v.to(dev), s.d_table, s.cu_all.to(dev), s.d_seq)
        q = (s.q(G).float() * qs).to(dtype)
        tree = _kv4().kv4_tree(parents, s.d_cu, s.d_seq, max_q=64)
        check(s, q, tree, see, max_q=64, max_kv=1500)
        check(s, q, tree, see, max_q=64, max_kv=512)
    # far scores: whole numbers, so that those that are equal are equal, and one row of them takes all
    s = Setup(dev, dtype, D, 1, 64, lens, news, seed=3)
    s.k = torch.randint(0, 16, s.k.shape, generator=torch.Generator().manual_seed(1)).to(dtype)
    s.k[:, :, 0], s.k[:, :, 1] = 0, 15  # a step of 1 and a least value of 0: every code is a whole number
    _kv4().kv4_append(s.cache, s.k.to(dev), s.v.to(dev), s.d_table, s.cu_all.to(dev), s.d_seq)
    q = (torch.randint(-2, 3, (sum(news), G, D), generator=torch.Generator().manual_seed(2)) * 2.0 ** 12).to(dtype)
    out = s.attend(q, tree=tree, sm_scale=64.0, max_q=64, max_kv=1500)
    want, _ = ref(q, cache_values(s.cache), s.table, s.page, lens, news, see, tree.positions.tolist(), 64.0)
    eps = 2.0 ** (-8 if dtype == torch.bfloat16 else -11)
    assert ((out.cpu().double() - want).abs() <= eps * want.abs() + 2.0 ** -9 * s.v.float().abs().max().item()).all()


@pytest.mark.gpu
def test_out_rows_streams_and_refusals(dev):
    kv4 = _kv4()
    s = Setup(dev, torch.bfloat16, 128, 2, 16, [100, 50], [6, 4], seed=3)
    q = s.q(8)
    parents = torch.tensor([-1, 0, 0, 1, 1, 2, -1, -1, 0, 1], dtype=torch.int32, device=dev)
    tree = kv4.kv4_tree(parents, s.d_cu, s.d_seq, max_q=6)
    want = s.attend(q, tree=tree)
    pad = torch.cat([torch.zeros_like(q[:2]), q, torch.zeros_like(q[:3])]).to(dev)
    mask = torch.cat([torch.full((2, 1), -1, dtype=torch.int32, device=dev), tree.mask, torch.full((3, 1), -1, dtype=torch.int32, device=dev)])
    pos = torch.cat([torch.zeros(2, dtype=torch.int32, device=dev), tree.positions, torch.zeros(3, dtype=torch.int32, device=dev)])
    out = torch.full_like(pad, 9.0)
    kv4.kv4_attention(pad, s.cache, s.d_table, s.d_cu + 2, s.d_seq, tree=kv4.KV4Tree(mask, pos), out=out)
    assert torch.equal(out[2:12], want) and (out[:2] == 9).all() and (out[12:] == 9).all()
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        t2 = kv4.kv4_tree(parents, s.d_cu, s.d_seq, max_q=6)
        got = s.attend(q, tree=t2)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    m, p = tree
    for bad, e in (((m[:9], p), TypeError), ((m.long(), p), TypeError), ((m, p[:9]), TypeError), ((m.cpu(), p), RuntimeError),
                   ((m[:, :0], p), TypeError), ((m.expand(10, 1).repeat(1, 129), p), TypeError)):
        with pytest.raises(e):
            s.attend(q, tree=kv4.KV4Tree(*bad))
    strided = m.repeat(1, 3)[:, ::3]
    assert torch.equal(s.attend(q, tree=kv4.KV4Tree(strided, p)), want)
    for kw, e in ((dict(max_q=0), ValueError), (dict(max_q=4097), ValueError), (dict(max_q=6, window=-1), ValueError)):
        with pytest.raises(e):
            kv4.kv4_tree(parents, s.d_cu, s.d_seq, **kw)
    with pytest.raises(ValueError, match="cu_q"):
        kv4.kv4_tree(parents, s.d_cu[:2], s.d_seq, max_q=6)
    none = kv4.kv4_tree(parents[:0], s.d_cu * 0, s.d_seq, max_q=6)
    assert none.mask.shape == (0, 1) and none.positions.shape == (0,)


@pytest.mark.gpu
@pytest.mark.parametrize("max_kv", [512, 2000])
def test_wide_trees_at_the_ends_of_fp16(dev, max_kv):
    """fp16 vectors from the least to the greatest number, whose steps and least values give 65536, and many small weights
    beside a great one."""
    lens, news = [2000], [40]
    s = Setup(dev, torch.float16, 128, 1, 64, lens, news, seed=3)
    s.v[100::7, 0, 0], s.v[100::7, 0, 5] = 65504, -65504
    s.k[:], s.k[::16, 0, 0] = 0, 0.25
    s.k[50, 0, 0] = 16
    _kv4().kv4_append(s.cache, s.k.to(dev), s.v.to(dev), s.d_table, s.cu_all.to(dev), s.d_seq)
    q = torch.zeros(40, 4, 128, dtype=torch.float16)
    q[:, :2, 0] = 11  # one score is 17.6 above the others; the other heads weigh all the same
    tree = _kv4().kv4_tree(torch.full((40,), -1, dtype=torch.int32, device=dev), s.d_cu, s.d_seq, max_q=40)
    see = [[i] for i in range(40)]
    out, lse = s.attend(q, tree=tree, max_q=40, max_kv=max_kv, sm_scale=0.1, return_lse=True)
    want, rl, A, C, _ = ref(q, cache_values(s.cache), s.table, s.page, lens, news, see, tree.positions.tolist(), 0.1, bounds=True)
    assert torch.isfinite(want).all() and (want.abs() > 2.0 ** -6 * 65504).any()
    # a weight below fp16's normal numbers is off by 2^-25 at most, where the largest, and so their sum, is 2^7 at least
    at = torch.arange(lens[0])
    v = cache_values(s.cache)[1][s.table[0, at // 64].long(), 0, at % 64]
    mid = (v.amax(-1, keepdim=True) + v.amin(-1, keepdim=True)) / 2
    least = 2.0 ** -32 * ((v - mid).abs() + mid.abs()).sum(0)
    assert ((out.cpu().double() - want).abs() <= 2.0 ** -11 * (C + 0.5 * A + 2 * want.abs()) + least + 2.0 ** -24).all()
    assert (lse.cpu().double() - rl).abs().max().item() < 2e-4 + 2.0 ** -11


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_wide_trees_in_place_and_padded(dev, dtype):
    """The output in q's place; a sequence with one token, one with none and one that is all new beside a long one; rows
    behind the last sequence; a captured launch replayed over other lengths; the same rows whatever lies beside them."""
    lens, news = [1200, 33, 0, 70, 900], [60, 1, 0, 70, 33]
    s = Setup(dev, dtype, 128, 2, 32, lens, news, seed=8)
    rng = random.Random(8)
    trees = [random_tree(n, rng) for n in news]
    see = [x for t in trees for x in lines(t)]
    parents = torch.tensor([p for t in trees for p in t], dtype=torch.int32, device=dev)
    tree = _kv4().kv4_tree(parents, s.d_cu, s.d_seq, max_q=70)
    q = s.q(8)
    a = check(s, q, tree, see, max_q=70, max_kv=1200)
    T = sum(news)
    mine = torch.full((T + 5, 8, 128), 7.0, dtype=dtype, device=dev)
    mine[:T] = q.to(dev)
    big = _kv4().KV4Tree(torch.cat([tree.mask, tree.mask[:5]]), torch.cat([tree.positions, tree.positions[:5]]))
    kw = dict(max_q=70, max_kv=1200, tree=big)
    _kv4().kv4_attention(mine, s.cache, s.d_table, s.d_cu, s.d_seq, out=mine, **kw)
    assert torch.equal(mine[:T], a) and (mine[T:] == 7).all()
    # replays over other contexts of the same tokens
    q2, seq, out = q.to(dev), s.d_seq.clone(), torch.empty_like(q, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s_kw = dict(max_q=70, max_kv=1200, tree=tree, out=out)
        _kv4().kv4_attention(q2, s.cache, s.d_table, s.d_cu, seq, **s_kw)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _kv4().kv4_attention(q2, s.cache, s.d_table, s.d_cu, seq, **s_kw)
    for less in (0, 100, 7, 0):
        seq.copy_(torch.tensor([lens[0] - less] + lens[1:], dtype=torch.int32))
        out.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        torch.empty(1 << 20, device=dev).normal_()
        _kv4().kv4_attention(q2, s.cache, s.d_table, s.d_cu, seq, **s_kw)
        assert torch.equal(replayed, out)
        assert torch.equal(replayed[60:], a[60:])
    assert torch.equal(out, a)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,D", [(1024, 64), (16384, 128), (131072, 64), (131072, 128)])
@pytest.mark.parametrize("T,kw", [(16, {}), (16, {"max_kv": 512}), (40, {"max_kv": 512})])
def test_wide_trees_error_does_not_grow_with_the_length(dev, dtype, n, D, T, kw):
    """As test_kv4_accuracy has it, a norm over the output's, of 8 T columns that all see everything. Beside the output's one
    rounding, fp16's 2^-11 is 2^-11 / sqrt(3) = 2.8e-4 in the square's mean. bf16 models: of p, of V' and, in a score, of
    K' (sqrt(D) terms of |q| 1.5 and |k| 1 at a scale of D^-1/2: 4.2e-4 of p), together 5.8e-4. fp16 models: of p s (c - 7.5),
    whose square's mean is below 1.1 times a value's variance, 3e-4; of the range's middle and of the sum that divides it,
    twice of less than a third of a value, 1.3e-4; sums 1.5e-4 (test_kv4_accuracy): 3.6e-4."""
    from test_kv4_accuracy import _case
    for scale in (0.0, 1.5):
        cache, table, cu, seq, q, want = _case(dev, dtype, n, D, 8, T, scale)
        tree = _kv4().KV4Tree(torch.full((T, 2), -1, dtype=torch.int32, device=dev), torch.zeros(T, dtype=torch.int32, device=dev))
        out = _kv4().kv4_attention(q, cache, table, cu, seq, tree=tree, **kw).double()
        norm = want.norm().item()
        rounding = ((want.to(dtype).double() - want).norm() / norm).item()
        err = ((out - want).norm() / norm).item()
        extra = 5.8e-4 if dtype == torch.bfloat16 else 3.6e-4
        print(f"{dtype} n={n} D={D} T={T} {kw} q={scale}: {err:.3e} rounding {rounding:.3e}", flush=True)
        assert err <= math.hypot(rounding, extra), f"{err:.3e}, of which the rounding is {rounding:.3e} (queries of {scale})"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,H,G,page,B", [(128, 2, 5, 16, 70), (64, 1, 7, 2048, 64), (128, 1, 32, 128, 3)])
def test_wide_trees_many_sequences_and_strides(dev, dtype, D, H, G, page, B):
    """More sequences than are put in order, and as many; heads that divide nothing; pages shorter and longer than tiles; q and
    out as columns of wider rows."""
    rng = random.Random(B)
    news = [rng.choice((0, 1, 5, 14, 20)) for _ in range(B)]
    lens = [n + rng.choice((0, 0, 3, 60, 64, 200, 700)) for n in news]
    s = Setup(dev, dtype, D, H, page, lens, news, seed=B)
    trees = [random_tree(n, rng) for n in news]
    see = [x for t in trees for x in lines(t)]
    parents = torch.tensor([p for t in trees for p in t], dtype=torch.int32, device=dev)
    tree = _kv4().kv4_tree(parents, s.d_cu, s.d_seq, max_q=20)
    q = s.q(H * G)
    out = check(s, q, tree, see, max_q=20, max_kv=max(520, max(lens)))
    T = sum(news)
    wide = torch.zeros(T, (H * G + 3) * D + 16, dtype=dtype, device=dev)
    mine = wide[:, 8:8 + H * G * D].view(T, H * G, D)
    mine.copy_(q)
    to = torch.full((T, 2 * H * G, D + 8), 5.0, dtype=dtype, device=dev)
    _kv4().kv4_attention(mine, s.cache, s.d_table, s.d_cu, s.d_seq, tree=tree, max_q=20, max_kv=max(520, max(lens)), out=to[:, ::2, :D])
    assert torch.equal(to[:, ::2, :D], out)
    assert (to[:, 1::2] == 5).all() and (to[:, :, D:] == 5).all()


@pytest.mark.gpu
def test_wide_trees_past_4_gib(dev):
    """The same bits from pages whose codes lie past 32 bits."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GiB")
    lens, news = [700, 90], [40, 33]
    s = Setup(dev, torch.bfloat16, 128, 8, 64, lens, news, seed=6)
    tree = _kv4().kv4_tree(torch.tensor([i - 1 for n in news for i in range(n)], dtype=torch.int32, device=dev), s.d_cu, s.d_seq, max_q=40)
    q = s.q(32)
    want = s.attend(q, tree=tree, max_q=40, max_kv=700)
    pages, bytes_ = 140000, 8 * 64 * 64
    far = _kv4().KV4Cache(pages, 64, 8, 128, torch.bfloat16, dev)
    table = pages - 1 - s.table
    assert int(table[:, :2].min()) * bytes_ > 1 << 32
    table = table.int().to(dev)
    _kv4().kv4_append(far, s.k.to(dev), s.v.to(dev), table, s.cu_all.to(dev), s.d_seq)
    got = _kv4().kv4_attention(q.to(dev), far, table, s.d_cu, s.d_seq, tree=tree, max_q=40, max_kv=700)
    assert torch.equal(got, want)
