"""Attention over whole prompts (layers/attention.py prompt_attention): refusals on the CPU, and on the GPU against
64-bit attention.

Tolerances, per output element, with h half a step of the type (2^-8 bf16, 2^-11 fp16), o the output and
A = sum p |v| / sum p:
  - the output is rounded: h |o|, and 2^-25 for fp16's subnormals;
  - p is rounded to the type before its product, and so is its sum or it is not: h (A + |o|) at most;
  - a score is an f32 sum of D products of the types' exact values; the matrix unit may cut where it does not round, so
    2^-23 per step of its sum and per its rounding into exp2's argument: d = (D + 8) 2^-23 max|q||k| scale + 2^-20 for
    M, the argument and exp2 itself. It moves p by d of itself, and o by 2 d A;
  - sums of p and of p v over n keys in f32: n 2^-23 (A + |o|) at the very most; the matrix unit adds 16 at a time and
    64-key parts, so (n / 8 + 16) 2^-23.
Rows without keys are 0 exactly, their lse -inf; lse is off by d, the sum's error and its own f32 rounding, 2^-22 |lse|
(a p in fp16 below 2^-14 is within 2^-25 of a sum that is at least 2^-8, and counted with A: 2^-17 A for fp16)."""
import math

import pytest
import torch

from conftest import pkg

DTYPES = [torch.bfloat16, torch.float16]


def _att():
    return pkg("layers.attention")


def _i32(dev, *a):
    return torch.tensor(a, dtype=torch.int32, device=dev)


def ref(q, k, v, cu, scale, causal=True, window=0):
    """out, A, lse and d's factor max|q||k| scale, in f64 on the CPU."""
    q, k, v = (t.cpu().double() for t in (q, k, v))
    T, Hq, D = q.shape
    G = Hq // k.shape[1]
    out, A = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64)
    most = torch.zeros(T, Hq, dtype=torch.float64)
    for a, b in zip(cu[:-1], cu[1:]):
        n = b - a
        if n <= 0:
            continue
        i, j = torch.arange(n).unsqueeze(1), torch.arange(n)
        see = j <= i if causal else torch.ones(n, n, dtype=torch.bool)
        if window:
            see = see & (j > i - window)
        for h in range(Hq):
            x = q[a:b, h] @ k[a:b, h // G].t() * scale
            most[a:b, h] = (q[a:b, h].abs() @ k[a:b, h // G].abs().t() * scale).where(see, 0.0).amax(1)
            x = x.masked_fill(~see, -math.inf)
            lse[a:b, h] = torch.logsumexp(x, 1)
            p = torch.softmax(x, 1).masked_fill(~see, 0.0)
            out[a:b, h], A[a:b, h] = p @ v[a:b, h // G], p @ v[a:b, h // G].abs()
    return out, A, lse, most


def compare(got, lse, want, dtype, D, n):
    out, A, rl, most = want
    h = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    d = ((D + 8) * 2.0 ** -23 * most + 2.0 ** -20).unsqueeze(-1)
    tol = h * out.abs() + (h + (n / 8 + 16) * 2.0 ** -23) * (A + out.abs()) + 2 * d * A
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25 + 2.0 ** -17 * A
    err = (got.cpu().double() - out).abs() - tol
    assert err.numel() == 0 or err.max().item() <= 0, f"off by {err.max().item():.3e} past the tolerance"
    if lse is not None:
        lse = lse.cpu().double()
        seen = torch.isfinite(rl)
        assert torch.equal(torch.isfinite(lse), seen)
        t = d.squeeze(-1) + h + (n / 8 + 16) * 2.0 ** -23 + 2.0 ** -22 * rl.abs()
        assert ((lse - rl).abs() - t)[seen].max().item() <= 0 if seen.any() else True


def make(T, Hq, H, D, dtype, dev, seed=0, scale=1.0):
    """q, k and v as a merged projection's output has them."""
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(T, (Hq + 2 * H) * D, generator=g)
    qkv[:, Hq * D:(Hq + H) * D] += torch.randn(H * D, generator=g) * (torch.rand(H * D, generator=g) < 0.05) * 4
    qkv = (qkv * scale).to(dtype).to(dev)
    return tuple(t.view(T, -1, D) for t in qkv.split([Hq * D, H * D, H * D], dim=1))


# ------------------------------------------------------------------------------------------------
# CPU: refusals
# ------------------------------------------------------------------------------------------------
def test_refusals():
    att = _att()
    x = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    cu = torch.tensor([0, 2], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="on the GPU"):
        att.prompt_attention(x(2, 2, 64), x(2, 1, 64), x(2, 1, 64), cu)
    for q in (x(2, 2, 96), x(2, 128), x(2, 2, 64).float()):
        with pytest.raises(TypeError, match="q must be"):
            att.prompt_attention(q, x(2, 1, 64), x(2, 1, 64), cu)


def test_abi_refusals():
    """Host checks of the C entry point, with pointers that are never read."""
    if torch.cuda.is_available():
        pytest.skip("the pointers are not real")
    lib = pkg("_abi").load()
    P = 1 << 20
    far = 1 << 40

    def call(dtype=0, T=4, Hq=4, H=2, D=64, cu=P, B=1, scale=1.0, window=0, max_q=4, q=P, k=far, v=2 * far, out=4 * far, ldq=256,
             hq=64, ldk=128, hk=64, ldo=256, ho=64):
        rc = lib.w4a8_prompt_attention(q, ldq, hq, k, ldk, hk, v, 128, 64, dtype, T, Hq, H, D, cu, B, scale, 1, window, max_q, out,
                                       ldo, ho, None, None)
        return rc, lib.w4a8_last_error().decode()

    for kw, code, what in ((dict(dtype=2), 1, "bf16 or fp16"), (dict(D=96), 2, "64, 128 or 256"), (dict(Hq=3), 1, "query heads"),
                           (dict(Hq=65536, H=1), 1, "query heads"), (dict(scale=0.0), 1, "scale"), (dict(scale=65536.0), 1, "scale"),
                           (dict(scale=float("nan")), 1, "scale"), (dict(window=-1), 1, "window"), (dict(max_q=-1), 1, "max_q"),
                           (dict(B=65536), 2, "index ranges"), (dict(T=1 << 28), 2, "index ranges"), (dict(cu=None), 1, "cu"),
                           (dict(q=P + 2), 1, "16-byte"), (dict(ldq=260), 1, "multiples of 8"), (dict(ldk=56), 2, "apart"),
                           (dict(ldk=1 << 23), 2, "apart"), (dict(ldo=128), 1, "overlap"), (dict(out=P + 64), 1, "overlaps q"),
                           (dict(out=far), 1, "overlaps k or v"), (dict(out=2 * far - 64), 1, "overlaps k or v"),
                           (dict(q=far, out=far, ldq=512, ldo=512, k=far + 4 * 64, ldk=512), 1, "overlaps k or v")):
        rc, msg = call(**kw)
        assert rc == code and what in msg, (kw, rc, msg)
    assert call(T=0)[0] == 0 and call(B=0)[0] == 0


# ------------------------------------------------------------------------------------------------
# GPU
# ------------------------------------------------------------------------------------------------
LENS = [0, 1, 63, 0, 64, 65, 257, 2, 130, 31]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,H,G", [(64, 2, 3), (128, 2, 4), (256, 1, 2), (128, 1, 1), (64, 1, 16), (128, 1, 5), (256, 2, 1), (64, 1, 300)])
def test_packed(dev, dtype, D, H, G):
    lens = LENS if G < 100 else [5, 0, 33]
    cu = [sum(lens[:i]) for i in range(len(lens) + 1)]
    q, k, v = make(cu[-1], H * G, H, D, dtype, dev, seed=D + G)
    for kw in (dict(), dict(window=1), dict(window=17), dict(window=100, max_q=max(lens)), dict(causal=False), dict(causal=False, window=40),
               dict(sm_scale=0.5, max_q=7)):
        out, lse = _att().prompt_attention(q, k, v, _i32(dev, *cu), return_lse=True, **kw)
        want = ref(q, k, v, cu, kw.get("sm_scale", D ** -0.5), kw.get("causal", True), kw.get("window", 0))
        compare(out, lse, want, dtype, D, max(lens))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,n,window", [(128, 1537, 0), (64, 2000, 0), (128, 1200, 511), (256, 700, 0)])
def test_long(dev, dtype, D, n, window):
    q, k, v = make(n, 4, 2, D, dtype, dev, seed=n)
    out, lse = _att().prompt_attention(q, k, v, _i32(dev, 0, n), window=window, return_lse=True)
    compare(out, lse, ref(q, k, v, [0, n], D ** -0.5, True, window), dtype, D, n)
    # a row's bits follow from the rows that it sees: of a prompt that is cut they are the same
    cut = n * 2 // 3
    again = _att().prompt_attention(q[:cut], k[:cut], v[:cut], _i32(dev, 0, cut), window=window)
    assert torch.equal(again, out[:cut])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_of_any_size(dev, dtype):
    """One score above all others, growing ones that raise the maximum in every tile, and scores past 2^24."""
    n, D = 300, 64
    q, k, v = make(n, 2, 1, D, dtype, dev, seed=3)
    ramp = torch.arange(n, device=dev).view(n, 1, 1) / 8
    for kk, qq in ((k * ramp.to(dtype), q.abs() + 1), (-(k.abs()) * ramp.to(dtype), q.abs())):
        out, lse = _att().prompt_attention(qq, kk.contiguous(), v, _i32(dev, 0, n), return_lse=True)
        compare(out, lse, ref(qq, kk, v, [0, n], D ** -0.5), dtype, D, n)
    # whole numbers times powers of two: scores are exact, some past 2^24, and those that are equal share a row evenly
    g = torch.Generator().manual_seed(5)
    big = 2.0 ** 14 if dtype == torch.bfloat16 else 2.0 ** 10
    qi = (torch.randint(-2, 3, (n, 2, D), generator=g).double() * big).to(dtype).to(dev)
    ki = (torch.randint(-2, 3, (n, 1, D), generator=g).double() * big).to(dtype).to(dev)
    out, lse = _att().prompt_attention(qi, ki, v, _i32(dev, 0, n), sm_scale=1.0, return_lse=True)
    want = ref(qi, ki, v, [0, n], 1.0)
    want = (*want[:3], torch.zeros_like(want[3]))
    compare(out, None, want, dtype, D, n)
    assert ((lse.cpu().double() - want[2]).abs() <= 2.0 ** -22 * want[2].abs() + 2.0 ** -7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("below", [13.5, 15.25, 18.0, 23.0])
def test_many_small_weights(dev, dtype, below):
    """One key before thousands that weigh 2^-below of it each, subnormal in fp16: together they weigh what they should, in
    the products and in the sum. In fp16 a weight below 2^-14 is off by up to 2^-25, of what n such weights are among 1."""
    n, D = 3001, 64
    q, k, v = (t.clone() for t in make(n, 1, 1, D, dtype, dev, seed=6))
    q.zero_()
    k.zero_()
    q[:, 0, 0] = 1
    k[1:, 0, 0] = -below * math.log(2)
    k[1:, 0, 1] = -below * math.log(2) - k[1:, 0, 0].float()  # what the type rounds away
    q[:, 0, 1] = 1
    v[1:] = v[1:].abs()
    out, lse = _att().prompt_attention(q, k, v, _i32(dev, 0, n), sm_scale=1.0, return_lse=True)
    want = ref(q, k, v, [0, n], 1.0)
    sub = n * 2.0 ** -25 if dtype == torch.float16 else 0.0
    most = v.float().abs().max().item()
    compare(out, None, (want[0], want[1] + 2 * sub * most * 2.0 ** 11, want[2], want[3]), dtype, D, n)
    assert ((lse.cpu().double() - want[2]).abs() <= sub + (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11) + n * 2.0 ** -26).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("at", [0, 5, 63, 64, 100])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_what_is_not_finite_stays_with_who_sees_it(dev, dtype, bad, at, D):
    n, ch = 150, 7
    q, k, v = (t.clone() for t in make(n, 2, 1, D, dtype, dev, seed=at))
    clean = _att().prompt_attention(q, k, v, _i32(dev, 0, n))
    v2 = v.clone()
    v2[at, 0, ch] = bad
    for window in (0, 20):
        base = clean if not window else _att().prompt_attention(q, k, v, _i32(dev, 0, n), window=window)
        out = _att().prompt_attention(q, k, v2, _i32(dev, 0, n), window=window)
        i = torch.arange(n, device=dev)
        sees = (i >= at) & ((i < at + window) if window else torch.ones_like(i, dtype=torch.bool))
        assert not torch.isfinite(out[sees][:, :, ch]).any()
        rest = torch.ones(D, dtype=torch.bool, device=dev)
        rest[ch] = False
        assert torch.equal(out[:, :, rest], base[:, :, rest]) and torch.equal(out[~sees], base[~sees])
    # and in a key: the row is NaN (a -inf score may be a key that weighs nothing)
    k2 = k.clone()
    k2[at, 0, ch] = math.nan
    out = _att().prompt_attention(q, k2, v, _i32(dev, 0, n))
    assert torch.isnan(out[at:]).all() and torch.equal(out[:at], clean[:at])
    # neighbours in the pack, and rows behind the last sequence, see nothing of it
    out = torch.full_like(q, 3.0)
    _att().prompt_attention(q, k2, v2, _i32(dev, 0, at, at + 1, n - 2), out=out)
    assert torch.equal(out[:at], clean[:at]) and torch.isfinite(out[at + 1:].float()).all() and (out[n - 2:] == 3).all()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
def test_layouts_and_outputs(dev, D):
    T, Hq, H, cu = 200, 6, 2, [3, 90, 90, 197]
    q, k, v = make(T, Hq, H, D, torch.bfloat16, dev, seed=1)
    c = _i32(dev, *cu)
    want = _att().prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), c)[3:197]
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(_att().prompt_attention(*heads_first, c)[3:197], want)
    odd = [torch.cat([t, t], -1)[:, :, 4:D + 4] for t in (torch.roll(t, 4, -1) for t in (q, k, v))]  # off 16 bytes: copied
    assert torch.equal(_att().prompt_attention(*odd, c)[3:197], want)
    wide = torch.full((T, 2 * Hq, D), 7.0, dtype=q.dtype, device=dev)
    got = _att().prompt_attention(q, k, v, c, out=wide[:, ::2])
    assert got.data_ptr() == wide.data_ptr() and torch.equal(got[3:197], want)
    assert (wide[:, 1::2] == 7).all() and (wide[:3] == 7).all() and (wide[197:] == 7).all()
    inplace = q.clone()
    assert torch.equal(_att().prompt_attention(inplace, k, v, c, out=inplace)[3:197], want) and torch.equal(inplace[:3], q[:3])
    # in place within a merged projection's output
    qkv = torch.cat([q.reshape(T, -1), k.reshape(T, -1), v.reshape(T, -1)], 1)
    qv, kv, vv = (t.view(T, -1, D) for t in qkv.split([Hq * D, H * D, H * D], 1))
    _att().prompt_attention(qv, kv, vv, c, out=qv)
    assert torch.equal(qv[3:197], want) and torch.equal(kv, k) and torch.equal(vv, v)
    # one key and value row for all tokens, by a stride of 0
    same = k[:1].expand(T, H, D), v[:1].expand(T, H, D)
    got = _att().prompt_attention(q, *same, c)[3:197]
    full = _att().prompt_attention(q, *(t.contiguous() for t in same), c)[3:197]
    assert torch.equal(got, full)


@pytest.mark.gpu
def test_gpu_refusals(dev):
    att = _att()
    q, k, v = make(8, 4, 2, 64, torch.bfloat16, dev)
    cu = _i32(dev, 0, 8)
    for args, kw, e in (((q, k.half(), v, cu), {}, TypeError), ((q, k[:7], v, cu), {}, TypeError), ((q, k, v[:, :1], cu), {}, TypeError),
                        ((q[:, :3], k, v, cu), {}, ValueError), ((q, k, v, cu.long()), {}, TypeError), ((q, k, v, cu.cpu()), {}, RuntimeError),
                        ((q, k.cpu(), v, cu), {}, RuntimeError), ((q, k, v, cu), dict(window=-1), ValueError),
                        ((q, k, v, cu), dict(max_q=-1), ValueError), ((q, k, v, cu), dict(out=torch.empty_like(k)), ValueError),
                        ((q, k, v, cu), dict(sm_scale=-1.0), RuntimeError),
                        ((q, k, v, cu), dict(out=q[:1].expand(8, 4, 64)), RuntimeError),
                        ((q[:, :2], k, v, cu), dict(out=k), RuntimeError), ((q[:, :2], k, v, cu), dict(out=v), RuntimeError),
                        ((q[:, :2], k, v, cu), dict(out=q[:, 1:3]), RuntimeError)):
        with pytest.raises(e):
            att.prompt_attention(*args, **kw)
    assert att.prompt_attention(q[:0], k[:0], v[:0], _i32(dev, 0)).shape == (0, 4, 64)
    out, lse = att.prompt_attention(q[:0], k[:0], v[:0], _i32(dev, 0, 0, 0), return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)


@pytest.mark.gpu
def test_captured_and_on_other_streams(dev):
    """A captured call replays with other rows and other sequences; two streams at once share nothing."""
    T, D = 400, 128
    q, k, v = (t.clone() for t in make(T, 8, 2, D, torch.bfloat16, dev))
    cu = _i32(dev, 0, 100, 400, 400)
    out = torch.zeros_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _att().prompt_attention(q, k, v, cu, out=out)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _att().prompt_attention(q, k, v, cu, out=out)
    for rep, lens in enumerate([(0, 400, 0), (1, 2, 300), (0, 0, 0), (133, 133, 134)]):
        cu.copy_(_i32(dev, 0, *[sum(lens[:i + 1]) for i in range(3)]))
        for t in (q, k, v):
            t.normal_()
        out.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        eager = torch.full_like(out, 5.0)
        _att().prompt_attention(q, k, v, cu, out=eager)
        assert torch.equal(got, eager), rep
        assert (got[sum(lens):] == 5).all()
    want = [_att().prompt_attention(q, k, v, cu, window=w) for w in (0, 9)]
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    got = []
    for s, w in ((side, 0), (other, 9)):
        with torch.cuda.stream(s):
            got.append(_att().prompt_attention(q, k, v, cu, window=w))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_rows_past_4_gib(dev):
    """A short prompt whose rows lie far behind the tensors' beginning, and rows of k and v far from each other."""
    D, ld = 64, 1 << 16
    T = 33000  # 4.3 GB
    buf = torch.zeros(T, ld, dtype=torch.bfloat16, device=dev)
    x = make(120, 2, 1, D, torch.bfloat16, dev, seed=8)
    a = T - 125
    q, k, v = buf[:, :2 * D].view(T, 2, D), buf[:, 2 * D:3 * D].view(T, 1, D), buf[:, ld - D:].view(T, 1, D)
    for dst, src in zip((q, k, v), x):
        dst[a:a + 120] = src
    out = buf[:, 3 * D:5 * D].view(T, 2, D)
    _att().prompt_attention(q, k, v, _i32(dev, a, a + 120), out=out, max_q=120)
    want = _att().prompt_attention(*x, _i32(dev, 0, 120))
    assert torch.equal(out[a:a + 120], want) and not out[:a].any() and not out[a + 120:].any()
