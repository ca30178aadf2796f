"""Rotary positions (layers/rotary.py): refusals on the CPU, and on the GPU against the formula in 64 bits.

Tolerance per output element a' = s (a cos t - b sin t): one rounding to the type, h |a'| with h half a step (2^-8 bf16,
2^-11 fp16; 2^-25 for fp16's subnormals), and before it |s| (|a| + |b|) times what cos and sin are off by: 2^-32 of a turn
of the cut angle, pi/4 2^-24 of its conversion to f32, 2^-24 of the factor's rounding, of the polynomial's coefficients and
steps within 5 2^-24, and the scale's product and the two products and the sum 4 2^-24: 2^-20 in all. The test's own
angle, an f64 product, is off by 2^-53 of itself, as is a frequency over 2 pi in 64 bits: 2^-51 |t| each side."""
import math

import pytest
import torch

from conftest import pkg

DTYPES = [torch.bfloat16, torch.float16]


def _rotary(*a, **kw):
    return pkg("layers.rotary").Rotary(*a, **kw)


def want(x, pos, freq, axis, R, adjacent, scale):
    """x (T, heads, D), pos (axes, T) -> turned in f64, and the tolerance without the final rounding."""
    x = x.cpu().double()
    t = pos.cpu().double()[axis].t().unsqueeze(1) * freq
    c, s = torch.cos(t) * scale, torch.sin(t) * scale
    r = x[..., :R]
    a, b = (r[..., 0::2], r[..., 1::2]) if adjacent else (r[..., :R // 2], r[..., R // 2:])
    u, v = a * c - b * s, a * s + b * c
    tol = (a.abs() + b.abs()) * abs(scale) * (2.0 ** -20 + 2.0 ** -50 * t.abs())
    put = (lambda p, q: torch.stack([p, q], -1).flatten(-2)) if adjacent else (lambda p, q: torch.cat([p, q], -1))
    return torch.cat([put(u, v), x[..., R:]], -1), torch.cat([put(tol, tol), torch.zeros_like(x[..., R:])], -1)


def check(got, x, pos, freq, axis, R, adjacent, scale):
    ref, tol = want(x, pos, freq, axis, R, adjacent, scale)
    h = 2.0 ** (-8 if x.dtype == torch.bfloat16 else -11)
    err = (got.cpu().double() - ref).abs() - h * ref.abs() - tol - 2.0 ** -25
    assert err.numel() == 0 or err.max().item() <= 0, f"off by {err.max().item():.3e} past the tolerance"
    assert torch.equal(got[..., R:], x[..., R:])


def freqs(base, R):
    return base ** (torch.arange(R // 2, dtype=torch.float64) * (-2.0 / R))


# ------------------------------------------------------------------------------------------------
# CPU
# ------------------------------------------------------------------------------------------------
def test_refusals():
    for kw in (dict(head_dim=12), dict(head_dim=1032), dict(head_dim=64, rotary_dim=24), dict(head_dim=64, rotary_dim=80),
               dict(head_dim=64, rotary_dim=0), dict(head_dim=64, base=0.0), dict(head_dim=64, sections=(8, 8, 8)),
               dict(head_dim=64, sections=(40, -8)), dict(head_dim=64, sections=(8, 16, 8), interleaved=True),
               dict(head_dim=64, inv_freq=[1.0] * 31), dict(head_dim=64, inv_freq=[math.inf] * 32),
               dict(head_dim=64, scale=math.nan), dict(head_dim=64, sections=(4,) * 9)):
        with pytest.raises(ValueError, match="Rotary"):
            _rotary(kw.pop("head_dim"), device="cpu", **kw)
    r = _rotary(64, device="cpu")
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    pos = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="one GPU"):
        r.forward(x, x, pos)
    for q, k, p in ((x.float(), x.float(), pos), (x, x.half(), pos), (x, x[:2], pos), (x[..., :32], x, pos), (x, x, pos.float()),
                    (x, x, pos[:2]), (x, x, pos.expand(2, 3)), (x[:, 0], x, pos), (x, x[:, :0], pos)):
        with pytest.raises(TypeError):
            r.forward(q, k, p)


def test_plan():
    """Turns are the frequencies over 2 pi, modulo 1, in 2^-64; pairs go to their axes."""
    r = _rotary(128, base=1e6, sections=(16, 24, 24), device="cpu")
    f = freqs(1e6, 128) / (2 * math.pi)
    turns = torch.tensor([t % 2 ** 64 for t in r.turns.tolist()], dtype=torch.float64) / 2.0 ** 64
    assert (turns - f).abs().max().item() <= 2.0 ** -53
    assert r.axis.tolist() == [0] * 16 + [1] * 24 + [2] * 24
    assert _rotary(64, sections=(12, 10, 10), interleaved=True, device="cpu").axis.tolist() == [0, 1, 2] * 10 + [0, 0]
    assert _rotary(64, sections=(20, 6, 6), interleaved=True, device="cpu").axis.tolist() == [0, 1, 2] * 6 + [0] * 14
    back = _rotary(32, inv_freq=[-0.25] * 16, device="cpu").turns.tolist()
    there = _rotary(32, inv_freq=[0.25] * 16, device="cpu").turns.tolist()
    assert all((a + b) % 2 ** 64 == 0 for a, b in zip(back, there))


def test_abi_refusals():
    if torch.cuda.is_available():
        pytest.skip("the pointers are not real")
    lib = pkg("_abi").load()
    P, F = 1 << 20, 1 << 40

    def call(dtype=0, T=4, Hq=2, Hk=1, D=64, R=64, q=P, qo=2 * F, k=F, ko=3 * F, ldq=128, hq=64, ldqo=128, hqo=64, pos=P, turns=P, axes=1,
             axis=None):
        rc = lib.w4a8_rotary(q, ldq, hq, Hq, k, 64, 64, Hk, dtype, T, D, R, 0, pos, 0, axes, T, turns, axis, 1.0, qo, ldqo, hqo, ko,
                             64, 64, None)
        return rc, lib.w4a8_last_error().decode()

    for kw, code, what in ((dict(dtype=2), 1, "bf16 or fp16"), (dict(D=60), 2, "channels"), (dict(R=24), 2, "channels"),
                           (dict(R=80), 2, "channels"), (dict(Hq=0), 1, "heads"), (dict(axes=9, axis=P), 1, "axes"), (dict(axes=2), 1, "axes"),
                           (dict(pos=None), 1, "positions"), (dict(turns=None), 1, "turns"), (dict(q=P + 8), 1, "16-byte"),
                           (dict(ldq=132), 1, "multiples of 8"), (dict(ldqo=64), 1, "overlap"), (dict(qo=P + 64), 1, "without being it"),
                           (dict(ko=2 * F), 1, "q and k overlap"), (dict(qo=F), 1, "q and k overlap"), (dict(ko=P), 1, "q and k overlap")):
        rc, msg = call(**kw)
        assert rc == code and what in msg, (kw, rc, msg)
    assert call(T=0)[0] == 0


# ------------------------------------------------------------------------------------------------
# GPU
# ------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,R,Hq,Hk", [(128, 128, 8, 2), (64, 64, 3, 3), (256, 128, 4, 1), (80, 48, 5, 1), (1024, 1024, 1, 1), (16, 16, 32, 8),
                                       (96, 96, 33, 7)])
@pytest.mark.parametrize("T", [1, 3, 70])
@pytest.mark.parametrize("adjacent", [False, True])
def test_one_axis(dev, dtype, D, R, Hq, Hk, T, adjacent):
    g = torch.Generator().manual_seed(D + T)
    qkv = torch.randn(T, (Hq + 2 * Hk) * D, generator=g).to(dtype).to(dev)
    q, k = (t.view(T, -1, D) for t in qkv.split([Hq * D, Hk * D, Hk * D], 1)[:2])
    pos = torch.randint(0, 1 << 20, (T,), generator=g)
    f = freqs(5e5, R)
    axis = torch.zeros(R // 2, dtype=torch.long)
    for scale, p in ((1.0, pos.int()), (1.25, pos)):
        r = _rotary(D, base=5e5, rotary_dim=R, adjacent=adjacent, scale=scale, device=dev)
        qo, ko = r.forward(q, k, p.to(dev))
        assert qo.is_contiguous() and ko.is_contiguous()
        check(qo, q, pos.view(1, T), f, axis, R, adjacent, scale)
        check(ko, k, pos.view(1, T), f, axis, R, adjacent, scale)
    held = qkv.clone()
    qi, ki = (t.view(T, -1, D) for t in held.split([Hq * D, Hk * D, Hk * D], 1)[:2])
    r.forward_inplace(qi, ki, pos.to(dev))
    assert torch.equal(qi, qo) and torch.equal(ki, ko) and torch.equal(held[:, (Hq + Hk) * D:], qkv[:, (Hq + Hk) * D:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sections,interleaved", [((16, 24, 24), False), ((24, 20, 20), True), ((32, 32), False), ((0, 64), False), ((8,) * 8, True)])
def test_several_axes(dev, dtype, sections, interleaved):
    T, D = 37, 128
    g = torch.Generator().manual_seed(len(sections))
    q, k = torch.randn(T, 4, D, generator=g).to(dtype).to(dev), torch.randn(T, 2, D, generator=g).to(dtype).to(dev)
    pos = torch.randint(0, 5000, (len(sections), T), generator=g, dtype=torch.int32)
    r = _rotary(D, base=1e4, sections=sections, interleaved=interleaved, device=dev)
    for a, b in zip(r.forward(q, k, pos.to(dev)), (q, k)):
        check(a, b, pos, freqs(1e4, D), r.axis.cpu().long(), D, False, 1.0)
    # positions as rows of a longer buffer
    wide = torch.zeros(len(sections), 50, dtype=torch.int32, device=dev)
    wide[:, 5:42] = pos.to(dev)
    assert torch.equal(r.forward(q, k, wide[:, 5:42])[0], r.forward(q, k, pos.to(dev))[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_any_position(dev, dtype):
    """Far, negative and 64-bit positions: angles in f64 are good to 2^-20 up to 2^31, and beyond that whole turns tell."""
    T, D = 64, 64
    g = torch.Generator().manual_seed(2)
    q = torch.randn(T, 2, D, generator=g).to(dtype).to(dev)
    pos = torch.cat([torch.randint(-2 ** 31, 2 ** 31, (T - 3,), generator=g), torch.tensor([2 ** 31 - 1, -2 ** 31, 0])])
    r = _rotary(D, device=dev)
    out = r.forward(q, q, pos.int().to(dev))
    check(out[0], q, pos.view(1, T), freqs(1e4, D), torch.zeros(D // 2, dtype=torch.long), D, False, 1.0)
    assert torch.equal(out[0], out[1]) and torch.equal(out[0], r.forward(q, q, pos.to(dev))[0])
    # a frequency of 2 pi / 2^20: 2^20 positions are a turn
    whole = _rotary(D, inv_freq=[2 * math.pi / 2 ** 20] * (D // 2), device=dev)
    p = torch.arange(T).to(dev)
    assert torch.equal(whole.forward(q, q, p)[0], whole.forward(q, q, p + (2 ** 20) * 12345)[0])


@pytest.mark.gpu
def test_layouts_refusals_and_empty(dev):
    T, D = 9, 64
    x = torch.randn(T, 6, D, device=dev).to(torch.bfloat16)
    pos = torch.arange(T, dtype=torch.int32, device=dev)
    r = _rotary(D, device=dev)
    q, k = r.forward(x[:, :4].contiguous(), x[:, 4:].contiguous(), pos)
    assert torch.equal(r.forward(x[:, :4], x[:, 4:], pos)[0], q)
    first = x.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(r.forward(first[:, :4], first[:, 4:], pos)[1], k)
    odd = torch.zeros(T, 6, D + 4, dtype=x.dtype, device=dev)
    odd[:, :, 2:D + 2] = x
    odd = odd[:, :, 2:D + 2]
    assert torch.equal(r.forward(odd[:, :4], odd[:, 4:], pos)[0], q)
    with pytest.raises(ValueError, match="in place"):
        r.forward_inplace(odd[:, :4], odd[:, 4:], pos)
    with pytest.raises(RuntimeError, match="overlap"):
        r.forward_inplace(x[:, :4], x[:, 3:], pos)
    with pytest.raises(RuntimeError, match="overlap"):
        r.forward_inplace(x[:, :1].expand(T, 4, D), x[:, 4:], pos)
    with pytest.raises(RuntimeError, match="one GPU"):
        r.forward(x, x, pos.cpu())
    with pytest.raises(RuntimeError, match="one GPU"):
        _rotary(D, device="cpu").forward(x, x, pos)
    a, b = r.forward(x[:0], x[:0], pos[:0])
    assert a.shape == b.shape == (0, 6, D)
    nan = x.clone()
    nan[2, 1, 5] = math.nan
    out = r.forward(nan, x, pos)[0]
    bad = torch.isnan(out)
    assert bad.sum().item() == 2 and bad[2, 1, 5] and bad[2, 1, 5 + D // 2]


@pytest.mark.gpu
def test_captured(dev):
    T, D = 5, 128
    x = torch.randn(T, 6, D, device=dev).to(torch.bfloat16)
    pos = torch.arange(T, dtype=torch.int32, device=dev)
    r = _rotary(D, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        r.forward(x[:, :4], x[:, 4:], pos)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = r.forward(x[:, :4], x[:, 4:], pos)
    for rep in range(4):
        x.normal_()
        pos.random_(0, 100000)
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in got]
        assert all(torch.equal(a, b) for a, b in zip(kept, r.forward(x[:, :4], x[:, 4:], pos))), rep


@pytest.mark.gpu
def test_rows_past_4_gib(dev):
    """Rows behind the first 2^32 bytes of their tensor."""
    D, ld, T = 64, 1 << 16, 33000
    buf = torch.zeros(T, ld, dtype=torch.bfloat16, device=dev)
    x = torch.randn(4, 3, D, device=dev).to(torch.bfloat16)
    q, k = buf[:, :2 * D].view(T, 2, D), buf[:, ld - D:].view(T, 1, D)
    q[-4:], k[-4:] = x[:, :2], x[:, 2:]
    pos = torch.arange(T, dtype=torch.int32, device=dev)
    r = _rotary(D, device=dev)
    r.forward_inplace(q, k, pos)
    a, b = r.forward(x[:, :2], x[:, 2:], pos[-4:])
    assert torch.equal(q[-4:], a) and torch.equal(k[-4:], b) and not q[:-4].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("adjacent,rotary_dim", [(False, 128), (True, 128), (False, 64)])
def test_many_rows_as_few(dev, dtype, adjacent, rotary_dim):
    """More rows than the caches hold, that take the way past them: the bits of the same rows a few at a time, in place too."""
    T, Hq, H, D = 1801, 37, 5, 128
    assert T * (Hq + H) * D * 4 > 32 << 20
    g = torch.Generator(device=dev).manual_seed(1)
    qkv = torch.randn(T, (Hq + 2 * H) * D, generator=g, device=dev).to(dtype)
    q, k, v = (t.view(T, -1, D) for t in qkv.split([Hq * D, H * D, H * D], dim=1))
    pos = torch.randint(0, 1 << 20, (T,), generator=g, device=dev)
    rot = pkg("layers.rotary").Rotary(D, rotary_dim=rotary_dim, adjacent=adjacent, scale=1.25, device=dev)
    want = [rot.forward(q[i:i + 100], k[i:i + 100], pos[i:i + 100]) for i in range(0, T, 100)]
    want = tuple(torch.cat(t) for t in zip(*want))
    got = rot.forward(q, k, pos)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    before = v.clone()
    rot.forward_inplace(q, k, pos)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, before)
