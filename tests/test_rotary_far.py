"""Rotary positions far from 0 and of many rows (layers/rotary.py): the fractions of a turn against pi in whole numbers, on the CPU,
and on the GPU 64-bit positions against exact angles, and rows that take the way past the caches against the same rows a few at a time."""
import math
import random
from fractions import Fraction

import pytest
import torch

from conftest import pkg

DTYPES = [torch.bfloat16, torch.float16]
# 200 digits of pi: 2^-660 of itself
PI = Fraction(int("31415926535897932384626433832795028841971693993751058209749445923078164062862089986280348253421170679821480865132823"
                  "066470938446095505822317253594081284811174502841027019385211055596446229489549303819"), 10 ** 199)


def exact_turns(f, position=1):
    """Turns modulo 1."""
    t = Fraction(f) * position / (2 * PI)
    return t - math.floor(t)


def test_turns_are_the_nearest():
    """Frequencies from far below a turn per position to far above one, and below what 2^-64 holds."""
    rng = random.Random(1)
    freqs = [1.0, -1.0, 0.0, 2.0 ** -70, -2.0 ** -64, 1e-12, 6.25, math.pi, 2 * math.pi, 1e15, -12345.678, 2.0 ** 300 + 2.0 ** 250]
    freqs += [rng.choice((-1, 1)) * math.exp(rng.uniform(-30, 10)) for _ in range(52)]
    r = pkg("layers.rotary").Rotary(128, inv_freq=freqs, device="cpu")
    for f, t in zip(freqs, r.turns.tolist()):
        off = abs(Fraction(t % 2 ** 64) - exact_turns(f) * 2 ** 64)
        # half a unit, and what pi itself may be off by
        assert min(off, 2 ** 64 - off) <= Fraction(1, 2) + Fraction(1, 2 ** 30), (f, t, float(off))
    r = pkg("layers.rotary").Rotary(64, base=5e5, device="cpu")
    for i, t in enumerate(r.turns.tolist()):
        assert abs(t % 2 ** 64 - exact_turns(5e5 ** (-2.0 * i / 64)) * 2 ** 64) <= Fraction(1, 2) + Fraction(1, 2 ** 30)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_far_positions(dev, dtype):
    """Positions up to 2^45: as test_rotary has it, with an exact angle and 2 pi |position| 2^-65 in its tolerances' place."""
    T, D = 24, 64
    rng = random.Random(3)
    g = torch.Generator().manual_seed(3)
    q = torch.randn(T, 2, D, generator=g).to(dtype)
    pos = [rng.choice((-1, 1)) * rng.randrange(2 ** 40, 2 ** 45) for _ in range(T - 2)] + [2 ** 45, -2 ** 45]
    freqs = [1e4 ** (-2.0 * i / D) for i in range(D // 2)]
    r = pkg("layers.rotary").Rotary(D, device=dev)
    out = r.forward(q.to(dev), q.to(dev), torch.tensor(pos).to(dev))
    t = torch.tensor([[2 * math.pi * float(exact_turns(f, p)) for f in freqs] for p in pos], dtype=torch.float64).unsqueeze(1)
    x = q.double()
    a, b = x[..., :D // 2], x[..., D // 2:]
    want = torch.cat([a * t.cos() - b * t.sin(), a * t.sin() + b * t.cos()], -1)
    each = 2.0 ** -20 + 2 * math.pi * torch.tensor(pos, dtype=torch.float64).abs().view(T, 1, 1) * 2.0 ** -65
    tol = ((a.abs() + b.abs()) * each).repeat(1, 1, 2)
    h = 2.0 ** (-8 if dtype == torch.bfloat16 else -11)
    for o in out:
        assert ((o.cpu().double() - want).abs() <= h * want.abs() + tol + 2.0 ** -25).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,R,T", [(128, 128, 5003), (256, 128, 2501), (256, 256, 2600)])
def test_rows_past_the_caches(dev, dtype, D, R, T):
    Hq, H = 37, 5
    assert T * (Hq + H) * D * 4 > 96 << 20
    g = torch.Generator(device=dev).manual_seed(1)
    qkv = torch.randn(T, (Hq + 2 * H) * D, generator=g, device=dev).to(dtype)
    q, k, v = (t.view(T, -1, D) for t in qkv.split([Hq * D, H * D, H * D], dim=1))
    pos = torch.randint(0, 1 << 20, (T,), generator=g, device=dev)
    rot = pkg("layers.rotary").Rotary(D, rotary_dim=R, scale=1.25, device=dev)
    want = [rot.forward(q[i:i + 100], k[i:i + 100], pos[i:i + 100]) for i in range(0, T, 100)]
    want = tuple(torch.cat(t) for t in zip(*want))
    got = rot.forward(q, k, pos)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    before = v.clone()
    rot.forward_inplace(q, k, pos)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, before)
