"""Low-rank adapters (quant/lora.py) at the edges of what a call may hold. Tolerances: test_lora.py."""
import ctypes

import pytest
import torch

import synth
from conftest import pkg
from test_lora import DTYPES, _eps, _lora, close, delta, make, to


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [1, 5, 70])
def test_contiguous_rows_that_begin_anywhere(dev, dtype, M):
    """x contiguous but not 16-byte aligned is copied, as x of other strides is."""
    m = _lora()
    K, N = 72, 48
    a, b, s = make(2, 8, K, [N], dtype, seed=M)
    ad = m.LoraAdapters(*to(dev, a, b, s))
    g = torch.Generator().manual_seed(M)
    x, y = torch.randn(M, K, generator=g).to(dtype), torch.randn(M, N, generator=g).to(dtype)
    ids = (torch.arange(M) % 3 - 1).int()
    buf = torch.zeros(M * K + 8, dtype=dtype, device=dev)
    shifted = buf[3:3 + M * K].view(M, K)
    shifted.copy_(x)
    assert shifted.is_contiguous() and shifted.data_ptr() % 16
    got = m.lora_add(y.to(dev), shifted, ad, ids.to(dev))
    assert torch.equal(got, m.lora_add(y.to(dev), x.to(dev), ad, ids.to(dev)))
    d, mag = delta(x, a, b, s, [N], ids)
    close(got, y.double() + d, mag, dtype)


def test_abi_refuses_an_output_on_top_of_its_base():
    """Host checks of the C entry point, with pointers that are never read: what passes them ends at the workspace."""
    lib = pkg("_abi").load()
    P = 1 << 20

    def call(base, ldb, out, ldo, M=4, n=48, base_dtype=0):
        c = (ctypes.c_int64 * 1)(n)
        rc = lib.w4a8_lora_add(P, 0, M, 64, 64, P, P, P, 2, 16, ctypes.addressof(c), 1, P, base, base_dtype, ldb, out, ldo, None, 0, None)
        assert rc == 1
        return lib.w4a8_last_error()

    # rows of 96 bytes (f32 base: 192)
    for kw in (dict(base=P, ldb=48, out=P + 96, ldo=48), dict(base=P + 96, ldb=48, out=P, ldo=48), dict(base=P, ldb=48, out=P, ldo=96),
               dict(base=P, ldb=128, out=P + 80, ldo=128), dict(base=P + 192, ldb=128, out=P, ldo=128), dict(base=P, ldb=48, out=P + 16, ldo=48, M=1),
               dict(base=P, ldb=48, out=P, ldo=48, base_dtype=2), dict(base=P, ldb=64, out=P + 128, ldo=128, base_dtype=2)):
        assert b"overlaps" in call(**kw), kw
    for kw in (dict(base=P, ldb=48, out=P, ldo=48), dict(base=P, ldb=48, out=P + 4 * 96, ldo=48), dict(base=P, ldb=128, out=P + 96, ldo=128),
               dict(base=P + 96, ldb=128, out=P, ldo=128), dict(base=P, ldb=128, out=P + 160, ldo=128), dict(base=P, ldb=48, out=P + 96, ldo=48, M=1),
               dict(base=P, ldb=48, out=P, ldo=128, M=1), dict(base=P, ldb=64, out=P + 1024, ldo=64, base_dtype=2)):
        assert b"workspace" in call(**kw), kw


@pytest.mark.gpu
def test_outputs_beside_and_on_top_of_y(dev):
    m = _lora()
    dtype, M, K, N = torch.bfloat16, 40, 128, 64
    a, b, s = make(3, 16, K, [N], dtype)
    ad = m.LoraAdapters(*to(dev, a, b, s))
    g = torch.Generator().manual_seed(2)
    x, wide = torch.randn(M, K, generator=g).to(dtype).to(dev), torch.randn(M + 1, 4 * N, generator=g).to(dtype).to(dev)
    ids = (torch.arange(M) % 4 - 1).int().to(dev)
    want = m.lora_add(wide[:M, :N].clone(), x, ad, ids)
    buf = wide.clone()
    m.lora_add(buf[:M, :N], x, ad, ids, out=buf[:M, N:2 * N])
    assert torch.equal(buf[:M, N:2 * N], want) and torch.equal(buf[:, :N], wide[:, :N]) and torch.equal(buf[:, 2 * N:], wide[:, 2 * N:])
    for out in (buf[1:, :N], buf[:M, N // 2:N + N // 2], buf[:M, 8:8 + N]):
        with pytest.raises(RuntimeError, match="overlaps"):
            m.lora_add(buf[:M, :N], x, ad, ids, out=out)
    assert torch.equal(m.lora_add(buf[:M, :N], x, ad, ids, out=buf[:M, :N]), want)
