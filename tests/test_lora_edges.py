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
