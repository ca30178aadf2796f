"""The 4-bit cache and its attention (quant/kv4.py) at the edges of what a call may hold: windows past the table, scales
that reach f32's end, one row of any stride, outputs on top of inputs, lengths near 2^31, and errors that keep their text."""
import math

import pytest
import torch

from conftest import pkg
from test_kv4 import DTYPES, Setup, _kv4


# ------------------------------------------------------------------------------------------------
# GPU
# ------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_window_past_the_table_is_nan(dev, dtype, causal):
    """A sequence longer than its table: a row whose window begins past the table's end sees missing tokens alone, and is
    NaN as a row is that sees some of them. In decode, over several rows, with the tokens split and not."""
    page = 16
    for width, past, news, window, kw in ((1, 24, 1, 8, {"max_q": 1}), (1, 24, 30, 8, {}), (1, 24, 39, 1, {}), (3, 1, 20, 8, {}),
                                          (256, 4000, 1, 3000, {"max_q": 1}), (256, 4000, 1, 3000, {"max_q": 1, "max_kv": 1}),
                                          (256, 4000, 40, 3000, {"max_q": 40}), (256, 600, 1200, 500, {})):
        cap = width * page
        s = Setup(dev, dtype, 64, 1, page, [cap], [1], seed=width)
        n = cap + past
        seq = torch.tensor([n], dtype=torch.int32, device=dev)
        cu = torch.tensor([0, news], dtype=torch.int32, device=dev)
        q = torch.randn(news, 2, 64, generator=torch.Generator().manual_seed(1)).to(dtype).to(dev)
        out, lse = _kv4().kv4_attention(q, s.cache, s.d_table, cu, seq, window=window, causal=causal, return_lse=True, **kw)
        # row i is at position n - news + i; not causal, it sees up to the sequence's end
        missing = torch.arange(n - news, n) >= cap if causal else torch.ones(news, dtype=torch.bool)
        where = (width, past, news, window, kw)
        assert torch.equal(torch.isnan(out).all(-1).all(-1).cpu(), missing), where
        assert torch.equal(torch.isnan(out).any(-1).any(-1).cpu(), missing), where
        assert torch.equal(torch.isnan(lse).all(-1).cpu(), missing) and torch.isfinite(lse.cpu()[~missing]).all(), where
