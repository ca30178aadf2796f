"""The error of attention over a 4-bit cache (quant/kv4.py) against the length of what it sums, as a norm over the
output's. Long contexts average values of no common sign, so outputs are a hundredth of the values that are summed:
a bound by the largest value says nothing about them.

Tolerance, beside the one rounding of the output (its norm is taken from the 64-bit result itself). bf16 models: p s
enters its product in 11 bits, off by 2^-11 at most and 2^-11 / sqrt(3) = 2.8e-4 in the square's mean, of s (c - 7.5), whose
square's mean is a value's variance and the square of its range's centre, below 1.1 times it: 3e-4. Either type: scores
are f32 sums of products up to 15 s |q| (here 15 * 0.4 * 6 * D^-0.5 * log2 e = 4.6 at D = 128), off by 2^-21 of that: 1e-5 in
log2, and a value's sums in f32 between 7.5 s = 1.3 and the output's 2e-3 to 6e-3, off by 2^-22 of the larger: 1.5e-4 at
most. Together 3.4e-4 for bf16 and 1.5e-4 for fp16; both squares add to the rounding's."""
import math

import pytest
import torch

from test_kv4 import DTYPES, _kv4


def _values(codes, scale):
    return codes.double() * scale[..., :1].double() + scale[..., 1:].double()


def _case(dev, dtype, n, D, G, T, scale, page=64):
    """A random sequence of n tokens on one head, and G T random queries that see all of it (non-causal)."""
    g = torch.Generator(device=dev).manual_seed(n + D)
    pages = n // page
    cache = _kv4().KV4Cache(pages, page, 1, D, dtype, dev)
    table = torch.randperm(pages, generator=g, device=dev).int().view(1, -1)
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    k = torch.randn(n, 1, D, generator=g, device=dev).to(dtype)
    v = (torch.randn(n, 1, D, generator=g, device=dev) * 0.5).to(dtype)
    _kv4().kv4_append(cache, k, v, table, i32(0, n), i32(n))
    q = (torch.randn(T, G, D, generator=g, device=dev) * scale).to(dtype)
    ids = table[0].long()
    kc, vw = cache.k[ids, 0], cache.v[ids, 0]
    kc = torch.stack([kc & 15, kc >> 4], -1).flatten(-2)
    vc = ((vw.unsqueeze(2) >> (torch.arange(8, dtype=torch.int32, device=dev) * 4).view(1, 1, 8, 1)) & 15).flatten(1, 2)
    kk, vv = _values(kc, cache.k_scale[ids, 0]).flatten(0, 1), _values(vc, cache.v_scale[ids, 0]).flatten(0, 1)
    x = torch.matmul(q.double().view(T * G, D), kk.t().contiguous()) * D ** -0.5
    ref = torch.matmul(torch.softmax(x, -1), vv).view(T, G, D)
    return cache, table, i32(0, T), i32(n), q, ref


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,D", [(1024, 64), (16384, 128), (65536, 128), (131072, 64), (65536, 256)])
# the tokens split over the card; over one workgroup's four waves; one wave for all of them (17 and 64 columns)
@pytest.mark.parametrize("G,T,kw", [(8, 1, {"max_q": 1}), (8, 1, {"max_q": 1, "max_kv": 1}), (17, 1, {"max_q": 1, "max_kv": 1}),
                                    (8, 16, {"max_kv": 1})])
def test_error_does_not_grow_with_the_length(dev, dtype, n, D, G, T, kw):
    for scale in (0.0, 1.5):
        cache, table, cu, seq, q, ref = _case(dev, dtype, n, D, G, T, scale)
        out = _kv4().kv4_attention(q, cache, table, cu, seq, causal=False, **kw).double()
        norm = ref.norm().item()
        rounding = ((ref.to(dtype).double() - ref).norm() / norm).item()
        err = ((out - ref).norm() / norm).item()
        extra = 3.4e-4 if dtype == torch.bfloat16 else 1.5e-4
        assert err <= math.hypot(rounding, extra), f"{err:.3e}, of which the rounding is {rounding:.3e} (queries of {scale})"
