"""The host extension's calls for the 4-bit cache and the low-rank adapters: they leave what they do not take to
the Python path, and both give the same tensors, bit for bit."""
import pytest
import torch

import synth
from conftest import pkg

NEW = {"kv4_append": 9, "kv4_read": 8, "kv4_attention": 15, "lora_add": 8, "linear_lora": 14}


def test_cpu_tensors_and_wrong_counts_are_left_alone():
    m = pkg("_host").load()
    t = torch.zeros(4, 4)
    for name, n in NEW.items():
        assert getattr(m, name)(*[t] * n) is None
        assert getattr(m, name)(*[None] * n) is None
        with pytest.raises(TypeError):
            getattr(m, name)(t)
        assert getattr(pkg("_host")._Absent, name)(*range(n)) is None


class _Off:
    """The extension as if it took no call."""

    linear = rms_norm = moe = kv4_append = kv4_read = kv4_attention = lora_add = linear_lora = staticmethod(lambda *a: None)


def _both(monkeypatch, name, fn):
    """fn() served by the extension (checked) and by the Python path."""
    host = pkg("_host")
    real, took = host.load(), []

    class Watch:
        def __getattr__(self, k):
            def call(*a):
                r = getattr(real, k)(*a)
                took.append((k, r is not None))
                return r

            return call

    with monkeypatch.context() as mp:
        mp.setattr(host, "_mod", Watch())
        a = fn()
    assert (name, True) in took
    with monkeypatch.context() as mp:
        mp.setattr(host, "_mod", _Off)
        b = fn()
    torch.cuda.synchronize()
    return a, b


def _same(a, b):
    if isinstance(a, tuple):
        assert len(a) == len(b)
        for x, y in zip(a, b):
            _same(x, y)
    else:
        assert a.dtype == b.dtype and torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_cache_calls(monkeypatch, dev, dtype):
    kv4 = pkg("quant.kv4")
    H, G, D, page = 2, 4, 128, 16
    table = torch.tensor([[3, 1, 0], [2, 4, 5]], dtype=torch.int32, device=dev)
    cu, seq = torch.tensor([0, 3, 8], dtype=torch.int32, device=dev), torch.tensor([40, 33], dtype=torch.int32, device=dev)
    qkv = torch.randn(8, (G * H + 2 * H) * D, device=dev).to(dtype)
    q, k, v = (t.view(8, -1, D) for t in qkv.split([G * H * D, H * D, H * D], dim=1))

    def append():
        c = kv4.KV4Cache(6, page, H, D, dtype, dev)
        kv4.kv4_append(c, k, v, table, cu, seq)
        return c.k, c.v, c.k_scale, c.v_scale

    _same(*_both(monkeypatch, "kv4_append", append))
    c = kv4.KV4Cache.from_tensors(*append())
    _same(*_both(monkeypatch, "kv4_read", lambda: kv4.kv4_read(c, table, cu, seq, 8)))
    for kw in ({}, dict(return_lse=True, window=7), dict(max_q=5, max_kv=40, sm_scale=0.5), dict(causal=False)):
        _same(*_both(monkeypatch, "kv4_attention", lambda: kv4.kv4_attention(q, c, table, cu, seq, **kw)))
    buf = torch.zeros(8, 3 * G * H, D, dtype=dtype, device=dev)
    got = _both(monkeypatch, "kv4_attention", lambda: kv4.kv4_attention(q, c, table, cu, seq, out=buf[:, :G * H]))
    assert got[0].data_ptr() == buf.data_ptr() and (buf[:, G * H:] == 0).all()
    with pytest.raises(ValueError, match="window"):
        kv4.kv4_attention(q, c, table, cu, seq, window=-1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [1, 16, 40, 130])
def test_adapter_calls(monkeypatch, kernels, dev, dtype, M):
    m = pkg("quant.lora")
    K, slices, rank, L = 512, [128, 64], 16, 3
    N = sum(slices)
    w, s, z = synth.int4_weight(N, K, 128, seed=1, asym=True)
    tiles, sd, zd = kernels.repack_w4(w.to(dev)), s.to(dev), z.to(dev)
    ad = m.LoraAdapters(torch.randn(L, 2 * rank, K, device=dev).to(dtype), torch.randn(L, N, rank, device=dev).to(dtype),
                        torch.rand(L, device=dev), slices)
    x = synth.activations(M, K, seed=M, dtype=dtype).to(dev)
    ids = (torch.arange(M) % 4 - 1).int().to(dev)
    y = torch.randn(M, 2 * N, device=dev).to(dtype)[:, N:]
    _same(*_both(monkeypatch, "lora_add", lambda: m.lora_add(y.clone(), x, ad, ids)))
    _same(*_both(monkeypatch, "lora_add", lambda: m.lora_add(y, x, ad, ids, out=torch.zeros(M, N, dtype=dtype, device=dev))))
    _same(*_both(monkeypatch, "linear_lora", lambda: m.w4a8_linear_lora(x, tiles, sd, zd, 128, ad, ids)))
    q, qs = kernels.act_quant(x)
    _same(*_both(monkeypatch, "linear_lora", lambda: m.w4a8_linear_lora(x, tiles, sd, zd, 128, ad, ids, x_fp8=q, act_scales=qs)))
