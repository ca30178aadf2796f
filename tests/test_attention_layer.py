"""The operators of a decoder layer's attention half as they are used together: norm, qkv with low-rank adapters,
the 4-bit cache and its attention, o projection with adapters, for a batch of prompts and then captured
decode steps whose sequences, adapters and lengths change from replay to replay."""
import pytest
import torch

import synth
from conftest import pkg
from test_kv4 import cache_values, ref_attention, ref_values
from test_lora import delta, make

HIDDEN, HQ, H, D, PAGE, L, RANK = 512, 8, 2, 64, 16, 4, 16
KV = H * D


class Half:
    """norm -> qkv -> attention -> o of one layer on int4 weights."""

    def __init__(self, dev, dtype):
        kernels, lora, att = pkg("quant.kernels"), pkg("quant.lora"), pkg("layers.attention")
        kv4, method, config = pkg("quant.kv4"), pkg("quant.method"), pkg("quant.config")
        self.dev, self.dtype = dev, dtype
        self.norm = pkg("layers.norm").RMSNorm(HIDDEN, 1e-6)
        self.norm.weight = (1 + 0.1 * torch.randn(HIDDEN, generator=torch.Generator().manual_seed(1))).to(dtype).to(dev)
        self.method = method.W4A8LinearMethod(config.QuantConfig(method="gptq", bits=4, group_size=128, sym=True))
        self.qkv, self.o = type("Layer", (), {})(), type("Layer", (), {})()
        self.slices = [HQ * D, KV, KV]
        for layer, n, k, seed in ((self.qkv, sum(self.slices), HIDDEN, 3), (self.o, HIDDEN, HQ * D, 4)):
            w, s, _ = synth.int4_weight(n, k, 128, seed=seed, asym=False)
            layer._w_packed_op, layer._scales_op, layer._zeros_op = kernels.repack_w4(w.to(dev)), s.to(dev), None
        self.raw = make(L, RANK, HIDDEN, self.slices, dtype, seed=5), make(L, RANK, HQ * D, [HIDDEN], dtype, seed=6)
        self.lora_qkv = lora.LoraAdapters(*(t.to(dev) for t in self.raw[0]), self.slices)
        self.lora_o = lora.LoraAdapters(*(t.to(dev) for t in self.raw[1]))
        self.att = att.KV4Attention(HQ, kv4.KV4Cache(40, PAGE, H, D, dtype, dev))

    def forward(self, x, adapters, batch):
        h, xq, xs = self.norm.forward_quant(x)
        qkv = self.method.apply(self.qkv, h, None, x_fp8=xq, act_scales=xs, lora=(self.lora_qkv, adapters))
        a = self.att.forward_qkv(qkv, batch)
        return h, qkv, a, self.method.apply(self.o, a, None, lora=(self.lora_o, adapters))


def _check_step(half, x, ids, lens, news, table, outs):
    """Each operator's output against its own formula in 64 bits, from the outputs before it."""
    kernels = pkg("quant.kernels")
    h, qkv, a, y = (t.cpu() for t in outs)
    eps = 2.0 ** (-8 if half.dtype == torch.bfloat16 else -11)
    for got, inp, layer, raw, slices in ((qkv, h, half.qkv, half.raw[0], half.slices), (y, a, half.o, half.raw[1], [HIDDEN])):
        base = kernels.w4a8_linear(inp.to(half.dev), layer._w_packed_op, layer._scales_op, None, 128).cpu().double()
        d, mag = delta(inp, *raw, slices, ids)
        want = base + d
        # here the projection alone is rounded to the type too; the operator rounds the sum only
        assert ((got.double() - want).abs() <= eps * (want.abs() + base.abs()) + 2.0 ** -14 * mag + 2.0 ** -24).all()
    ref, _ = ref_attention(qkv[:, :HQ * D].reshape(-1, HQ, D), cache_values(half.att.cache), table, PAGE, lens, news, D ** -0.5)
    vmax = qkv[:, HQ * D + KV:].double().abs().max().item() + 4
    assert ((a.double().view(-1, HQ, D) - ref).abs() <= eps * ref.abs() + 3.5e-4 * vmax).all()
    # the cache holds what the projection gave
    row = 0
    ck, cv = cache_values(half.att.cache)
    for b, (n, new) in enumerate(zip(lens, news)):
        pos = torch.arange(n - new, n)
        pages, slot = table[b, pos // PAGE].long(), pos % PAGE
        for c, at in ((ck, HQ * D), (cv, HQ * D + KV)):
            assert torch.equal(c[pages, :, slot], ref_values(qkv[row:row + new, at:at + KV].reshape(new, H, D)))
        row += new


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompts_then_captured_decode_steps(dev, dtype):
    half = Half(dev, dtype)
    att = pkg("layers.attention")
    g = torch.Generator().manual_seed(9)
    lens = [70, 1, 33]
    table = torch.randperm(40, generator=g).int()[:24].view(3, 8)
    d_table = table.to(dev)
    # prompts
    T = sum(lens)
    x = (torch.randn(T, HIDDEN, generator=g) * 0.7).to(dtype)
    ids = torch.tensor([0] * 70 + [-1] + [2] * 33, dtype=torch.int32)
    batch = att.KV4Batch(d_table, torch.tensor([0, 70, 71, 104], dtype=torch.int32, device=dev),
                         torch.tensor(lens, dtype=torch.int32, device=dev), 70, 70)
    outs = half.forward(x.to(dev), ids.to(dev), batch)
    torch.cuda.synchronize()
    _check_step(half, x, ids, lens, lens, table, outs)

    # decode: one token each, captured once
    xs, dids = torch.zeros(3, HIDDEN, dtype=dtype, device=dev), torch.zeros(3, dtype=torch.int32, device=dev)
    seq = torch.zeros(3, dtype=torch.int32, device=dev)  # padded: no tokens yet, nothing is appended
    step = att.KV4Batch(d_table, torch.arange(4, dtype=torch.int32, device=dev), seq, 1, 8 * PAGE)
    before = [t.clone() for t in (half.att.cache.k, half.att.cache.v)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        half.forward(xs, dids, step)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = half.forward(xs, dids, step)
    assert torch.equal(before[0], half.att.cache.k) and torch.equal(before[1], half.att.cache.v)
    for rep in range(4):
        lens = [n + 1 for n in lens]
        x = (torch.randn(3, HIDDEN, generator=g) * 0.7).to(dtype)
        ids = torch.randint(-1, L, (3,), generator=g, dtype=torch.int32)
        xs.copy_(x)
        dids.copy_(ids)
        seq.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [o.clone() for o in outs]
        torch.empty(1 << 20, device=dev).normal_()
        _check_step(half, x, ids, lens, [1, 1, 1], table, replayed)
        eager = half.forward(xs, dids, step)  # writes the same tokens again
        torch.cuda.synchronize()
        for a, b in zip(replayed, eager):
            assert torch.equal(a, b), rep


def test_layer_refusals():
    att, kv4 = pkg("layers.attention"), pkg("quant.kv4")
    cache = kv4.KV4Cache(2, 16, 2, 64, device="cpu")
    with pytest.raises(ValueError, match="query heads"):
        att.KV4Attention(3, cache)
    layer = att.KV4Attention(4, cache)
    t = lambda n: torch.zeros(1, n, dtype=torch.bfloat16)  # noqa: E731
    with pytest.raises(RuntimeError, match="on the GPU"):
        layer.forward(t(256), t(128), t(128), att.KV4Batch(torch.zeros(1, 1, dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32),
                                                           torch.ones(1, dtype=torch.int32)))
