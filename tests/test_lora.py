"""Low-rank adapters beside a projection (quant/lora.py): refusals on the CPU, and on the GPU the sum against
64 bits.

Tolerances. The sum is rounded once: 2^-8 of it for bf16, 2^-11 for fp16. Before that the adapters' part d
carries f32 sums over K and rank and, for bf16, the split of x A^T into two terms (2^-17 of it): together
below 2^-14 of sum_r |v_r| |B_nr| |scaling|, which is what is allowed on top. fp16's numbers below 2^-14
are 2^-24 apart, so a result there is rounded by up to 2^-25 whatever its size (a result of 2.4e-5 by
3e-8, where 2^-11 of it is 1.2e-8): 2^-25 is allowed too."""
import pytest
import torch

import synth
from conftest import pkg

DTYPES = [torch.bfloat16, torch.float16]


def _lora():
    return pkg("quant.lora")


def _eps(dtype):
    return 2.0 ** (-8 if dtype == torch.bfloat16 else -11)


def make(L, rank, K, slices, dtype, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    N = sum(slices)
    a = (torch.randn(L, len(slices) * rank, K, generator=g) / K ** 0.5 * scale).to(dtype)
    b = (torch.randn(L, N, rank, generator=g) * 0.3).to(dtype)
    s = torch.rand(L, generator=g) * 2 + 0.25
    return a, b, s


def delta(x, a, b, s, slices, ids):
    """(d, its sum of magnitudes) in f64."""
    M, N, rank = x.shape[0], b.shape[1], b.shape[2]
    d, mag = torch.zeros(M, N, dtype=torch.float64), torch.zeros(M, N, dtype=torch.float64)
    for m in range(M):
        l = int(ids[m])
        if not 0 <= l < a.shape[0]:
            continue
        v = a[l].double() @ x[m].double()
        col = 0
        for i, w in enumerate(slices):
            vi, bi = v[i * rank:(i + 1) * rank], b[l, col:col + w].double()
            d[m, col:col + w] = float(s[l]) * (bi @ vi)
            mag[m, col:col + w] = abs(float(s[l])) * (bi.abs() @ vi.abs())
            col += w
    return d, mag


def close(got, want, mag, dtype, what=""):
    err = (got.cpu().double() - want).abs() - _eps(dtype) * want.abs() - 2.0 ** -14 * mag - (2.0 ** -25 if dtype == torch.float16 else 0.0)
    assert not torch.isnan(got).any(), what
    assert err.max().item() <= 0, f"{what}: {err.max().item():.3e} past the tolerance"


def to(dev, *ts):
    return [t.to(dev) for t in ts]


# ------------------------------------------------------------------------------------------------ CPU
def test_adapter_set_refusals():
    m = _lora()
    a, b, s = make(3, 16, 64, [32, 16], torch.bfloat16)
    ok = m.LoraAdapters(a, b, s, [32, 16])
    assert (len(ok), ok.rank, ok.in_features, ok.out_features, ok.slices) == (3, 16, 64, 48, (32, 16))
    for args, err, msg in (((a, b, s, [24, 24]), ValueError, "multiples of 16"), ((a, b, s, [48, 16]), ValueError, "add up"),
                           ((a, b, s, []), ValueError, "slices"), ((a, b, s), ValueError, "a must be"),
                           ((a.float(), b, s, [32, 16]), TypeError, "bf16 or fp16"), ((a.half(), b, s, [32, 16]), TypeError, "bf16"),
                           ((a, b, s.double(), [32, 16]), TypeError, "scaling"), ((a, b, s[:2], [32, 16]), TypeError, "scaling"),
                           ((a[:2], b, s, [32, 16]), ValueError, "a must be"), ((a, b[..., :12].contiguous(), s, [32, 16]), ValueError, "rank"),
                           ((a, b.transpose(0, 1).contiguous().transpose(0, 1), s, [32, 16]), ValueError, "contiguous"),
                           ((a[..., :60].contiguous(), b, s, [32, 16]), ValueError, "multiple of 8")):
        with pytest.raises(err, match=msg):
            m.LoraAdapters(*args)


def test_cpu_calls_are_refused():
    m = _lora()
    a, b, s = make(2, 8, 64, [32], torch.bfloat16)
    ad = m.LoraAdapters(a, b, s)
    x, y, ids = torch.zeros(4, 64).bfloat16(), torch.zeros(4, 32).bfloat16(), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="one GPU"):
        m.lora_add(y, x, ad, ids)
    with pytest.raises(TypeError, match="x must be"):
        m.lora_add(y, x.half(), ad, ids)
    with pytest.raises(TypeError, match="adapters must be"):
        m.lora_add(y, x, ad, ids.long())
    with pytest.raises(TypeError, match="adapters must be"):
        m.w4a8_linear_lora(x, None, None, None, 128, ad, ids[:3])


def test_grids_past_32_bits_are_refused():
    """2^22 blocks of rows by 8 slices: each has a workgroup of its own, and the launch would not fit."""
    import ctypes

    if torch.cuda.is_available():
        pytest.skip("the pointers are not real")
    lib = pkg("_abi").load()
    P = 1 << 20
    cols = (ctypes.c_int64 * 8)(*[16] * 8)
    M = 1 << 26
    rc = lib.w4a8_lora_add(P, 0, M, 8, 8, P, P, P, 2, 8, ctypes.addressof(cols), 8, P, P, 0, 128, P, 128, P, 1 << 50, None)
    assert rc == 2 and b"w4a8_lora_add: past its index ranges" in lib.w4a8_last_error()


def test_abi_refuses_before_any_launch():
    import ctypes

    lib = pkg("_abi").load()
    P = 1 << 20

    def call(dtype=0, M=4, K=128, ldx=128, a=P, L=2, rank=16, cols=(32, 16), base_dtype=0, ldb=48, out=P, ldo=48, ws=P, wsb=1 << 20):
        c = (ctypes.c_int64 * len(cols))(*cols)
        rc = lib.w4a8_lora_add(P, dtype, M, K, ldx, a, P, P, L, rank, ctypes.addressof(c), len(cols), P, P, base_dtype, ldb,
                               out, ldo, ws, wsb, None)
        return rc, lib.w4a8_last_error()

    for kw, code, msg in ((dict(dtype=2), 1, b"bf16 or fp16"), (dict(base_dtype=1), 1, b"base"), (dict(K=100), 1, b"multiple of 8"),
                          (dict(L=0), 1, b"adapters"), (dict(rank=12), 2, b"ranks"), (dict(rank=264), 2, b"ranks"),
                          (dict(cols=(24,)), 1, b"columns"), (dict(cols=(16,) * 9), 2, b"slices"), (dict(M=-1), 1, b"M=-1"),
                          (dict(a=None), 1, b"aligned"), (dict(out=P + 8), 1, b"aligned"), (dict(ldx=120), 1, b"strides"),
                          (dict(ldo=40), 1, b"strides"), (dict(ldb=52), 1, b"strides"), (dict(ws=None), 1, b"workspace"),
                          (dict(wsb=16), 1, b"workspace")):
        rc, err = call(**kw)
        assert rc == code and msg in err, (kw, rc, err)
    assert call(M=0)[0] == 0
    f = lib.w4a8_lora_workspace_bytes
    assert f(0, 128, 16, 1) == 0 and f(4, 128, 12, 1) == -1 and f(4, 128, 16, 9) == -1 and f(-1, 128, 16, 1) == -1
    assert f(4, 128, 16, 2) >= 4 * 32 * 4


# ------------------------------------------------------------------------------------------------ GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,rank,slices", [(1, 512, 16, [64]), (2, 520, 8, [16]), (5, 2048, 16, [256, 64, 64]), (16, 1032, 24, [48, 80]),
                                             (17, 256, 64, [320]), (63, 8, 8, [16, 32]), (64, 640, 128, [64, 16]),
                                             (65, 640, 40, [112]), (130, 1288, 256, [64, 32]), (300, 384, 32, [208, 32])])
def test_add_matches(dev, dtype, M, K, rank, slices):
    m = _lora()
    L = 7
    a, b, s = make(L, rank, K, slices, dtype, seed=M)
    g = torch.Generator().manual_seed(M + 1)
    x, y = torch.randn(M, K, generator=g).to(dtype), torch.randn(M, sum(slices), generator=g).to(dtype)
    ad = m.LoraAdapters(*to(dev, a, b, s), slices)
    every = torch.randint(-1, L, (M,), generator=g, dtype=torch.int32)
    runs = (torch.arange(M) * 4 // M).to(torch.int32) - 1
    for ids in (every, runs, torch.full((M,), 3, dtype=torch.int32), torch.full((M,), -1, dtype=torch.int32)):
        yd = y.to(dev)
        out = torch.full((M, sum(slices)), 9.0, dtype=dtype, device=dev)
        assert m.lora_add(yd, x.to(dev), ad, ids.to(dev), out=out) is out
        assert torch.equal(yd.cpu(), y)
        d, mag = delta(x, a, b, s, slices, ids)
        close(out, y.double() + d, mag, dtype, "out of place")
        bare = ids < 0
        assert torch.equal(out.cpu()[bare], y[bare]), "rows without an adapter keep their values"
        assert m.lora_add(yd, x.to(dev), ad, ids.to(dev)) is yd
        assert torch.equal(yd, out), "in place"


@pytest.mark.gpu
def test_add_on_views_and_ids_out_of_range(dev):
    """Strided x, y and out (columns of wider rows), and ids on both sides of 0 .. L-1."""
    m = _lora()
    dtype, M, K, rank, slices = torch.bfloat16, 21, 264, 16, [64, 48]
    a, b, s = make(2, rank, K, slices, dtype)
    g = torch.Generator().manual_seed(5)
    ids = torch.tensor([0, 1, 2, -1, -5, 2 ** 31 - 1, -2 ** 31] * 3, dtype=torch.int32)
    wide, ywide = torch.randn(M, 512, generator=g).to(dtype), torch.randn(M, 256, generator=g).to(dtype)
    ad = m.LoraAdapters(*to(dev, a, b, s), slices)
    xd, yd = wide.to(dev), ywide.to(dev)
    d, mag = delta(wide[:, 8:8 + K], a, b, s, slices, ids)
    m.lora_add(yd[:, 16:16 + 112], xd[:, 8:8 + K], ad, ids.to(dev))
    close(yd[:, 16:128], ywide[:, 16:128].double() + d, mag, dtype)
    assert torch.equal(yd[:, :16].cpu(), ywide[:, :16]) and torch.equal(yd[:, 128:].cpu(), ywide[:, 128:])
    # an x whose rows are not aligned, and one transposed, are copied
    y2 = ywide[:, :112].contiguous().to(dev)
    m.lora_add(y2, xd[:, 3:3 + K], ad, ids.to(dev))
    d, mag = delta(wide[:, 3:3 + K], a, b, s, slices, ids)
    close(y2, ywide[:, :112].double() + d, mag, dtype)
    with pytest.raises(ValueError, match="y must be"):
        m.lora_add(yd[:, 1:113], xd[:, :K], ad, ids.to(dev))
    with pytest.raises(ValueError, match="out must be"):
        m.lora_add(y2, xd[:, :K], ad, ids.to(dev), out=torch.empty(M, 112, device=dev))
    empty = m.lora_add(y2[:0], xd[:0, :K], ad, ids[:0].to(dev))
    assert empty.shape == (0, 112)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_one_users_infinity_stays_with_that_user(dev, dtype):
    m = _lora()
    M, K, rank, slices = 33, 256, 16, [64]
    a, b, s = make(4, rank, K, slices, dtype)
    g = torch.Generator().manual_seed(7)
    x, y = torch.randn(M, K, generator=g).to(dtype), torch.randn(M, 64, generator=g).to(dtype)
    ids = (torch.arange(M) % 5 - 1).to(torch.int32)
    want = m.lora_add(y.to(dev), x.to(dev), m.LoraAdapters(*to(dev, a, b, s)), ids.to(dev)).cpu()
    a2, b2, x2 = a.clone(), b.clone(), x.clone()
    a2[1, 3, 5] = float("inf")
    b2[2, 7, 1] = float("nan")
    x2[4] = float("nan")  # id 3
    got = m.lora_add(y.to(dev), x2.to(dev), m.LoraAdapters(*to(dev, a2, b2, s)), ids.to(dev)).cpu()
    bad = torch.zeros(M, 64, dtype=torch.bool)
    bad[ids == 1] = True
    bad[ids == 2, 7] = True
    bad[4] = True
    assert torch.equal(got[~bad], want[~bad]) and torch.isnan(got[bad]).float().mean() > 0.9


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-6, 1e3])
def test_fp16_ranges(dev, scale):
    """x A^T far below fp16's normal numbers (1e-6), and, with scaling to match, past its largest (1e5)."""
    m = _lora()
    dtype, M, K, rank, slices = torch.float16, 9, 512, 16, [64]
    a, b, s = make(2, rank, K, slices, dtype, scale=min(scale, 50.0) * (20 if scale < 1 else 1))
    g = torch.Generator().manual_seed(8)
    x = (torch.randn(M, K, generator=g) * (1e4 if scale > 1 else 1.0)).to(dtype)
    s = s * (1e-5 if scale > 1 else 1e4)
    y = torch.randn(M, 64, generator=g).to(dtype)
    ids = (torch.arange(M) % 2).to(torch.int32)
    got = m.lora_add(y.to(dev), x.to(dev), m.LoraAdapters(*to(dev, a, b, s)), ids.to(dev))
    d, mag = delta(x, a, b, s, slices, ids)
    assert d.abs().max() > 0.01
    close(got, y.double() + d, mag, dtype)


def _weight(kernels, fmt, N, K, dev):
    if fmt == "mxfp4":
        w, s = synth.mxfp4_weight(N, K, seed=N)
        return w.to(dev), s.to(dev), None, 32, True
    if fmt == "nvfp4":
        w, s, z = synth.nvfp4_weight(N, K, seed=N)
        return w.to(dev), s.to(dev), z.view(torch.int32).to(dev), 16, True
    w, s, z = synth.int4_weight(N, K, 128, seed=N, asym=fmt == "asym", scale_floor=1e-4)
    return w.to(dev), s.to(dev), None if z is None else z.to(dev), 128, False


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", ["sym", "asym", "mxfp4", "nvfp4"])
@pytest.mark.parametrize("M", [1, 2, 8, 16, 17, 128, 129, 200])
def test_linear_lora(kernels, dev, dtype, fmt, M):
    """The projection's own output in f32, from the C ABI, plus the adapters in f64, rounded once at every size."""
    m = _lora()
    K, slices, rank, L = 1024, [256, 64, 64], 16, 5
    N = sum(slices)
    w, sc, z, grp, e2 = _weight(kernels, fmt, N, K, dev)
    tiles = kernels.repack_w4(w, e2)
    a, b, s = make(L, rank, K, slices, dtype, seed=M)
    ad = m.LoraAdapters(*to(dev, a, b, s), slices)
    x = synth.activations(M, K, seed=M, dtype=dtype)
    xd = x.to(dev)
    g = torch.Generator().manual_seed(M)
    ids = torch.randint(-1, L, (M,), generator=g, dtype=torch.int32)
    arm = 1 if M <= 16 else 2
    f32, _ = kernels._dense(xd, tiles, sc, z, grp, e2, None, None, False, arm, torch.float32)
    plain = kernels.w4a8_linear(xd, tiles, sc, z, grp, weight_is_e2m1=e2)
    out = m.w4a8_linear_lora(xd, tiles, sc, z, grp, ad, ids.to(dev), weight_is_e2m1=e2)
    d, mag = delta(x, a, b, s, slices, ids)
    close(out, f32.cpu().double() + d, mag, dtype)
    assert torch.equal(out[ids.to(dev) < 0], plain[ids.to(dev) < 0])
    # the producer pair and the op layout give the same
    q, qs = kernels.act_quant(xd)
    assert torch.equal(out, m.w4a8_linear_lora(xd, tiles, sc, z, grp, ad, ids.to(dev), weight_is_e2m1=e2, x_fp8=q, act_scales=qs))
    assert torch.equal(out, m.w4a8_linear_lora(xd, w, sc, z, grp, ad, ids.to(dev), weight_is_e2m1=e2))


@pytest.mark.gpu
def test_linear_methods_take_adapters(kernels, dev, monkeypatch):
    """LinearMethod.apply(lora=...) is the linear plus lora_add for the quantized methods, their W4A16 arm and
    the unquantized one; the fused gate_up + silu leaves a batch with adapters to the unfused pair."""
    m, method, config = _lora(), pkg("quant.method"), pkg("quant.config")
    K, N, M, L = 512, 256, 7, 3
    dtype = torch.bfloat16
    a, b, s = make(L, 16, K, [N], dtype)
    ad = m.LoraAdapters(*to(dev, a, b, s))
    ids = torch.tensor([0, 2, -1, 1, 1, 0, -1], dtype=torch.int32, device=dev)
    x = synth.activations(M, K, seed=2, dtype=dtype).to(dev)

    class Layer:
        pass

    layer = Layer()
    layer.weight = torch.randn(N, K, device=dev).to(dtype) * 0.03
    bias = torch.randn(N, device=dev).to(dtype)
    un = method.UnquantizedLinearMethod()
    assert torch.equal(un.apply(layer, x, bias, lora=(ad, ids)), m.lora_add(un.apply(layer, x, bias), x, ad, ids))
    w, sc, z = synth.int4_weight(N, K, 128, seed=1, asym=False)
    layer._w_packed_op, layer._scales_op, layer._zeros_op = kernels.repack_w4(w.to(dev)), sc.to(dev), None
    quant = config.QuantConfig(method="gptq", bits=4, group_size=128, sym=True)
    q = method.W4A8LinearMethod(quant)
    want = m.w4a8_linear_lora(x, layer._w_packed_op, layer._scales_op, None, 128, ad, ids)
    assert torch.equal(q.apply(layer, x, None, lora=(ad, ids)), want)
    assert torch.equal(q.apply(layer, x, bias, lora=(ad, ids)), want + bias)
    assert torch.equal(q.apply(layer, x, None), kernels.w4a8_linear(x, layer._w_packed_op, layer._scales_op, None, 128))
    assert q.apply_swiglu(layer, x) is not None and q.apply_swiglu(layer, x, lora=(ad, ids)) is None
    monkeypatch.setattr(kernels, "MOE_W4A16", "1")
    assert torch.equal(q.apply(layer, x, None, lora=(ad, ids)), m.lora_add(q.apply(layer, x, None), x, ad, ids))


@pytest.mark.gpu
def test_captured_call_replays_with_other_adapters(kernels, dev):
    m = _lora()
    dtype, K, slices, rank, L, M = torch.bfloat16, 1024, [256, 128], 16, 6, 5
    w, sc, z, grp, e2 = _weight(kernels, "sym", sum(slices), K, dev)
    tiles = kernels.repack_w4(w, e2)
    ad = m.LoraAdapters(*to(dev, *make(L, rank, K, slices, dtype)), slices)
    x, ids = torch.zeros(M, K, dtype=dtype, device=dev), torch.zeros(M, dtype=torch.int32, device=dev)
    step = lambda: m.w4a8_linear_lora(x, tiles, sc, z, grp, ad, ids)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    g = torch.Generator().manual_seed(3)
    for rep in range(4):
        x.copy_(torch.randn(M, K, generator=g))
        ids.copy_(torch.randint(-1, L, (M,), generator=g, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.empty(1 << 20, device=dev).normal_()
        torch.cuda.synchronize()
        assert torch.equal(out, want), rep


@pytest.mark.gpu
def test_rows_do_not_depend_on_their_batch(dev):
    """Up to 64 rows, where the parts of K are the same, a row gives the same bits alone and among others."""
    m = _lora()
    dtype, K, slices, rank, L = torch.float16, 2048, [128], 32, 9
    ad = m.LoraAdapters(*to(dev, *make(L, rank, K, slices, dtype)), slices)
    g = torch.Generator().manual_seed(4)
    x, y = torch.randn(16, K, generator=g).to(dtype).to(dev), torch.randn(16, 128, generator=g).to(dtype).to(dev)
    ids = torch.randint(-1, L, (16,), generator=g, dtype=torch.int32).to(dev)
    all_rows = m.lora_add(y.clone(), x, ad, ids)
    for i in range(16):
        assert torch.equal(all_rows[i:i + 1], m.lora_add(y[i:i + 1].clone(), x[i:i + 1], ad, ids[i:i + 1]))
