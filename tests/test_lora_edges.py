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
@pytest.mark.parametrize("dtype", DTYPES)
def test_calls_without_rows(kernels, dev, dtype):
    """A step in which nobody has a token."""
    m = _lora()
    K, N = 256, 64
    w, sc, _ = synth.int4_weight(N, K, 128, seed=1, asym=False)
    a, b, s = make(2, 8, K, [N], dtype)
    ad = m.LoraAdapters(*to(dev, a, b, s))
    x, ids = torch.zeros(0, K, dtype=dtype, device=dev), torch.zeros(0, dtype=torch.int32, device=dev)
    out = m.w4a8_linear_lora(x, kernels.repack_w4(w.to(dev)), sc.to(dev), None, 128, ad, ids)
    assert out.shape == (0, N) and out.dtype == dtype
    assert m.lora_add(out, x, ad, ids) is out
    att, kv4 = pkg("layers.attention"), pkg("quant.kv4")
    layer = att.KV4Attention(4, kv4.KV4Cache(2, 16, 2, 64, dtype, dev))
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    for B in (0, 2):
        batch = att.KV4Batch(torch.zeros(B, 1, dtype=torch.int32, device=dev), i32(*[0] * (B + 1)), i32(*[0] * B), 0, 0)
        assert layer.forward_qkv(torch.zeros(0, 8 * 64, dtype=dtype, device=dev), batch).shape == (0, 4 * 64)


def test_the_projection_runs_on_its_tensors_device(monkeypatch):
    """On another device than the current one the extension leaves the call to the Python path, whose launches are all made
    with the tensors' device as the current one."""
    m = _lora()
    a, b, s = make(2, 8, 64, [32], torch.bfloat16)
    current, seen = ["another"], []

    class Device:
        def __init__(self, d):
            self.d = d

        def __enter__(self):
            current.append(self.d)

        def __exit__(self, *exc):
            current.pop()

    class Lib:
        w4a8_lora_workspace_bytes = staticmethod(lambda *a: 64)
        w4a8_lora_add = staticmethod(lambda *a: seen.append(("add", current[-1])) or 0)

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(m, "_check", lambda *a: None)
    monkeypatch.setattr(m.kernels, "_n_of", lambda w: 32)
    monkeypatch.setattr(m.kernels, "_dense_arm", lambda *a: (1, "decode_gemv"))
    monkeypatch.setattr(m.kernels, "_dense", lambda *a: (seen.append(("linear", current[-1])) or torch.zeros(4, 32), False))
    monkeypatch.setattr(m._abi, "load", lambda: Lib)
    monkeypatch.setattr(m._abi, "stream_of", lambda t: 0)
    x = torch.zeros(4, 64).bfloat16()
    m.w4a8_linear_lora(x, None, None, None, 128, m.LoraAdapters(a, b, s), torch.zeros(4, dtype=torch.int32))
    assert seen == [("linear", x.device), ("add", x.device)] and current == ["another"]


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


# ------------------------------------------------------------------------------------------------ calls of large sizes
def delta_on(dev, x, a, b, s, slices, ids):
    """test_lora.delta with the products of an adapter's rows at once, on the GPU."""
    M, rank, L = x.shape[0], b.shape[2], b.shape[0]
    d, mag = (torch.zeros(M, b.shape[1], dtype=torch.float64, device=dev) for _ in range(2))
    ids = ids.to(dev)
    for l in range(L):
        rows = (ids == l).nonzero().squeeze(1)
        v = x.to(dev)[rows].double() @ a[l].to(dev).double().t().contiguous()
        col = 0
        for i, w in enumerate(slices):
            vi, bi = v[:, i * rank:(i + 1) * rank], b[l, col:col + w].to(dev).double().t().contiguous()
            d[rows, col:col + w] = float(s[l]) * (vi @ bi)
            mag[rows, col:col + w] = abs(float(s[l])) * (vi.abs() @ bi.abs())
            col += w
    return d, mag


def close_on(got, want, mag, dtype, slack=0.0):
    err = (got.double() - want).abs() - _eps(dtype) * want.abs() - 2.0 ** -14 * mag - (2.0 ** -25 if dtype == torch.float16 else 0.0) - slack
    assert not torch.isnan(got).any() and err.max().item() <= 0, err.max().item()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
# spans of 512 and of 2048 columns, the last of a slice and its last step cut anywhere; ranks in registers and from LDS
@pytest.mark.parametrize("M,rank,slices", [(2048, 16, [8192, 272]), (2050, 40, [5136, 4112]), (8200, 8, [8208]), (2048, 72, [16, 8304])])
def test_spans_of_many_columns(dev, dtype, M, rank, slices):
    m = _lora()
    K, L, N = 64, 5, sum(slices)
    a, b, s = make(L, rank, K, slices, dtype, seed=M)
    ad = m.LoraAdapters(*to(dev, a, b, s), slices)
    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, K, generator=g).to(dtype)
    y = torch.randn(M, N, generator=torch.Generator(device=dev).manual_seed(M), device=dev).to(dtype)
    runs = (torch.arange(M) * 7 // M).int() - 1  # prompts; the first and the last have no adapter
    mixed = torch.randint(-1, L, (M,), generator=g, dtype=torch.int32)
    for ids in (runs, mixed):
        d, mag = delta_on(dev, x, a, b, s, slices, ids)
        out = m.lora_add(y, x.to(dev), ad, ids.to(dev), out=torch.full_like(y, 9.0))
        close_on(out, y.double() + d, mag, dtype)
        bare = ((ids < 0) | (ids >= L)).to(dev)
        assert torch.equal(out[bare], y[bare])
        assert torch.equal(m.lora_add(y.clone(), x.to(dev), ad, ids.to(dev)), out), "in place"
        # an f32 base, as the merged projection's call has it
        f32 = y.float() * 1.001
        got = m._add(f32, x.to(dev), ad, ids.to(dev), torch.full_like(y, 9.0), "test")
        close_on(got, f32.double() + d, mag, dtype)
        assert torch.equal(got[bare], f32[bare].to(dtype))


def _dense64(fmt, w, sc, z, group, xq, xs):
    """x W^T in f64 from the fp8 codes and the packed weight."""
    dev = xq.device
    codes = ((w.to(dev).unsqueeze(-1) >> torch.arange(0, 32, 4, dtype=torch.int32, device=dev)) & 15).flatten(1)
    if fmt in ("sym", "asym"):
        zero = 8.0 if z is None else ((z.to(dev).unsqueeze(-1) >> torch.arange(0, 32, 4, dtype=torch.int32, device=dev)) & 15).flatten(1)
        zero = zero if z is None else zero.double().repeat_interleave(group, 0).t()
        val = (codes.double() - zero) * sc.to(dev).double().repeat_interleave(group, 0).t()
    else:
        e2m1 = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64, device=dev)
        step = torch.pow(2.0, sc.to(dev).double() - 127) if fmt == "mxfp4" else sc.to(dev).double()
        val = e2m1[codes.long()] * step.repeat_interleave(group, 0).t()
        if fmt == "nvfp4":
            val = val * z.to(dev).view(torch.float32).double().unsqueeze(1)
    xv = xq.view(torch.float8_e4m3fn).double() * xs.double().unsqueeze(1)
    return xv @ val.t().contiguous()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt,M,slices", [("sym", 130, [2048, 512]), ("sym", 1100, [2048, 512]), ("asym", 130, [2048, 512]), ("asym", 1100, [8192, 8192]),
                                          ("mxfp4", 130, [2048, 512]), ("mxfp4", 1100, [2048, 512]), ("nvfp4", 130, [2048, 512]),
                                          ("nvfp4", 1100, [2048, 512])])
def test_linear_lora_of_prompts(kernels, dev, dtype, fmt, M, slices):
    """Sizes whose projection runs in the operand order of the GEMM, its f32 epilogue among them, against 64 bits from the
    packed weights. The projection's own error: 1e-4 of its largest output (test_gpu_dense.py)."""
    m = _lora()
    K, rank, L, N = 512, 16, 4, sum(slices)
    e2 = fmt in ("mxfp4", "nvfp4")
    if fmt == "mxfp4":
        (w, sc), z, group = synth.mxfp4_weight(N, K, seed=N), None, 32
    elif fmt == "nvfp4":
        w, sc, z = synth.nvfp4_weight(N, K, seed=N)
        z, group = z.view(torch.int32), 16
    else:
        w, sc, z = synth.int4_weight(N, K, 128, seed=N, asym=fmt == "asym", scale_floor=1e-4)
        group = 128
    a, b, s = make(L, rank, K, slices, dtype, seed=M)
    ad = m.LoraAdapters(*to(dev, a, b, s), slices)
    x = synth.activations(M, K, seed=M, dtype=dtype)
    ids = (torch.arange(M) * 5 // M).int() - 1
    args = kernels.repack_w4(w.to(dev), e2), sc.to(dev), None if z is None else z.to(dev), group, ad, ids.to(dev)
    out = m.w4a8_linear_lora(x.to(dev), *args, weight_is_e2m1=e2)
    xq, xs = kernels.act_quant(x.to(dev))
    base = _dense64(fmt, w, sc, z, group, xq, xs)
    d, mag = delta_on(dev, x, a, b, s, slices, ids)
    close_on(out, base + d, mag, dtype, 1e-4 * base.abs().max().item())
    assert ((out.double() - (base + d).to(dtype).double()).norm() / (base + d).norm()).item() <= 5e-4
    assert torch.equal(out, m.w4a8_linear_lora(x.to(dev), *args, weight_is_e2m1=e2, x_fp8=xq, act_scales=xs))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [1, 40, 100])
def test_an_infinity_in_x_a_is_nan_in_its_slice(dev, dtype, M):
    """An infinite x A^T, from a weight or from x: NaN in all of that row's slice; the row's other slices and the other
    rows keep every bit. One in B: its column alone is not finite."""
    m = _lora()
    K, rank, slices = 128, 16, [64, 48]
    a, b, s = make(3, rank, K, slices, dtype, seed=M)
    g = torch.Generator().manual_seed(M)
    x, y = (torch.randn(M, K, generator=g) + 3).to(dtype), torch.randn(M, sum(slices), generator=g).to(dtype)
    ids = ((torch.arange(M) + 1) % 4 - 1).int()  # row 0: adapter 0
    run = lambda x, a, b: m.lora_add(y.to(dev), x.to(dev), m.LoraAdapters(*to(dev, a, b, s), slices), ids.to(dev)).cpu()  # noqa: E731
    want = run(x, a, b)
    a2, b2 = a.clone(), b.clone()
    a2[0, rank + 2, 7] = float("inf")  # the second slice's
    got = run(x, a2, b)
    rows = ids == 0
    assert torch.isnan(got[rows][:, 64:]).all() and torch.equal(got[rows][:, :64], want[rows][:, :64]) and torch.equal(got[~rows], want[~rows])
    b2[0, 5, 3] = float("-inf")
    got = run(x, a, b2)
    keep = torch.ones(M, sum(slices), dtype=torch.bool)
    keep[rows, 5] = False
    assert not torch.isfinite(got[~keep]).any() and torch.equal(got[keep], want[keep])
    x2 = x.clone()
    x2[0, 9] = float("inf")
    got = run(x2, a, b)
    assert torch.isnan(got[0]).all() and torch.equal(got[1:], want[1:])


@pytest.mark.gpu
@pytest.mark.parametrize("inplace", [True, False])
def test_outputs_past_4_gib(dev, inplace):
    """Rows past 2^32 bytes of y and of a strided out: the bits that the same rows give in a call of their own."""
    m = _lora()
    dtype, K, slices, rank, M = torch.bfloat16, 64, [16384, 16384 + 16], 16, 65600
    N = sum(slices)
    a, b, s = make(3, rank, K, slices, dtype)
    ad = m.LoraAdapters(*to(dev, a, b, s), slices)
    g = torch.Generator(device=dev).manual_seed(4)
    x = torch.randn(M, K, generator=g, device=dev).to(dtype)
    y = torch.empty(M, N, dtype=dtype, device=dev).normal_(generator=g)
    ids = (torch.arange(M, device=dev) * 5 // M).int() - 1
    assert y.numel() * 2 > 1 << 32
    pick = [slice(0, 2048), slice(M // 2, M // 2 + 2048), slice(M - 2048, M)]
    before = [y[p].clone() for p in pick]
    out = y if inplace else torch.empty(M, N + 48, dtype=dtype, device=dev)[:, 16:N + 16]
    m.lora_add(y, x, ad, ids, out=out)
    for p, t in zip(pick, before):
        # more than 64 rows and as many parts of K: the same sums
        assert torch.equal(out[p], m.lora_add(t, x[p].contiguous(), ad, ids[p].contiguous(), out=torch.empty_like(t)))
        assert inplace or torch.equal(y[p], t)
