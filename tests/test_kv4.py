"""The 4-bit key/value cache and its attention (quant/kv4.py): what is refused, on the CPU, and on the GPU
the cache's contents against the formulas and attention against 64-bit attention over the cached values.

Tolerances. Codes, steps and least values follow from exact f32 steps and are compared for equality.
Attention's output is rounded once (2^-8 of the value for bf16, 2^-11 for fp16). Before that: scores are f32
sums of four (D = 128) MFMA steps of at most 31 sum|q| s, about 3e-5 on a score of these sizes, which moves
the output by twice that of the largest cached value; and p s enters its product within 2^-18, or for more
than 16 columns of bf16 within 2^-12 on the codes' distance from 7.5, that is 2^-12 (2.5e-4) of half a
vector's range, which the largest cached value bounds. Together 2e-4 of it, and 3.5e-4 for bf16. (fp16's 2^-25 for results
below 2^-14 is far inside that, but for cached values below 1e-4, where it is allowed on top.)"""
import math

import pytest
import torch

from conftest import pkg

DTYPES = [torch.bfloat16, torch.float16]


def _kv4():
    return pkg("quant.kv4")


# ------------------------------------------------------------------------------------------------
# the formulas, in 64 bits where nothing is rounded to 32
# ------------------------------------------------------------------------------------------------
def ref_quantize(x):
    """(..., D) -> codes, step, least (f64)."""
    f = x.float()
    lo, hi = f.amin(-1), f.amax(-1)
    raw = torch.maximum((hi - lo) / torch.full_like(lo, 15.0), torch.maximum(hi, -lo) * 2.0 ** -14)
    s = raw.to(x.dtype).float().clamp_min(2.0 ** -24 if x.dtype == torch.float16 else 2.0 ** -126)
    c = torch.round((f - lo.unsqueeze(-1)) / s.unsqueeze(-1)).clamp(0, 15)
    bad = ~torch.isfinite(f).all(-1) | ~torch.isfinite(s) | ~torch.isfinite(raw)
    c[bad] = 0
    nan = torch.full_like(s, math.nan)
    return c.double(), torch.where(bad, nan, s).double(), torch.where(bad, nan, lo).double()


def ref_values(x):
    c, s, m = ref_quantize(x)
    return c * s.unsqueeze(-1) + m.unsqueeze(-1)


def cache_values(cache):
    """Every slot's values, (pages, heads, page, D) f64 k and v, from the documented layout."""
    k, v = cache.k.cpu(), cache.v.cpu()
    kc = torch.stack([k & 15, k >> 4], -1).flatten(-2).double()
    j = torch.arange(8, dtype=torch.int32) * 4
    vc = ((v.unsqueeze(3) >> j.view(1, 1, 1, 8, 1)) & 15).flatten(2, 3).double()
    out = []
    for c, sc in ((kc, cache.k_scale), (vc, cache.v_scale)):
        sc = sc.cpu().double()
        out.append(c * sc[..., :1] + sc[..., 1:])
    return out


def ref_attention(q, kv, table, page, lens, news, scale, causal=True, window=0):
    """q (T, Hq, D) and per-slot values (pages, H, page, D) -> out, lse in f64."""
    k, v = kv
    H = k.shape[1]
    T, Hq, D = q.shape
    G = Hq // H
    out = torch.zeros(T, Hq, D, dtype=torch.float64)
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64)
    row = 0
    for b, (n, new) in enumerate(zip(lens, news)):
        if n > 0 and new > 0:
            ids = table[b, :(n + page - 1) // page].long()
            kb = k[ids].transpose(0, 1).flatten(1, 2)[:, :n].repeat_interleave(G, 0)
            vb = v[ids].transpose(0, 1).flatten(1, 2)[:, :n].repeat_interleave(G, 0)
            x = torch.einsum("thd,hnd->htn", q[row:row + new].double(), kb) * scale
            pos = torch.arange(n - new, n).unsqueeze(1)
            key = torch.arange(n).unsqueeze(0)
            see = key <= pos if causal else torch.ones(new, n, dtype=torch.bool)
            if window:
                see = see & (key > pos - window)
            x = x.masked_fill(~see, -math.inf)
            vb = vb.unsqueeze(1)
            p = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-1e300)).masked_fill(~see, 0.0)
            s = p.sum(-1, keepdim=True)
            # a masked value is not part of the sum, whatever it is
            o = torch.where(see[None, :, :, None], p.unsqueeze(-1) * vb, 0.0).sum(2) if n * new * Hq * D < 1 << 24 else \
                torch.matmul(p, vb.squeeze(1))
            o = torch.where(s == 0, 0.0, o / s)
            out[row:row + new] = o.transpose(0, 1)
            lse[row:row + new] = (x.amax(-1).clamp_min(-1e300) + torch.log(s.squeeze(-1))).transpose(0, 1)
        row += new
    return out, lse


class Setup:
    """A cache with the sequences' tokens appended, their last `news` of them to be attended from."""

    def __init__(self, dev, dtype, D, H, page, lens, news, seed=0, spare=2, scale=1.0):
        kv4 = _kv4()
        g = torch.Generator().manual_seed(seed)
        self.page, self.lens, self.news, self.dev = page, lens, news, dev
        count = [-(-n // page) for n in lens]
        pages = max(1, sum(count) + spare)
        perm = torch.randperm(pages, generator=g).int()
        width = max(1, max(count))
        self.table = torch.full((len(lens), width), 2 ** 31 - 1, dtype=torch.int32)  # past a sequence's end: nothing
        at = 0
        for b, c in enumerate(count):
            self.table[b, :c] = perm[at:at + c]
            at += c
        self.cache = kv4.KV4Cache(pages, page, H, D, dtype, dev)
        # what was in the memory before: NaN scales and arbitrary codes
        self.cache.k.random_(0, 256)
        self.cache.v.random_(-2 ** 31, 2 ** 31 - 1)
        self.cache.k_scale.fill_(math.nan)
        self.cache.v_scale.fill_(math.inf)
        self.k = (torch.randn(sum(lens), H, D, generator=g) * scale + torch.randn(H, D, generator=g)).to(dtype)
        self.v = (torch.randn(sum(lens), H, D, generator=g) * scale * 0.5).to(dtype)
        self.cu_all = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)
        self.seq = torch.tensor(lens, dtype=torch.int32)
        self.cu = torch.tensor([sum(news[:i]) for i in range(len(news) + 1)], dtype=torch.int32)
        self.d_table, self.d_seq, self.d_cu = self.table.to(dev), self.seq.to(dev), self.cu.to(dev)
        if sum(lens):
            kv4.kv4_append(self.cache, self.k.to(dev), self.v.to(dev), self.d_table, self.cu_all.to(dev), self.d_seq)

    def q(self, Hq, seed=1, scale=1.0):
        g = torch.Generator().manual_seed(seed)
        return (torch.randn(sum(self.news), Hq, self.cache.head_dim, generator=g) * scale).to(self.cache.dtype)

    def attend(self, q, **kw):
        return _kv4().kv4_attention(q.to(self.dev), self.cache, self.d_table, self.d_cu, self.d_seq, **kw)

    def check(self, q, what="", causal=True, window=0, **kw):
        D = self.cache.head_dim
        out, lse = self.attend(q, causal=causal, window=window, return_lse=True, **kw)
        kv = cache_values(self.cache)
        ref, rl = ref_attention(q, kv, self.table, self.page, self.lens, self.news, kw.get("sm_scale", D ** -0.5), causal, window)
        eps = 2.0 ** (-8 if q.dtype == torch.bfloat16 else -11)
        vmax = self.v.float().abs().max().item() if self.v.numel() else 0.0
        err = (out.cpu().double() - ref).abs() - eps * ref.abs() - (3.5e-4 if q.dtype == torch.bfloat16 else 2e-4) * vmax - 2.0 ** -25
        assert not torch.isnan(out).any(), what
        assert err.max().item() <= 0 if err.numel() else True, f"{what}: off by {err.max().item():.3e} past the tolerance"
        lf = torch.isfinite(rl)
        assert torch.equal(torch.isfinite(lse.cpu()), lf), what
        if lf.any():
            # A score is s (q c) + m sum(q): both terms may be far larger than it, up to a key's range times sum|q|, and
            # that is at most twice the largest key value times sum|q|. Each passes about eight f32 roundings (the
            # products' four steps, the two terms, the scale, M and the logarithm of the sum), 2^-24 of it each.
            most = 2 * self.k.double().abs().max().item() * q.double().abs().sum(-1).max().item() * kw.get("sm_scale", D ** -0.5)
            assert (lse.cpu().double() - rl)[lf].abs().max().item() < 2e-4 + 2.0 ** -21 * most, what
        return out


# ------------------------------------------------------------------------------------------------
# CPU: refusals
# ------------------------------------------------------------------------------------------------
def test_cache_refusals():
    kv4 = _kv4()
    with pytest.raises(TypeError, match="bf16 or fp16"):
        kv4.KV4Cache(4, 16, 2, 128, torch.float32, "cpu")
    with pytest.raises(ValueError, match="64, 128 or 256"):
        kv4.KV4Cache(4, 16, 2, 96, device="cpu")
    for page in (0, 8, 24, 131072):
        with pytest.raises(ValueError, match="power of two"):
            kv4.KV4Cache(4, page, 2, 128, device="cpu")
    with pytest.raises(ValueError):
        kv4.KV4Cache(0, 16, 2, 128, device="cpu")
    c = kv4.KV4Cache(4, 32, 2, 128, device="cpu")
    assert c.nbytes == 4 * 32 * 2 * 2 * (64 + 4)
    again = kv4.KV4Cache.from_tensors(c.k, c.v, c.k_scale, c.v_scale)
    assert again.k is c.k and (again.num_pages, again.page_size, again.num_kv_heads, again.head_dim) == (4, 32, 2, 128)
    with pytest.raises(ValueError, match="v must be"):
        kv4.KV4Cache.from_tensors(c.k, c.v[:, :, :2], c.k_scale, c.v_scale)
    with pytest.raises(ValueError, match="contiguous"):
        kv4.KV4Cache.from_tensors(c.k, c.v, c.k_scale, c.v_scale.transpose(0, 1).contiguous().transpose(0, 1))
    with pytest.raises(TypeError):
        kv4.KV4Cache.from_tensors(c.k.int(), c.v, c.k_scale, c.v_scale)


def test_calls_on_the_cpu_are_refused():
    kv4 = _kv4()
    c = kv4.KV4Cache(4, 32, 2, 128, device="cpu")
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32)  # noqa: E731
    x = torch.zeros(1, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="on the GPU"):
        kv4.kv4_append(c, x, x, i32([0]).view(1, 1), i32(0, 1), i32(1))
    with pytest.raises(RuntimeError, match="on the GPU"):
        kv4.kv4_read(c, i32([0]).view(1, 1), i32(0, 1), i32(1), 1)
    with pytest.raises(RuntimeError, match="on the GPU"):
        kv4.kv4_attention(x, c, i32([0]).view(1, 1), i32(0, 1), i32(1))
    with pytest.raises(TypeError, match="as the cache is"):
        kv4.kv4_append(c, x.half(), x, i32([0]).view(1, 1), i32(0, 1), i32(1))
    with pytest.raises(ValueError, match="query heads"):
        kv4.kv4_attention(torch.zeros(1, 3, 128, dtype=torch.bfloat16), c, i32([0]).view(1, 1), i32(0, 1), i32(1))


def test_abi_refuses_outputs_that_overlap():
    """Host checks of the C entry point, with pointers that are never read: what passes them ends at the workspace."""
    lib = pkg("_abi").load()
    P = 1 << 20

    def attend(T, Hq, ldo, ho, D=128):
        rc = lib.w4a8_kv4_attention(P, 0, Hq * D, D, T, Hq, 1, D, P, P, P, P, 16, 16, P, 1 << 12, 1 << 12, P, P, 1, 1.0, 1, 0,
                                    1, 1 << 16, P, ldo, ho, None, None, 0, None)
        assert rc == 1
        return lib.w4a8_last_error()

    for T, Hq, ldo, ho in ((2, 4, 0, 128), (2, 4, 512, 0), (2, 4, 504, 128), (2, 4, 512, 120), (2, 4, 128, 248), (2, 1, 120, 128),
                           (1, 2, 0, 120), (3, 2, -256, 128)):
        assert b"overlap" in attend(T, Hq, ldo, ho), (T, Hq, ldo, ho)
    for T, Hq, ldo, ho in ((2, 4, 512, 128), (2, 4, 128, 256), (2, 4, 1024, 256), (2, 4, 136, 512), (2, 1, 128, 0), (1, 4, 0, 128),
                           (1, 1, 0, 0)):
        assert b"workspace" in attend(T, Hq, ldo, ho), (T, Hq, ldo, ho)


def test_grids_past_32_bits_are_refused():
    """Sizes whose launch would not fit, refused by the host, and bounds of a call that do not size its grid."""
    if torch.cuda.is_available():
        pytest.skip("the pointers are not real")
    lib = pkg("_abi").load()
    P = 1 << 20
    rows = (1 << 31) - 256
    rc = lib.w4a8_kv4_append(P, 64, 64, P, 64, 64, 0, rows, 1, 64, P, P, P, P, 16, 16, P, 4, 4, P, P, 1, None)
    assert rc == 2 and b"w4a8_kv4_append: past its index ranges" in lib.w4a8_last_error()
    rc = lib.w4a8_kv4_read(P, P, P, P, 0, 16, 16, 1, 64, P, 4, 4, P, P, 1, rows, P, P, None)
    assert rc == 2 and b"w4a8_kv4_read: past its index ranges" in lib.w4a8_last_error()
    # 256 channels: 64 columns a workgroup
    rows = (1 << 30) - 1
    rc = lib.w4a8_kv4_attention(P, 0, 256, 256, rows, 1, 1, 256, P, P, P, P, 16, 16, P, 4, 4, P, P, 1, 1.0, 1, 0, rows, 64, P,
                                256, 256, None, None, 0, None)
    assert rc == 2 and b"past its index ranges" in lib.w4a8_last_error()
    rc = lib.w4a8_kv4_attention(P, 0, 64 * 40000, 64, 1, 40000, 1, 64, P, P, P, P, 16, 16, P, 4, 4, P, P, 1, 1.0, 1, 0, 1, 64,
                                P, 64 * 40000, 64, None, None, 0, None)
    assert rc == 1 and b"up to 32768" in lib.w4a8_last_error()
    f = lib.w4a8_kv4_attention_workspace_bytes
    assert f(4, 40000, 1, 64, 1, 1, 64) == -1
    assert f(4, 8, 8, 128, 1, (1 << 31) - 1, 1 << 17) == f(4, 8, 8, 128, 1, 4, 1 << 17) > 0


def test_abi_refuses_before_any_launch():
    """Host checks of the C entry points, with pointers that are never read."""
    lib = pkg("_abi").load()
    P = 1 << 20

    def attend(dtype=0, ldq=4096, hq=128, T=4, Hq=32, H=8, D=128, kc=P, pages=16, page=16, table=P, ldt=4, width=4, cu=P,
               B=2, window=0, max_q=1, max_kv=64, out=P, ws=None, ws_bytes=0, scale=1.0):
        rc = lib.w4a8_kv4_attention(P, dtype, ldq, hq, T, Hq, H, D, kc, P, P, P, pages, page, table, ldt, width, cu, P, B,
                                    scale, 1, window, max_q, max_kv, out, 4096, 128, None, ws, ws_bytes, None)
        return rc, lib.w4a8_last_error()

    for kw, code, msg in ((dict(dtype=2), 1, b"bf16 or fp16"), (dict(D=96), 2, b"64, 128 or 256"),
                          (dict(page=24), 2, b"power of two"), (dict(page=8), 2, b"power of two"),
                          (dict(Hq=12, H=8), 1, b"query heads"), (dict(Hq=4, H=8), 1, b"query heads"),
                          (dict(T=-1), 1, b"sizes"), (dict(pages=0), 1, b"sizes"), (dict(B=65536), 2, b"index ranges"),
                          (dict(pages=1 << 28), 2, b"index ranges"), (dict(width=1 << 28), 2, b"index ranges"),
                          (dict(scale=0.0), 1, b"positive"), (dict(scale=-1.0), 1, b"positive"),
                          (dict(scale=float("nan")), 1, b"positive"), (dict(scale=float("inf")), 1, b"positive"),
                          (dict(T=1 << 26), 2, b"index ranges"), (dict(window=-1), 1, b"window"), (dict(max_kv=-1), 1, b"max_kv"),
                          (dict(kc=P + 8), 1, b"aligned"), (dict(kc=None), 1, b"aligned"), (dict(cu=None), 1, b"cu"),
                          (dict(table=None), 1, b"page table"), (dict(ldt=3), 1, b"page table"),
                          (dict(ldq=4100), 1, b"multiples of 8"), (dict(hq=4), 1, b"multiples of 8"),
                          (dict(out=P + 2), 1, b"aligned"),
                          (dict(max_kv=1 << 16, width=1 << 12, ldt=1 << 12), 1, b"workspace")):
        rc, err = attend(**kw)
        assert rc == code and msg in err, (kw, rc, err)
    # nothing to do
    assert attend(T=0)[0] == 0 and attend(B=0)[0] == 0
    bytes_for = lib.w4a8_kv4_attention_workspace_bytes
    assert bytes_for(4, 32, 8, 96, 2, 1, 64) == -1 and bytes_for(4, 12, 8, 128, 2, 1, 64) == -1
    assert bytes_for(0, 32, 8, 128, 0, 0, 0) == 0 and bytes_for(1, 32, 8, 128, 1, 1, 32) == 0
    assert bytes_for(1, 32, 8, 128, 1, 1, 1 << 17) > 0

    rc = lib.w4a8_kv4_append(P, 1024, 128, P, 1024, 100, 0, 4, 8, 128, P, P, P, P, 16, 16, P, 4, 4, P, P, 2, None)
    assert rc == 1 and b"multiples of 8" in lib.w4a8_last_error()
    rc = lib.w4a8_kv4_append(P, 1024, 128, P, 1024, 128, 0, 4, 8, 32, P, P, P, P, 16, 16, P, 4, 4, P, P, 2, None)
    assert rc == 2 and b"64, 128 or 256" in lib.w4a8_last_error()
    rc = lib.w4a8_kv4_read(P, P, P, P, 0, 16, 16, 8, 128, P, 4, 4, P, P, 2, 4, None, P, None)
    assert rc == 1 and b"aligned" in lib.w4a8_last_error()


# ------------------------------------------------------------------------------------------------
# GPU: the cache
# ------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,H,page", [(64, 3, 16), (128, 8, 32), (256, 1, 16)])
def test_append_and_read_match_the_formulas(dev, dtype, D, H, page):
    """Whole sequences in one call, of lengths that end anywhere in a block and a page."""
    lens = [1, 7, 8, 9, 15, 16, 17, 40, 2 * page + 3]
    s = Setup(dev, dtype, D, H, page, lens, lens)
    k, v = _kv4().kv4_read(s.cache, s.d_table, s.cu_all.to(dev), s.d_seq, sum(lens))
    for got, x in ((k, s.k), (v, s.v)):
        assert torch.equal(got.cpu(), ref_values(x).to(torch.float32).to(dtype))
    ck, cv = cache_values(s.cache)
    row = 0
    for b, n in enumerate(lens):
        pos = torch.arange(n)
        pages, slot = s.table[b, pos // page].long(), pos % page
        assert torch.equal(ck[pages, :, slot], ref_values(s.k[row:row + n]))
        assert torch.equal(cv[pages, :, slot], ref_values(s.v[row:row + n]))
        row += n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_appended_one_by_one_give_the_same_cache(dev, dtype):
    """Steps of 1 to 5 tokens per sequence against one call, from strided views of a merged qkv."""
    kv4 = _kv4()
    H, D, page, n = 2, 128, 16, 37
    whole = Setup(dev, dtype, D, H, page, [n, n], [n, n])
    steps = kv4.KV4Cache(whole.cache.num_pages, page, H, D, dtype, dev)
    for t in (steps.k, steps.v, steps.k_scale, steps.v_scale):
        t.copy_({id(steps.k): whole.cache.k, id(steps.v): whole.cache.v, id(steps.k_scale): whole.cache.k_scale,
                 id(steps.v_scale): whole.cache.v_scale}[id(t)])
    # every slot of the sequences holds something else before
    for b in range(2):
        steps.k[whole.table[b].long().to(dev)] = 0x5a
        steps.v[whole.table[b].long().to(dev)] = 0x5a5a5a5a
        steps.k_scale[whole.table[b].long().to(dev)] = math.nan
        steps.v_scale[whole.table[b].long().to(dev)] = math.nan
    qkv = torch.zeros(2 * n, (4 + 2 * H) * D, dtype=dtype, device=dev)
    k, v = qkv[:, 4 * D:(4 + H) * D].view(-1, H, D), qkv[:, (4 + H) * D:].view(-1, H, D)
    k.copy_(whole.k)
    v.copy_(whole.v)
    assert not k.is_contiguous()
    at = 0
    for step in (1, 5, 1, 3, 8, 1, 9, 2, 7):
        rows = torch.cat([torch.arange(at, at + step), torch.arange(n + at, n + at + step)]).to(dev)
        kk, vv = qkv[rows][:, 4 * D:(4 + H) * D].view(-1, H, D), qkv[rows][:, (4 + H) * D:].view(-1, H, D)
        at += step
        kv4.kv4_append(steps, kk, vv, whole.d_table, torch.tensor([0, step, 2 * step], dtype=torch.int32, device=dev),
                       torch.tensor([at, at], dtype=torch.int32, device=dev))
    assert at == n
    a, b = cache_values(whole.cache), cache_values(steps)
    for x, y in zip(a, b):
        for q in range(2):
            pos = torch.arange(n)
            pages, slot = whole.table[q, pos // page].long(), pos % page
            assert torch.equal(x[pages, :, slot], y[pages, :, slot])
        # the rest of the last block: as it was
    last = whole.table[0, -1].item()
    assert torch.isnan(steps.k_scale[last, :, n % page:]).all() and torch.isnan(steps.v_scale[last, :, n % page:]).all()
    words = steps.v[last, :, (n % page) // 8].cpu()
    assert torch.equal((words >> (4 * (n % 8))) & 15, (torch.tensor(0x5a5a5a5a, dtype=torch.int32) >> (4 * (n % 8))).expand_as(words) & 15)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_special_vectors(dev, dtype):
    """Constants, zeros, one outlier, the type's extremes, subnormals, and vectors with an infinity or NaN."""
    kv4 = _kv4()
    D, page = 128, 16
    fi = torch.finfo(dtype)
    g = torch.Generator().manual_seed(3)
    rows = [torch.zeros(D), torch.full((D,), 1.5), torch.full((D,), -3.25e-3), torch.full((D,), 1e-5),
            torch.cat([torch.full((1,), 1000.0), torch.zeros(D - 1)]), torch.linspace(-1, 1, D), torch.randn(D, generator=g) * 1e-6,
            torch.cat([torch.full((D // 2,), 7.0), torch.full((D // 2,), 7.0 + 7.0 * fi.eps)]),
            torch.cat([torch.full((1,), fi.max), torch.full((1,), fi.min), torch.zeros(D - 2)]),
            torch.full((D,), fi.smallest_normal), torch.cat([torch.full((1,), math.inf), torch.ones(D - 1)]),
            torch.cat([torch.ones(D - 1), torch.full((1,), math.nan)]), torch.full((D,), -math.inf), torch.randn(D, generator=g)]
    x = torch.stack(rows).to(dtype).unsqueeze(1)
    n = x.shape[0]
    cache = kv4.KV4Cache(2, page, 1, D, dtype, dev)
    tab = torch.tensor([[1]], dtype=torch.int32, device=dev)
    cu, seq = torch.tensor([0, n], dtype=torch.int32, device=dev), torch.tensor([n], dtype=torch.int32, device=dev)
    kv4.kv4_append(cache, x.to(dev), x.to(dev), tab, cu, seq)
    k, v = kv4.kv4_read(cache, tab, cu, seq, n)
    ref = ref_values(x)
    assert torch.equal(torch.isnan(ref), torch.isnan(k.cpu()))
    assert torch.equal(torch.isnan(ref).any(-1).flatten(), torch.isnan(k.cpu()).all(-1).flatten())
    want = ref.float().to(dtype)
    for got in (k, v):
        assert torch.equal(torch.nan_to_num(got.cpu(), nan=123.0), torch.nan_to_num(want, nan=123.0))
    ck, cv = cache_values(cache)
    assert torch.equal(torch.nan_to_num(ck[1, 0, :n], nan=123.0), torch.nan_to_num(ref[:, 0], nan=123.0))
    assert torch.equal(torch.nan_to_num(cv[1, 0, :n], nan=123.0), torch.nan_to_num(ref[:, 0], nan=123.0))
    # what fits is within half a step
    c, st, _ = ref_quantize(x)
    fits = torch.isfinite(st).flatten()
    assert ((ref - x.double()).abs().squeeze(1)[fits] <= 0.55 * st[fits]).all()
    assert int(c.max()) == 15


@pytest.mark.gpu
def test_bad_pages_and_lengths_touch_nothing(dev):
    """Pages that do not exist, tokens past the table and before the sequence: not written, read as NaN; the
    cache has guard pages on either side that stay as they are."""
    kv4 = _kv4()
    H, D, page = 2, 64, 16
    cache = kv4.KV4Cache(4, page, H, D, torch.bfloat16, dev)
    for t in (cache.k, cache.v):
        t.fill_(17)
    cache.k_scale.fill_(3.0)
    cache.v_scale.fill_(3.0)
    x = torch.randn(40, H, D, device=dev).bfloat16()
    # page 4 and -1 do not exist; sequence 1 has 20 rows but a table of 1 page in use; 2 has more rows than tokens
    table = torch.tensor([[4], [-1], [1]], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 10, 30, 40], dtype=torch.int32, device=dev)
    seq = torch.tensor([10, 20, 4], dtype=torch.int32, device=dev)
    kv4.kv4_append(cache, x, x, table, cu, seq)
    k, v = kv4.kv4_read(cache, table, cu, seq, 40)
    torch.cuda.synchronize()
    assert torch.isnan(k[:36]).all() and torch.isnan(v[:36]).all()
    want = ref_values(x[36:].cpu()).float().bfloat16()
    assert torch.equal(k[36:].cpu(), want) and torch.equal(v[36:].cpu(), want)
    for p in (0, 2, 3):
        assert (cache.k[p] == 17).all() and (cache.v[p] == 17).all() and (cache.k_scale[p] == 3).all()
    assert (cache.k[1, :, 4:] == 17).all() and (cache.v_scale[1, :, 4:] == 3).all()
    # attention: rows that would read them are NaN, the others are not
    q = torch.randn(40, 4, D, device=dev).bfloat16()
    for kw in ({}, {"max_q": 1}, {"max_q": 40, "max_kv": 4}):
        out = kv4.kv4_attention(q, cache, table, cu, seq, **kw)
        torch.cuda.synchronize()
        assert torch.isnan(out[:30]).all()
        assert (out[30:36] == 0).all(), "rows before the first token see nothing"
        assert torch.isfinite(out[36:]).all() and (out[36:] != 0).any()
    # a length past the table: NaN where it is seen, and the rows that end before the table's end are whole
    seq2 = torch.tensor([0, 0, 20], dtype=torch.int32, device=dev)
    cu2 = torch.tensor([0, 0, 0, 12], dtype=torch.int32, device=dev)
    out = kv4.kv4_attention(q[:12], cache, table, cu2, seq2)
    assert torch.isfinite(out[:8]).all() and torch.isnan(out[8:]).all()


# ------------------------------------------------------------------------------------------------
# GPU: attention
# ------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,H,G,page", [(128, 2, 4, 16), (128, 1, 1, 64), (64, 2, 3, 32), (256, 1, 2, 16), (128, 1, 16, 128), (64, 1, 17, 16), (128, 1, 128, 32)])
def test_decode(dev, dtype, D, H, G, page):
    lens = [1, 2, 31, 32, 33, 64, 100, 257, 1000, 0, 5]
    s = Setup(dev, dtype, D, H, page, lens, [1] * len(lens))
    s.check(s.q(H * G), "max_q=1", max_q=1)
    s.check(s.q(H * G), "bounds of nothing", max_q=1, max_kv=1)
    s.check(s.q(H * G), "no bounds")
    s.check(s.q(H * G), "window", max_q=1, window=40)
    s.check(s.q(H * G), "window 1", max_q=1, window=1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,H,G,page", [(128, 2, 4, 16), (128, 1, 1, 64), (64, 2, 3, 32), (256, 1, 2, 16)])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 50), (False, 0), (False, 33)])
def test_prompts(dev, dtype, D, H, G, page, causal, window):
    lens = [1, 33, 0, 64, 130, 200, 17]
    news = [1, 33, 0, 20, 130, 7, 3]
    s = Setup(dev, dtype, D, H, page, lens, news, seed=5)
    s.check(s.q(H * G), "whole", causal, window)
    s.check(s.q(H * G), "bounds", causal, window, max_q=130, max_kv=200)
    s.check(s.q(H * G), "bounds too low", causal, window, max_q=2, max_kv=8)
    s.check(s.q(H * G), "scale", causal, window, sm_scale=0.25)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_long_contexts_in_splits(dev, dtype):
    s = Setup(dev, dtype, 128, 2, 64, [20011, 7, 4096], [1, 1, 1], seed=9)
    s.check(s.q(8), "decode", max_q=1, max_kv=20011)
    s = Setup(dev, dtype, 64, 1, 16, [6001, 300], [33, 50], seed=10)
    s.check(s.q(2), "chunk", max_q=50, max_kv=6001)
    s.check(s.q(2), "chunk, window", window=1000, max_q=50, max_kv=6001)


@pytest.mark.gpu
def test_window_past_2_30_keys(dev):
    """A table that repeats two pages: 2^30 + 65536 keys. Only the last 7 slots of the first page have large scores, and
    a window of 2^30 + 7 keys begins with them; one of 2^30 does not reach them. exp(60) against 2^30 keys of score 0."""
    kv4 = _kv4()
    D, page, width = 64, 65536, 16385
    cache = kv4.KV4Cache(2, page, 1, D, device=dev)  # zeros: keys of score 0, values 0
    k = torch.zeros(page, 1, D, dtype=torch.bfloat16)
    v = torch.zeros(page, 1, D, dtype=torch.bfloat16)
    k[-7:] = 15.0 / 16
    v[-7:, :, 0] = 15.0
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    kv4.kv4_append(cache, k.to(dev), v.to(dev), i32([1]), i32(0, page), i32(page))
    table = torch.zeros(1, width, dtype=torch.int32, device=dev)
    table[0, 0] = 1
    q = torch.full((1, 1, D), 1.0, dtype=torch.bfloat16, device=dev)
    for window, want in ((2 ** 30 + 7, 15.0), (2 ** 30, 0.0)):
        out = kv4.kv4_attention(q, cache, table, i32(0, 1), i32(width * page), sm_scale=1.0, window=window)
        # the 7 keys' share is 1 - 2^30 / (7 e^60) of the whole, and a row's error is within 3.5e-4 of the largest value
        assert (out[0, 0, 0].float().cpu() - want).abs() <= 15 * (2.0 ** -9 + 3.5e-4)
        assert out[0, 0, 1:].abs().max() <= 15 * 3.5e-4


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [1e-4, 30.0])
def test_small_and_large_values(dev, dtype, scale):
    """Values whose steps are far below fp16's normal range, and scores in the hundreds (one key takes all)."""
    s = Setup(dev, dtype, 128, 1, 16, [70, 200], [1, 30], seed=11, scale=scale)
    s.check(s.q(4), f"scale {scale}", max_q=30)


def check_one_hot(s, q, causal, window, **kw):
    """Scores so far apart that all but the largest have weights below 2^-100, or are equal to it: the output is the mean
    of the values with the largest score."""
    D, dtype = s.cache.head_dim, s.cache.dtype
    kv = cache_values(s.cache)
    out, lse = s.attend(q, causal=causal, window=window, return_lse=True, **kw)
    ref, rl = ref_attention(q, kv, s.table, s.page, s.lens, s.news, kw.get("sm_scale", D ** -0.5), causal, window)
    eps = 2.0 ** (-8 if dtype == torch.bfloat16 else -11)
    vmax = s.v.float().abs().max().item()
    err = (out.cpu().double() - ref).abs() - eps * ref.abs() - (3.5e-4 if dtype == torch.bfloat16 else 2e-4) * vmax
    assert not torch.isnan(out).any() and err.max().item() <= 0, err.max().item()
    # a score's roundings, 16 of 2^-24 of it as in Setup.check, and the f32 result's own
    assert ((lse.cpu().double() - rl).abs() <= 2.0 ** -20 * rl.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,power", [(t, p) for t in DTYPES for p in (20, 23, 24, 25, 30)] + [(torch.bfloat16, 60)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("new", [1, 40])
def test_scores_far_from_zero(dev, dtype, power, sign, new):
    """Keys that are integers 0 .. 15 in channel 0 and 15 in channel 1, or their negatives, and queries that are powers of
    two there: scores are whole multiples of the score of a step, so the largest is shared by a sixteenth of the keys,
    which are in all splits, with steps of V that grow along the sequence."""
    kv4 = _kv4()
    D, n = 64, 700
    s = Setup(dev, dtype, D, 1, 16, [n], [new], seed=21)
    g = torch.Generator().manual_seed(5)
    k = torch.zeros(n, 1, D)
    k[:, 0, 0] = torch.randint(0, 16, (n,), generator=g).float()
    k[:, 0, 1] = 15.0
    s.k = (sign * k).to(dtype)
    s.v = (torch.randn(n, 1, D, generator=g) * torch.logspace(-3, 3, n, base=2.0).view(n, 1, 1)).to(dtype)
    kv4.kv4_append(s.cache, s.k.to(dev), s.v.to(dev), s.d_table, s.cu_all.to(dev), s.d_seq)
    q = torch.zeros(new, 2, D)
    qp = 15 if power <= 30 else power - 15
    q[:, 0, :2] = 2.0 ** qp
    q[:, 1, :2] = 2.0 ** (qp - 1)
    for kw in ({}, {"max_q": 1, "max_kv": 1 << 16}):
        check_one_hot(s, q.to(dtype), True, 0, sm_scale=2.0 ** (power - qp), **kw)
    if dtype == torch.bfloat16 and power == 60:
        q = torch.zeros(new, 2, D)
        q[:, :, :2] = 2.0 ** 90
        check_one_hot(s, q.to(dtype), True, 0)


@pytest.mark.gpu
def test_unseen_tokens_do_not_reach_the_output(dev):
    """A NaN vector among the keys is seen by the rows behind it only; slots past the end, which hold NaN and
    infinite scales in every setup here, by none."""
    kv4 = _kv4()
    s = Setup(dev, torch.bfloat16, 128, 1, 16, [60], [60], seed=12)
    q = s.q(2)
    clean = s.attend(q)
    s.k[40] = math.nan
    s.v[50, 0, 3] = math.inf
    kv4.kv4_append(s.cache, s.k.to(dev), s.v.to(dev), s.d_table, s.cu_all.to(dev), s.d_seq)
    out = s.attend(q)
    assert torch.equal(out[:40], clean[:40]) and torch.isnan(out[40:]).all()
    out = s.attend(q, window=5)
    seen = torch.zeros(60, dtype=torch.bool)
    seen[40:45] = seen[50:55] = True
    assert torch.equal(torch.isnan(out.cpu()).all(-1).all(-1), seen) and torch.equal(torch.isnan(out.cpu()).any(-1).any(-1), seen)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_do_not_depend_on_what_they_do_not_see(dev, dtype):
    """A later token with huge values (its V step 2^25 times the others') in the same tile and the same block of
    columns: the rows before it keep every bit, the rows after it are right."""
    kv4 = _kv4()
    s = Setup(dev, dtype, 128, 1, 16, [60], [60], seed=21)
    s.v *= 1e-3
    kv4.kv4_append(s.cache, s.k.to(dev), s.v.to(dev), s.d_table, s.cu_all.to(dev), s.d_seq)
    q = s.q(2)
    before = s.attend(q)
    s.v[45] *= 2.0 ** 25
    s.k[52] *= 100.0
    kv4.kv4_append(s.cache, s.k.to(dev), s.v.to(dev), s.d_table, s.cu_all.to(dev), s.d_seq)
    after = s.check(q, "outlier")
    assert torch.equal(before[:45], after[:45])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,page", [(65, 16), (300, 32)])
def test_many_sequences(dev, dtype, B, page):
    """More sequences than lanes, empty ones and ones without new tokens among them, in calls of one row and of many."""
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 25, (B,), generator=g).tolist()
    lens[7:20] = [0] * 13
    s = Setup(dev, dtype, 64, 1, page, lens, [min(n, i % 3) for i, n in enumerate(lens)], seed=B)
    k, v = _kv4().kv4_read(s.cache, s.d_table, s.cu_all.to(dev), s.d_seq, sum(lens))
    assert torch.equal(k.cpu(), ref_values(s.k).float().to(dtype)) and torch.equal(v.cpu(), ref_values(s.v).float().to(dtype))
    s.check(s.q(2), "decode", max_q=2)
    # the whole again through the few-rows path, one call per sequence
    for b in (0, 6, 21, B - 1):
        if lens[b]:
            at = sum(lens[:b])
            cu = torch.tensor([0, lens[b]], dtype=torch.int32, device=dev)
            k1, v1 = _kv4().kv4_read(s.cache, s.d_table[b:b + 1], cu, s.d_seq[b:b + 1], lens[b])
            assert torch.equal(k1, k[at:at + lens[b]]) and torch.equal(v1, v[at:at + lens[b]])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_large_append_of_prompts(dev, dtype):
    """Enough rows that a wave looks at 8 of them, prompts that start and end anywhere in a block."""
    lens = [1003, 2, 777, 4001, 13, 8, 1]
    s = Setup(dev, dtype, 128, 2, 16, lens, [1] * 7, seed=3)
    assert sum(lens) * 2 > 8192
    k, v = _kv4().kv4_read(s.cache, s.d_table, s.cu_all.to(dev), s.d_seq, sum(lens))
    assert torch.equal(k.cpu(), ref_values(s.k).float().to(dtype)) and torch.equal(v.cpu(), ref_values(s.v).float().to(dtype))


@pytest.mark.gpu
def test_rows_behind_the_last_sequence_stay(dev):
    s = Setup(dev, torch.float16, 64, 1, 16, [9, 4, 0, 0], [2, 1, 0, 0], seed=13)
    q = torch.cat([s.q(2), torch.full((5, 2, 64), math.nan, dtype=torch.float16)])
    for kw in ({}, {"max_q": 1, "max_kv": 4096}):
        buf = torch.full((8, 4, 64), 7.0, dtype=torch.float16, device=dev)
        got = s.attend(q, out=buf[:, 1:3], **kw)
        assert got.data_ptr() == buf[:, 1:3].data_ptr()
        assert (buf[3:] == 7).all() and (buf[:, 0] == 7).all() and (buf[:, 3] == 7).all()
        assert torch.equal(buf[:3, 1:3], s.attend(s.q(2), **kw))
    k, v = torch.full((8, 1, 64), 5.0, device=dev).half(), torch.full((8, 1, 64), 5.0, device=dev).half()
    before = [t.clone() for t in (s.cache.k, s.cache.v)]
    _kv4().kv4_append(s.cache, k, v, s.d_table, torch.zeros(5, dtype=torch.int32, device=dev), s.d_seq)
    assert torch.equal(before[0], s.cache.k) and torch.equal(before[1], s.cache.v)


@pytest.mark.gpu
def test_captured_step_replays_with_new_lengths(dev):
    """Append and attention of a decode step in one graph, replayed over growing sequences, with eager work
    between: each replay gives what the eager calls give."""
    kv4 = _kv4()
    dtype, D, H, page, B = torch.bfloat16, 128, 2, 16, 3
    cap = 40
    s = Setup(dev, dtype, D, H, page, [cap * page] * B, [1] * B, seed=14)
    seq = torch.zeros(B, dtype=torch.int32, device=dev)
    k, v, q = (torch.zeros(B, h, D, dtype=dtype, device=dev) for h in (H, H, 4 * H))

    def step(cache):
        kv4.kv4_append(cache, k, v, s.d_table, s.d_cu, seq)
        return kv4.kv4_attention(q, cache, s.d_table, s.d_cu, seq, max_q=1)

    other = kv4.KV4Cache.from_tensors(*(t.clone() for t in (s.cache.k, s.cache.v, s.cache.k_scale, s.cache.v_scale)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(s.cache)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(s.cache)
    g = torch.Generator().manual_seed(2)
    for lens in ([1, 17, 0], [2, 18, 600], [33, 19, 601], [34, 640, 602]):
        seq.copy_(torch.tensor(lens, dtype=torch.int32))
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        want = step(other)
        torch.empty(1 << 20, device=dev).normal_()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(s.cache.v, other.v) and torch.equal(s.cache.k, other.k)


@pytest.mark.gpu
def test_calls_on_two_streams_do_not_share_anything(dev):
    s = Setup(dev, torch.bfloat16, 128, 2, 16, [3000, 700], [1, 1], seed=15)
    qs = [s.q(8, seed=i) for i in range(4)]
    want = [s.attend(q, max_q=1) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    d = [q.to(dev) for q in qs]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for q, st in zip(d, streams):
            with torch.cuda.stream(st):
                got.append(_kv4().kv4_attention(q, s.cache, s.d_table, s.d_cu, s.d_seq, max_q=1))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 4])


@pytest.mark.gpu
def test_gpu_refusals(dev):
    kv4 = _kv4()
    c = kv4.KV4Cache(4, 16, 2, 128, device=dev)
    tab = torch.zeros(2, 2, dtype=torch.int32, device=dev)
    cu, seq = torch.tensor([0, 1, 2], dtype=torch.int32, device=dev), torch.ones(2, dtype=torch.int32, device=dev)
    q = torch.zeros(2, 4, 128, dtype=torch.bfloat16, device=dev)
    for args, err in (((tab.long(), cu, seq), TypeError), ((tab, cu[:2], seq), ValueError), ((tab[:1], cu, seq), ValueError),
                      ((tab.cpu(), cu, seq), RuntimeError), ((tab.t(), cu, seq), ValueError)):
        with pytest.raises(err):
            kv4.kv4_attention(q, c, *args)
    with pytest.raises(ValueError, match="out must be"):
        kv4.kv4_attention(q, c, tab, cu, seq, out=torch.empty(2, 4, 64, dtype=torch.bfloat16, device=dev))
    with pytest.raises(RuntimeError, match="overlap"):
        kv4.kv4_attention(q, c, tab, cu, seq, out=torch.empty(1, 4, 128, dtype=torch.bfloat16, device=dev).expand(2, 4, 128))
    with pytest.raises(ValueError, match="window"):
        kv4.kv4_attention(q, c, tab, cu, seq, window=-1)
    with pytest.raises(TypeError, match="as the cache is"):
        kv4.kv4_attention(q.half(), c, tab, cu, seq)
    with pytest.raises(ValueError, match="rows"):
        kv4.kv4_append(c, q[:, :2], q[:1, :2], tab, cu, seq)
    # no tokens and no sequences
    assert kv4.kv4_attention(q[:0], c, tab, cu, seq).shape == (0, 4, 128)
    kv4.kv4_append(c, q[:0, :2], q[:0, :2], tab[:0], cu[:1], seq[:0])
