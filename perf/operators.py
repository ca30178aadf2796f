"""What serving a 4-bit model needs beside its linears, as cases that can be timed and checked: the
low-rank adapters of many requests beside a shared 4-bit projection, and attention over keys and
values that are held in 4 bits themselves.

kind "lora":   y = x W^T + scaling[a] (x A_a^T) B_a^T with a the adapter of each row, through
               lora.w4a8_linear_lora: W in 4 bits and x in fp8 per row as in w4a8_linear, A and B in
               x's type.
kind "add":    y += scaling[a] (x A_a^T) B_a^T on the output of any projection, through lora.lora_add.
kind "append": new keys and values into a paged cache in 4 bits, and those tokens read back, through
               kv4.kv4_append and kv4.kv4_read.
kind "attend": attention of new tokens over such a cache, through kv4.kv4_attention.

A cached vector x of one token and head is stored as codes c in 0..15 with a step s and a least value
m in the model's type, and stands for s c + m:
    m = min x,  s = max((max x - min x) / 15, 2^-14 max |x|), rounded to the type and at least its
    smallest positive value (2^-24 for fp16, 2^-126 for bf16),  c = clamp(rint((x - m) / s), 0, 15).

Sizes are those of the benchmark and the other timed cases (hidden sizes 2560 to 8192, heads of 64
and 128, 8 or 4 key/value heads), from one token of decode to a prompt of 8192 tokens and contexts
of 131072.
"""
from __future__ import annotations

import importlib
import math

import torch

own = False

_PKG = "minisglang-rdna4_amd"
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
_MOST_MACS = 4096 * 4096 * 14336
_MOST_PAIRS = 64 * 5120 * 5120
_MOST_CACHE = 2 * 131072 * 8 * 128


# ------------------------------------------------------------------------------------------------
# the cases
# ------------------------------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # one user's decode step through one projection, with that user's adapter: latency
        dict(name="lora_m1_o_proj", kind="lora", fmt="int4", group=128, dtype="bf16", m=1, k=4096, slices="4096",
             rank=16, adapters=8, used=1, bare=0.0, spread=True),
        # a decode step of 16 users, each with another adapter or none, through the merged q, k and v
        dict(name="lora_m16_qkv", kind="lora", fmt="int4", group=128, dtype="bf16", m=16, k=4096,
             slices="4096+1024+1024", rank=16, adapters=32, used=12, bare=0.2, spread=True),
        # prompts of a few users back to back through the gate and up projection of a smaller AWQ model
        dict(name="lora_m1777_gate_up", kind="lora", fmt="awq", group=128, dtype="fp16", m=1777, k=2560,
             slices="9728+9728", rank=32, adapters=8, used=5, bare=0.1, spread=False),
        # 48 decoding users with large adapters beside a down projection that another path computed
        dict(name="add_m48_down", kind="add", dtype="fp16", m=48, k=14336, slices="4096", rank=64, adapters=64,
             used=40, bare=0.1, spread=True),
        # a chunk of 4096 prompt tokens, gate and up
        dict(name="add_m4096_gate_up", kind="add", dtype="bf16", m=4096, k=4096, slices="14336+14336", rank=16,
             adapters=16, used=6, bare=0.0, spread=False),
        # 64 users' new tokens of one decode step
        dict(name="append_64_users", kind="append", dtype="bf16", heads=8, dim=128, page=16, seqs=64, new=1, most=4000,
             least=0.05),
        # the new tokens of a few prompts, on top of what the cache holds of them
        dict(name="append_prompts", kind="append", dtype="fp16", heads=4, dim=128, page=64, seqs=5, new=1733, most=5000,
             least=0.4),
        # one user's decode step over a short context: latency
        dict(name="attend_1_user", kind="attend", dtype="bf16", heads=8, group=4, dim=128, page=16, seqs=1, new=1,
             most=1999, least=1.0, window=0),
        # a decode step of 64 users whose contexts have all lengths up to 8192
        dict(name="attend_64_users", kind="attend", dtype="bf16", heads=8, group=4, dim=128, page=32, seqs=64, new=1,
             most=8192, least=0.01, window=0),
        # two users with very long documents, on a 70B-sized model's 64 query heads
        dict(name="attend_long", kind="attend", dtype="bf16", heads=8, group=8, dim=128, page=64, seqs=2, new=1,
             most=131072, least=0.9, window=0),
        # chunks of 257 new tokens on top of a context, sliding window, heads of 64 in fp16
        dict(name="attend_chunks", kind="attend", dtype="fp16", heads=8, group=3, dim=64, page=16, seqs=7, new=257,
             most=6001, least=0.05, window=4096),
        # whole prompts: every position is new
        dict(name="attend_prompts", kind="attend", dtype="bf16", heads=8, group=4, dim=128, page=64, seqs=3, new=8192,
             most=8192, least=0.2, window=0),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    """lo..hi, uniform in the logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def _multiple(rng, lo: int, hi: int, step: int) -> int:
    return max(1, _log_int(rng, lo, hi) // step) * step


def draw(rng) -> dict:
    kind = rng.choice(["lora", "lora", "add", "append", "attend", "attend", "attend"])
    case = dict(kind=kind, dtype=rng.choice(["bf16", "fp16"]))
    if kind in ("lora", "add"):
        case["m"] = _log_int(rng, 1, 4096)
        case["rank"] = 8 * _log_int(rng, 1, 16)
        case["adapters"] = _log_int(rng, 1, 128)
        case["used"] = min(case["adapters"], _log_int(rng, 1, 48))
        case["bare"] = rng.choice([0.0, 0.0, 0.2, 0.6])
        case["spread"] = case["m"] <= 64 or rng.random() < 0.2
        case["k"] = _multiple(rng, 1024, 14336, 128)
        case["slices"] = "+".join(str(_multiple(rng, 512, 14336, 16)) for _ in range(rng.choice([1, 1, 2, 3])))
        if kind == "lora":
            case["fmt"] = rng.choice(["int4", "int4", "awq", "mxfp4"])
            case["group"] = 32 if case["fmt"] == "mxfp4" else rng.choice([128, 128, 64, 32])
        while case["m"] * case["k"] * sum(_slices(case)) > _MOST_MACS:
            case["m"] = case["m"] * 3 // 4
        return case
    case["dim"] = rng.choice([64, 128, 128, 128, 256])
    case["heads"] = rng.choice([1, 2, 4, 8, 8])
    case["page"] = rng.choice([16, 16, 32, 64, 128])
    case["least"] = rng.choice([0.01, 0.3, 1.0])
    case["seqs"] = _log_int(rng, 1, 96)
    case["most"] = _log_int(rng, 1, 40000)
    if kind == "append":
        case["new"] = _log_int(rng, 1, 8192)
        cost = lambda: case["seqs"] * (case["most"] + 8 * case["new"]) * case["heads"] * case["dim"] * 2  # noqa: E731
    else:
        case["group"] = rng.choice([1, 2, 3, 4, 5, 8, 16])
        case["new"] = rng.choice([1, 1, 1, _log_int(rng, 2, 16), _log_int(rng, 16, 8192)])
        case["window"] = rng.choice([0, 0, 0, _log_int(rng, 16, 8192)])
        cost = lambda: max(  # noqa: E731
            case["seqs"] * case["most"] * case["heads"] * case["dim"] * 2 / _MOST_CACHE,
            case["seqs"] * min(case["new"], case["most"]) * case["most"] * case["heads"] * case["group"]
            / _MOST_PAIRS) * _MOST_CACHE
    while case["seqs"] > 1 and cost() > _MOST_CACHE:
        case["seqs"] = case["seqs"] * 3 // 4
    while cost() > _MOST_CACHE:
        case["most"], case["new"] = case["most"] * 3 // 4, max(1, case["new"] * 3 // 4)
    return case


# ------------------------------------------------------------------------------------------------
# what a case's sizes imply (the same for every seed)
# ------------------------------------------------------------------------------------------------
def _lengths(case: dict) -> list[tuple[int, int]]:
    """(length with the new tokens, new tokens) of each sequence: lengths spread from least * most to
    most, the longest first."""
    out = []
    for i in range(case["seqs"]):
        f = 1.0 if i == 0 else case["least"] + (1.0 - case["least"]) * ((i * 0.6180339887) % 1.0)
        n = max(1, int(round(case["most"] * f)))
        out.append((n, min(n, case["new"])))
    return out


def _slices(case: dict) -> list[int]:
    """Output widths of the projections that are merged in one, each with a low-rank pair of its own."""
    return [int(w) for w in case["slices"].split("+")]


def _adapter_rows(case: dict) -> list[int]:
    """How many rows the cases' used adapters have, the rows without an adapter last."""
    m, used = case["m"], case["used"]
    bare = int(m * case["bare"])
    used = max(1, min(used, m - bare))
    return [(m - bare) * (i + 1) // used - (m - bare) * i // used for i in range(used)] + [bare]


def _pairs(case: dict) -> int:
    """Query and key pairs that the masks leave, per query head."""
    total = 0
    for n, new in _lengths(case):
        w = case["window"] or n
        lo, hi = n - new + 1, n  # keys that the first and the last new token see without a window
        full = min(max(w - lo + 1, 0), new)  # the new tokens that see all of theirs: lo, lo + 1, ...
        total += full * lo + full * (full - 1) // 2 + (new - full) * min(w, hi)
    return total


def _keys(case: dict) -> int:
    """Cached tokens that some query sees."""
    return sum(min(n, (case["window"] or n) + new - 1) for n, new in _lengths(case))


# ------------------------------------------------------------------------------------------------
# inputs, made on the GPU from the seed alone
# ------------------------------------------------------------------------------------------------
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(g, m: int, k: int, dtype) -> torch.Tensor:
    """N(0, 1) with one channel in a thousand 20 times as large, as a norm's output has them."""
    x = torch.randn(m, k, generator=g, device="cuda")
    idx = torch.randint(0, k, (max(1, k // 1000),), generator=g, device="cuda")
    x[:, idx] *= 20.0
    return x.to(dtype)


def _pack8(codes: torch.Tensor) -> torch.Tensor:
    """(..., L) codes 0..15 -> (..., L/8) int32, code 8 i + j in nibble j of word i."""
    c = codes.view(*codes.shape[:-1], codes.shape[-1] // 8, 8)
    out = torch.zeros(c.shape[:-1], dtype=torch.int32, device=codes.device)
    for j in range(8):
        out |= c[..., j].to(torch.int32) << (4 * j)
    return out


def _unpack8(words: torch.Tensor) -> torch.Tensor:
    """The codes of _pack8, as int32."""
    shifts = torch.arange(0, 32, 4, dtype=torch.int32, device=words.device)
    return ((words.unsqueeze(-1) >> shifts) & 15).reshape(*words.shape[:-1], words.shape[-1] * 8)


def _weight(g, n: int, k: int, fmt: str, group: int) -> dict:
    """Packed codes, group-major scales and zero points of a weight of about N(0, 0.02)."""
    dev = "cuda"
    if fmt == "mxfp4":
        codes = torch.randint(0, 16, (n, k), generator=g, device=dev, dtype=torch.uint8)
        return dict(w=_pack8(codes), zeros=None, codes=codes,
                    scales=torch.randint(119, 122, (k // 32, n), generator=g, device=dev, dtype=torch.uint8))
    codes = torch.randn(n, k, generator=g, device=dev).mul_(2.7).add_(8.0).round_().clamp_(0, 15).to(torch.uint8)
    scales = (0.0075 * (0.6 + 0.8 * torch.rand(k // group, n, generator=g, device=dev))).to(torch.float16)
    zeros = torch.randint(5, 12, (k // group, n), generator=g, device=dev, dtype=torch.uint8) if fmt == "awq" else None
    return dict(w=_pack8(codes), zeros=zeros, codes=codes, scales=scales)


def _lora_inputs(case: dict, seed: int) -> dict:
    g, dt = _gen(seed), _DT[case["dtype"]]
    m, k, n, r, total = case["m"], case["k"], sum(_slices(case)), case["rank"], case["adapters"]
    s = dict(x=_activations(g, m, k, dt))
    if case["kind"] == "lora":
        s["weight"] = _weight(g, n, k, case["fmt"], case["group"])
    else:
        s["y"] = torch.randn(m, n, generator=g, device="cuda").to(dt)
    # trained adapters: a product of about a tenth of the projection's output
    s["a"] = (torch.randn(total, len(_slices(case)) * r, k, generator=g, device="cuda") / math.sqrt(k)).to(dt)
    s["b"] = (torch.randn(total, n, r, generator=g, device="cuda") * (0.1 / math.sqrt(r))).to(dt)
    s["scaling"] = 0.5 + 1.5 * torch.rand(total, generator=g, device="cuda")
    rows = _adapter_rows(case)
    chosen = torch.randperm(total, generator=g, device="cuda")[:len(rows) - 1].to(torch.int32)
    chosen = torch.cat([chosen, torch.full((1,), -1, dtype=torch.int32, device="cuda")])
    ids = torch.repeat_interleave(chosen, torch.tensor(rows, device="cuda"), output_size=m)
    if case["spread"]:  # decoding users in any order; prompts come as runs
        ids = ids[torch.randperm(m, generator=g, device="cuda")]
    s["ids"] = ids.contiguous()
    return s


def _quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(..., D) keys or values in their type -> codes (..., D) int32, (step, least) (..., 2) in that type."""
    f = x.float()
    lo, hi = f.amin(-1, keepdim=True), f.amax(-1, keepdim=True)
    # by a tensor: a division by a Python number may become a multiplication by its reciprocal
    step = torch.maximum((hi - lo) / torch.full_like(lo, 15.0), torch.maximum(hi, -lo) * 2.0 ** -14)
    step = step.to(x.dtype).float().clamp_min(2.0 ** -24 if x.dtype == torch.float16 else 2.0 ** -126)
    codes = torch.round((f - lo) / step).clamp_(0, 15).to(torch.int32)
    return codes, torch.cat([step, lo], -1).to(x.dtype)


def _table(g, case: dict) -> tuple[torch.Tensor, int]:
    """Page numbers (seqs, most pages of one) in no order, and how many pages there are: some are
    other users'."""
    page = case["page"]
    count = [-(-n // page) for n, _ in _lengths(case)]
    pages = sum(count) + 3
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    width = max(count)
    at = torch.tensor([sum(count[:i]) for i in range(len(count))], device="cuda")
    col = torch.arange(width, device="cuda")
    table = perm[(at[:, None] + col[None, :]).clamp_max(pages - 1)]
    return table.contiguous(), pages


def _cache_inputs(case: dict, seed: int) -> dict:
    g, dt = _gen(seed), _DT[case["dtype"]]
    heads, dim, page = case["heads"], case["dim"], case["page"]
    lens = _lengths(case)
    table, pages = _table(g, case)
    s = dict(table=table, lens=lens)
    s["seq_lens"] = torch.tensor([n for n, _ in lens], dtype=torch.int32, device="cuda")
    cu = [0]
    for _, new in lens:
        cu.append(cu[-1] + new)
    s["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
    s["tokens"] = cu[-1]
    # keys have a few channels with a large mean, values do not
    mean = torch.randn(heads, dim, generator=g, device="cuda") * (torch.rand(heads, dim, generator=g, device="cuda") < 0.05) * 6.0

    def keys(*shape):
        return (torch.randn(*shape, dim, generator=g, device="cuda") + mean.view(*([1] * (len(shape) - 1)), heads, dim)).to(dt)

    def values(*shape):
        return (torch.randn(*shape, dim, generator=g, device="cuda") * 0.5).to(dt)

    k = torch.empty(pages, heads, page, dim // 2, dtype=torch.uint8, device="cuda")
    v = torch.empty(pages, heads, page // 8, dim, dtype=torch.int32, device="cuda")
    ks = torch.empty(pages, heads, page, 2, dtype=dt, device="cuda")
    vs = torch.empty_like(ks)
    part = max(1, (1 << 25) // (heads * page * dim))
    for p in range(0, pages, part):
        q = min(pages, p + part)
        c, ks[p:q] = _quantize(keys(q - p, page, heads).transpose(1, 2))
        k[p:q] = _pack8(c).view(torch.uint8)
        c, vs[p:q] = _quantize(values(q - p, page, heads).transpose(1, 2))
        v[p:q] = _pack8(c.view(q - p, heads, page // 8, 8, dim).transpose(-1, -2).contiguous()).squeeze(-1)
    s["cache"] = dict(k=k, v=v, k_scale=ks, v_scale=vs)
    if case["kind"] == "append":
        s["k_new"], s["v_new"] = keys(cu[-1], heads), values(cu[-1], heads)
        pos = [p for n, new in lens for p in range(n - new, n)]
        seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"),
                                      torch.tensor([new for _, new in lens], device="cuda"), output_size=cu[-1])
        p = torch.tensor(pos, device="cuda")
        s["slot"] = table[seq, p // page].long() * page + p % page
        # rows of the new tokens by their place among the 8 tokens that share a word
        s["by_nibble"] = [torch.tensor([i for i, q in enumerate(pos) if q % 8 == j], dtype=torch.int64, device="cuda")
                          for j in range(8)]
    else:
        s["q"] = (torch.randn(cu[-1], heads * case["group"], dim, generator=g, device="cuda") * 1.5).to(dt)
    return s


def prepare(case: dict, seed: int) -> dict:
    s = _lora_inputs(case, seed) if case["kind"] in ("lora", "add") else _cache_inputs(case, seed)
    s["case"] = case
    if "weight" in s and s["weight"]["zeros"] is not None:
        s["weight"]["packed_zeros"] = _pack8(s["weight"]["zeros"])
    if own:
        if case["kind"] in ("lora", "add"):
            s["lora"] = importlib.import_module(_PKG + ".quant.lora")
            s["set"] = s["lora"].LoraAdapters(s["a"], s["b"], s["scaling"], _slices(case))
            if case["kind"] == "lora":
                kernels = importlib.import_module(_PKG + ".quant.kernels")
                s["weight"]["tiles"] = kernels.repack_w4(s["weight"]["w"], case["fmt"] == "mxfp4")
        else:
            s["kv4"] = importlib.import_module(_PKG + ".quant.kv4")
            s["cache"] = s["kv4"].KV4Cache.from_tensors(**s["cache"])
    return s


# ------------------------------------------------------------------------------------------------
# one pass: the framework's calls, or the plain forms
# ------------------------------------------------------------------------------------------------
def run(state: dict):
    case = state["case"]
    kind = case["kind"]
    if not own:
        return {"lora": _plain_lora, "add": _plain_add, "append": _plain_append, "attend": _plain_attend}[kind](state)
    if kind == "lora":
        w = state["weight"]
        return state["lora"].w4a8_linear_lora(state["x"], w["tiles"], w["scales"], w.get("packed_zeros"), case["group"],
                                              state["set"], state["ids"], weight_is_e2m1=case["fmt"] == "mxfp4")
    if kind == "add":
        return state["lora"].lora_add(state["y"], state["x"], state["set"], state["ids"], out=torch.empty_like(state["y"]))
    kv4 = state["kv4"]
    if kind == "append":
        kv4.kv4_append(state["cache"], state["k_new"], state["v_new"], state["table"], state["cu"], state["seq_lens"])
        return kv4.kv4_read(state["cache"], state["table"], state["cu"], state["seq_lens"], state["tokens"])
    return kv4.kv4_attention(state["q"], state["cache"], state["table"], state["cu"], state["seq_lens"],
                             max_q=state["lens"][0][1], max_kv=state["lens"][0][0], window=case["window"])


def _delta(s: dict) -> torch.Tensor:
    """The adapters' part in f32, (m, n)."""
    case = s["case"]
    x, ids, r = s["x"].float(), s["ids"], case["rank"]
    out = torch.zeros(case["m"], sum(_slices(case)), device="cuda")
    for a in range(case["adapters"]):
        has = (ids == a).unsqueeze(1)
        low = torch.where(has, x, 0.0) @ s["a"][a].float().t()  # (m, slices * rank)
        col = 0
        for i, w in enumerate(_slices(case)):
            out[:, col:col + w] += (low[:, i * r:(i + 1) * r] @ s["b"][a, col:col + w].float().t()) * s["scaling"][a]
            col += w
    return out


def _plain_add(s: dict) -> torch.Tensor:
    return (s["y"].float() + _delta(s)).to(s["y"].dtype)


def _plain_lora(s: dict) -> torch.Tensor:
    case, w = s["case"], s["weight"]
    codes, grp = _unpack8(w["w"]), case["group"]
    if case["fmt"] == "mxfp4":
        v = torch.tensor(_E2M1, device="cuda")[codes]
        sc, z = torch.exp2(w["scales"].float() - 127.0), 0.0
    else:
        v, sc = codes.float(), w["scales"].float()
        z = 8.0 if w["zeros"] is None else w["zeros"].t().float().unsqueeze(-1)
    v = ((v.view(v.shape[0], -1, grp) - z) * sc.t().unsqueeze(-1)).view(codes.shape)
    f = s["x"].float()
    amax = f.abs().amax(dim=1, keepdim=True)
    step = (amax / torch.full_like(amax, 448.0)).clamp_min(1e-8)
    q = (f * torch.reciprocal(step)).to(torch.float8_e4m3fn).float() * step
    return (q @ v.t() + _delta(s)).to(s["x"].dtype)


def _values(words: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """Codes (..., D) and (step, least) (..., 2) -> what they stand for, in f32."""
    f = scale.float()
    return words.float() * f[..., :1] + f[..., 1:]


def _plain_append(s: dict):
    cache, page = s["cache"], s["case"]["page"]
    slot = s["slot"]
    p, t = slot // page, slot % page
    kc, ks = _quantize(s["k_new"])
    vc, vs = _quantize(s["v_new"])
    cache["k"][p, :, t] = _pack8(kc).view(torch.uint8)
    cache["k_scale"][p, :, t] = ks
    cache["v_scale"][p, :, t] = vs
    for j, rows in enumerate(s["by_nibble"]):
        at = (p[rows], slice(None), t[rows] // 8)
        cache["v"][at] = (cache["v"][at] & ~(15 << (4 * j))) | (vc[rows] << (4 * j))
    k = _values(_unpack8(cache["k"][p, :, t].view(torch.int32)), cache["k_scale"][p, :, t])
    v = _values((cache["v"][p, :, t // 8] >> (4 * (t % 8))[:, None, None]) & 15, cache["v_scale"][p, :, t])
    return k.to(s["k_new"].dtype), v.to(s["v_new"].dtype)


def _plain_attend(s: dict) -> torch.Tensor:
    case, cache = s["case"], s["cache"]
    heads, grp, dim = case["heads"], case["group"], case["dim"]
    out = torch.empty_like(s["q"])
    row = 0
    for b, (n, new) in enumerate(s["lens"]):
        first = max(0, n - new + 1 - case["window"]) if case["window"] else 0
        p0 = first // case["page"]
        table = s["table"][b, p0:-(-n // case["page"])].long()
        at0 = p0 * case["page"]
        pos = torch.arange(n - new, n, device="cuda").unsqueeze(1)
        key = torch.arange(at0, n, device="cuda")
        hidden = key > pos
        if case["window"]:
            hidden |= key <= pos - case["window"]
        hidden = hidden.unsqueeze(1)
        together = heads if heads * grp * new * n <= 1 << 28 else 1
        for h in range(0, heads, together):
            hs = slice(h, h + together)
            k = _values(_unpack8(cache["k"][table, hs].view(torch.int32)), cache["k_scale"][table, hs])
            k = k.transpose(0, 1).reshape(together, -1, dim)[:, :n - at0]
            v = _unpack8(cache["v"][table, hs].unsqueeze(-1)).transpose(-1, -2).reshape(len(table), together, -1, dim)
            v = _values(v, cache["v_scale"][table, hs]).transpose(0, 1).reshape(together, -1, dim)[:, :n - at0]
            q = s["q"][row:row + new].view(new, heads, grp, dim)[:, hs].float()
            q = q.permute(1, 0, 2, 3).reshape(together, new * grp, dim)
            x = torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(dim)
            x = x.view(together, new, grp, -1).masked_fill_(hidden, -math.inf).view(together, new * grp, -1)
            x = torch.exp(x - x.amax(-1, keepdim=True))
            o = torch.matmul(x, v) / x.sum(-1, keepdim=True)
            o = o.view(together, new, grp, dim).permute(1, 0, 2, 3)
            out[row:row + new].view(new, heads, grp, dim)[:, hs] = o.to(out.dtype)
        row += new
    return out


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without, and what it gives in 64 bits
# ------------------------------------------------------------------------------------------------
def work(case: dict) -> dict:
    if case["kind"] in ("lora", "add"):
        m, k, n, r = case["m"], case["k"], sum(_slices(case)), case["rank"]
        rows = _adapter_rows(case)
        low = len(_slices(case)) * r
        size = 2 * m * (k + n) + 4 * m + (len(rows) - 1) * 2 * (low * k + n * r)
        flops = 2.0 * sum(rows[:-1]) * (low * k + n * r)
        if case["kind"] == "add":
            return dict(bytes=size + 2 * m * n, flops=flops)
        per_group = {"int4": 2.0, "awq": 2.5, "mxfp4": 1.0}[case["fmt"]]
        return dict(bytes=size + n * k / 2 + (k // case["group"]) * n * per_group, flops=flops + 2.0 * m * n * k)
    tokens = sum(new for _, new in _lengths(case))
    vector = case["dim"] // 2 + 4  # codes, step and least value
    if case["kind"] == "append":  # in, into the cache, out of it, and as values
        return dict(bytes=2 * tokens * case["heads"] * (4 * case["dim"] + 2 * vector),
                    flops=16.0 * tokens * case["heads"] * case["dim"])
    return dict(bytes=4 * tokens * case["heads"] * case["group"] * case["dim"]
                + 2 * _keys(case) * case["heads"] * vector + 4 * case["seqs"] * (-(-case["most"] // case["page"])),
                flops=4.0 * _pairs(case) * case["heads"] * case["group"] * case["dim"])


def exact(case: dict, seed: int):
    if case["kind"] in ("lora", "add"):
        return _exact_lora(case, _lora_inputs(case, seed))
    s = _cache_inputs(case, seed)
    return _exact_append(s) if case["kind"] == "append" else _exact_attend(case, s)


def _exact_lora(case: dict, s: dict) -> torch.Tensor:
    x, r = s["x"].double(), case["rank"]
    if case["kind"] == "add":
        y = s["y"].double()
    else:
        w = s["weight"]
        sc = w["scales"]
        if case["fmt"] == "mxfp4":
            val = torch.tensor(_E2M1, dtype=torch.float64, device="cuda").index_select(0, w["codes"].flatten().long())
            val = val.view(w["codes"].shape)
            sc = torch.pow(2.0, sc.double() - 127.0)
        else:
            zero = torch.full(sc.shape, 8.0, dtype=torch.float64, device="cuda") if w["zeros"] is None else w["zeros"].double()
            val = w["codes"].double() - zero.repeat_interleave(case["group"], 0).t()
            sc = sc.double()
        # per row fp8 of x: step max(max |x| / 448, 1e-8) in f32 and codes to nearest even, as the operator
        # defines them
        peak = s["x"].abs().max(dim=1).values.float()
        step = torch.clamp(torch.div(peak, torch.tensor(448.0, device="cuda")), min=1e-8)
        xq = (s["x"].float() * (1.0 / step)[:, None]).to(torch.float8_e4m3fn).double() * step.double()[:, None]
        y = xq @ (val * sc.repeat_interleave(case["group"], 0).t()).t()
    for a in s["ids"].unique().tolist():
        if a < 0:
            continue
        rows = (s["ids"] == a).nonzero().squeeze(1)
        low = (x[rows] @ s["a"][a].double().t()) * float(s["scaling"][a])
        for i, w in enumerate(_slices(case)):
            c = slice(sum(_slices(case)[:i]), sum(_slices(case)[:i + 1]))
            y[rows, c] += low[:, i * r:(i + 1) * r] @ s["b"][a, c].double().t()
    return y


def _exact_append(s: dict):
    out = []
    for x in (s["k_new"], s["v_new"]):
        least = 2.0 ** -24 if x.dtype == torch.float16 else 2.0 ** -126
        f = x.double()
        lo, hi = f.min(dim=-1).values, f.max(dim=-1).values
        step = torch.maximum((hi - lo) / 15.0, f.abs().max(dim=-1).values / 16384.0).to(x.dtype).double()
        step = torch.clamp(step, min=least).unsqueeze(-1)
        code = torch.clamp(torch.round((f - lo.unsqueeze(-1)) / step), 0.0, 15.0)
        out.append(lo.unsqueeze(-1) + step * code)
    return tuple(out)


def _exact_attend(case: dict, s: dict) -> torch.Tensor:
    cache, page, dim, grp = s["cache"], case["page"], case["dim"], case["group"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    nib = torch.arange(8, device="cuda", dtype=torch.int32) * 4
    row = 0
    for b, (n, new) in enumerate(s["lens"]):
        ids = s["table"][b].long()[:-(-n // page)]
        for h in range(case["heads"]):
            low, high = cache["k"][ids, h] & 15, cache["k"][ids, h] >> 4
            kc = torch.stack([low, high], -1).reshape(-1, dim)[:n].double()
            vc = ((cache["v"][ids, h].unsqueeze(2) >> nib.view(1, 1, 8, 1)) & 15).reshape(-1, dim)[:n].double()
            ks = cache["k_scale"][ids, h].reshape(-1, 2)[:n].double()
            vs = cache["v_scale"][ids, h].reshape(-1, 2)[:n].double()
            k, v = kc * ks[:, :1] + ks[:, 1:], vc * vs[:, :1] + vs[:, 1:]
            for q0 in range(0, new, 1024):
                q1 = min(new, q0 + 1024)
                first, end = 0, n - new + q1
                if case["window"]:
                    first = max(0, n - new + q0 + 1 - case["window"])
                at = torch.arange(first, end, device="cuda")
                pos = torch.arange(n - new + q0, end, device="cuda")[:, None, None]
                seen = at <= pos
                if case["window"]:
                    seen &= at > pos - case["window"]
                q = s["q"][row + q0:row + q1, h * grp:(h + 1) * grp].double()
                x = (q.reshape(-1, dim) @ k[first:end].t()).view(q1 - q0, grp, -1) * dim ** -0.5
                p = torch.softmax(torch.where(seen, x, -torch.inf), dim=-1)
                out[row + q0:row + q1, h * grp:(h + 1) * grp] = (p.reshape(-1, end - first) @ v[first:end]).view(q1 - q0, grp, dim)
        row += new
    return out
