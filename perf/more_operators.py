"""What the attention half of a layer needs around a 4-bit cache, as cases that can be timed and checked:
rotary positions, attention over whole prompts, trees of drafted tokens, and what moves in the cache when
drafted tokens are accepted or a sequence is forked.

kind "rotate": queries and keys turned by their positions, through rotary.Rotary.forward. Pair i of a head's first
               R channels (i and i + R/2, or 2 i and 2 i + 1) turns by position[axis of i] * base^(-2 i / R).
kind "prompt": attention over whole prompts, packed, causal, query heads sharing key/value heads, through
               attention.prompt_attention.
kind "tree":   one verification step of drafted tokens: from their parents the ancestors' bits and positions, and
               attention over the 4-bit cache, where a drafted token sees the context and its ancestors, through
               kv4.kv4_tree and kv4.kv4_attention.
kind "copy":   pages of several layers' caches copied to other pages, and read there, through kv4.kv4_copy_pages
               and kv4.kv4_read.
kind "keep":   drafted tokens written into the cache, the accepted ones moved behind the context and read there,
               through kv4.kv4_append, kv4.kv4_keep and kv4.kv4_read.

A cached vector of one token and head is codes c in 0..15 with a step s and a least value m in the model's type and
stands for s c + m:
    m = min x,  s = max((max x - min x) / 15, 2^-14 max |x|), rounded to the type and at least its smallest positive
    value (2^-24 for fp16, 2^-126 for bf16),  c = clamp(rint((x - m) / s), 0, 15).

Sizes are those of the benchmark and the other timed cases (heads of 64, 128 and 256, 8 or 4 key/value heads), from
one token to prompts of 8192 tokens and contexts of 65536.
"""
from __future__ import annotations

import importlib
import math
import random

import torch

own = False

_PKG = "minisglang-rdna4_amd"
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
_BASE = 1000000.0
_MOST_ROWS = 8192 * 40 * 128
_MOST_PAIRS = 3 * 8192 * 4096 * 32 * 128
_MOST_CACHE = 2 * 65536 * 8 * 128
_MOST_MOVED = 2048 * 64 * 8 * 128


# ------------------------------------------------------------------------------------------------
# the cases
# ------------------------------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # one user's decode step: latency
        dict(name="rotate_1_user", kind="rotate", dtype="bf16", tokens=1, heads=8, group=4, dim=128, rotary=128, axes=1,
             interleaved=False, adjacent=False),
        # prompts with images, their positions in time, height and width
        dict(name="rotate_images", kind="rotate", dtype="bf16", tokens=8191, heads=8, group=4, dim=128, rotary=128, axes=3,
             interleaved=False, adjacent=False),
        # a short question: latency
        dict(name="prompt_short", kind="prompt", dtype="bf16", heads=8, group=4, dim=128, seqs=1, most=61, least=1.0,
             window=0),
        # prompts of many lengths back to back, heads of 64 in fp16
        dict(name="prompt_packed", kind="prompt", dtype="fp16", heads=8, group=3, dim=64, seqs=23, most=1999, least=0.02,
             window=0),
        # a few long prompts
        dict(name="prompt_long", kind="prompt", dtype="bf16", heads=8, group=4, dim=128, seqs=3, most=8192, least=0.2,
             window=0),
        # one user's drafted tokens over a short context: latency
        dict(name="tree_1_user", kind="tree", dtype="bf16", heads=8, group=4, dim=128, page=16, seqs=1, new=13, most=1999,
             least=1.0),
        # a verification step of 48 users whose contexts have all lengths up to 8192
        dict(name="tree_48_users", kind="tree", dtype="bf16", heads=8, group=4, dim=128, page=32, seqs=48, new=26, most=8192,
             least=0.02),
        # two users with long documents and wide trees, fp16
        dict(name="tree_long", kind="tree", dtype="fp16", heads=8, group=4, dim=128, page=64, seqs=2, new=60, most=65536,
             least=0.9),
        # 64 users' sequences forked: the partial page of each, in four layers
        dict(name="copy_forks", kind="copy", dtype="bf16", heads=8, dim=128, page=16, layers=4, pages=64),
        # a cache made compact: many pages of one layer
        dict(name="copy_compact", kind="copy", dtype="bf16", heads=8, dim=128, page=64, layers=1, pages=2048),
        # one user's accepted tokens
        dict(name="keep_1_user", kind="keep", dtype="bf16", heads=8, group=1, dim=128, page=16, seqs=1, new=13, most=1999,
             least=1.0, kept=5),
        # those of many users with wide trees, heads of 64 in fp16
        dict(name="keep_96_users", kind="keep", dtype="fp16", heads=8, group=1, dim=64, page=32, seqs=96, new=61, most=4000,
             least=0.05, kept=11),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    """lo..hi, uniform in the logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng) -> dict:
    kind = rng.choice(["rotate", "prompt", "prompt", "tree", "tree", "copy", "keep"])
    case = dict(kind=kind, dtype=rng.choice(["bf16", "fp16"]), heads=rng.choice([1, 2, 4, 8, 8]),
                dim=rng.choice([64, 128, 128, 256]))
    if kind in ("rotate", "prompt", "tree"):
        case["group"] = rng.choice([1, 2, 3, 4, 5, 8, 16])
    if kind == "rotate":
        case["rotary"] = case["dim"] // rng.choice([1, 1, 1, 2])
        case["axes"] = rng.choice([1, 1, 3])
        case["interleaved"] = rng.random() < 0.3
        case["adjacent"] = rng.random() < 0.3
        case["tokens"] = _log_int(rng, 1, 16384)
        while case["tokens"] * case["heads"] * (case["group"] + 1) * case["dim"] > _MOST_ROWS:
            case["tokens"] = case["tokens"] * 3 // 4
        return case
    if kind == "copy":
        case["page"] = rng.choice([16, 16, 32, 64, 128])
        case["layers"] = rng.choice([1, 2, 4])
        case["pages"] = _log_int(rng, 1, 4096)
        while case["pages"] * case["page"] * case["heads"] * case["dim"] * case["layers"] > _MOST_MOVED:
            case["pages"] = case["pages"] * 3 // 4
        return case
    case["least"] = rng.choice([0.01, 0.3, 1.0])
    case["seqs"] = _log_int(rng, 1, 96)
    if kind == "prompt":
        case["most"] = _log_int(rng, 1, 12000)
        case["window"] = rng.choice([0, 0, 0, _log_int(rng, 16, 4096)])
        while case["seqs"] > 1 and case["seqs"] * case["most"] ** 2 // 2 * case["heads"] * case["group"] * case["dim"] \
                > _MOST_PAIRS:
            case["seqs"] = case["seqs"] * 3 // 4
        while case["seqs"] * case["most"] ** 2 // 2 * case["heads"] * case["group"] * case["dim"] > _MOST_PAIRS:
            case["most"] = case["most"] * 3 // 4
        return case
    case["page"] = rng.choice([16, 16, 32, 64, 128])
    case["new"] = _log_int(rng, 2, 150)
    case["most"] = _log_int(rng, case["new"], 40000)
    if kind == "keep":
        case["group"] = 1
        case["kept"] = _log_int(rng, 1, min(case["new"], 24))
    cost = lambda: case["seqs"] * case["most"] * case["heads"] * case["dim"] * max(  # noqa: E731
        2, case["group"] * case["new"] / 128)
    while case["seqs"] > 1 and cost() > _MOST_CACHE:
        case["seqs"] = case["seqs"] * 3 // 4
    while cost() > _MOST_CACHE:
        case["most"] = max(case["new"], case["most"] * 3 // 4)
    return case


# ------------------------------------------------------------------------------------------------
# what a case's sizes imply (the same for every seed)
# ------------------------------------------------------------------------------------------------
def _lengths(case: dict) -> list[tuple[int, int]]:
    """(length with the new tokens, new tokens) of each sequence: lengths spread from least * most to most, the longest
    first; of prompts every token is new."""
    out = []
    for i in range(case["seqs"]):
        f = 1.0 if i == 0 else case["least"] + (1.0 - case["least"]) * ((i * 0.6180339887) % 1.0)
        n = max(1, int(round(case["most"] * f)))
        new = n if case["kind"] == "prompt" else min(n, max(1, case["new"] - i % 5))
        out.append((n, new))
    return out


def _kept(case: dict) -> list[int]:
    """Accepted tokens of each sequence, none of some."""
    return [min(new, max(0, case["kept"] - i % (case["kept"] + 1))) for i, (_, new) in enumerate(_lengths(case))]


def _sections(case: dict) -> list[int]:
    """Pairs of each axis."""
    pairs = case["rotary"] // 2
    if case["axes"] == 1:
        return [pairs]
    t = pairs // 4
    return [pairs - 2 * ((pairs - t) // 2), (pairs - t) // 2, (pairs - t) // 2] if not case["interleaved"] else \
        [pairs - 2 * (pairs // 3), pairs // 3, pairs // 3]


def _pairs(case: dict) -> int:
    """Query and key pairs that the causal mask leaves in a prompt, per query head."""
    total = 0
    for n, _ in _lengths(case):
        w = min(case["window"] or n, n)
        total += w * (w + 1) // 2 + (n - w) * w
    return total


# ------------------------------------------------------------------------------------------------
# inputs, made on the GPU from the seed alone
# ------------------------------------------------------------------------------------------------
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _running(counts: list[int]) -> list[int]:
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


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


def _quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(..., D) keys or values in their type -> codes (..., D) int32, (step, least) (..., 2) in that type."""
    f = x.float()
    lo, hi = f.amin(-1, keepdim=True), f.amax(-1, keepdim=True)
    # by a tensor: a division by a Python number may become a multiplication by its reciprocal
    step = torch.maximum((hi - lo) / torch.full_like(lo, 15.0), torch.maximum(hi, -lo) * 2.0 ** -14)
    step = step.to(x.dtype).float().clamp_min(2.0 ** -24 if x.dtype == torch.float16 else 2.0 ** -126)
    codes = torch.round((f - lo) / step).clamp_(0, 15).to(torch.int32)
    return codes, torch.cat([step, lo], -1).to(x.dtype)


def _vectors(g, case: dict):
    """Makers of keys, a few channels of which have a large mean, and of values: (rows, heads, dim)."""
    heads, dim, dt = case["heads"], case["dim"], _DT[case["dtype"]]
    mean = torch.randn(heads, dim, generator=g, device="cuda") * 6.0
    mean *= torch.rand(heads, dim, generator=g, device="cuda") < 0.05

    def keys(rows):
        return (torch.randn(rows, heads, dim, generator=g, device="cuda") + mean).to(dt)

    def values(rows):
        return (torch.randn(rows, heads, dim, generator=g, device="cuda") * 0.5).to(dt)

    return keys, values


def _cache(g, case: dict, pages: int) -> dict:
    """A layer's cache, every slot of it written."""
    heads, dim, page, dt = case["heads"], case["dim"], case["page"], _DT[case["dtype"]]
    keys, values = _vectors(g, case)
    k = torch.empty(pages, heads, page, dim // 2, dtype=torch.uint8, device="cuda")
    v = torch.empty(pages, heads, page // 8, dim, dtype=torch.int32, device="cuda")
    ks = torch.empty(pages, heads, page, 2, dtype=dt, device="cuda")
    vs = torch.empty_like(ks)
    part = max(1, (1 << 25) // (heads * page * dim))
    for p in range(0, pages, part):
        q = min(pages, p + part)
        c, ks[p:q] = _quantize(keys((q - p) * page).view(q - p, page, heads, dim).transpose(1, 2))
        k[p:q] = _pack8(c).view(torch.uint8)
        c, vs[p:q] = _quantize(values((q - p) * page).view(q - p, page, heads, dim).transpose(1, 2))
        v[p:q] = _pack8(c.view(q - p, heads, page // 8, 8, dim).transpose(-1, -2).contiguous()).squeeze(-1)
    return dict(k=k, v=v, k_scale=ks, v_scale=vs)


def _rotate_inputs(g, case: dict, seed: int) -> dict:
    T, heads, dim = case["tokens"], case["heads"], case["dim"]
    qkv = (torch.randn(T, heads * (case["group"] + 2) * dim, generator=g, device="cuda") * 1.5).to(_DT[case["dtype"]])
    # a few sequences' tokens, each from where its context ends
    at = torch.arange(T, device="cuda")
    run = max(1, T // 3)
    first = torch.randint(0, 100000, (T // run + 1,), generator=g, device="cuda")[at // run]
    if case["axes"] == 1:
        pos = (first + at % run).to(torch.int32)
    else:  # images of 32 x 32 patches, one after another
        pos = torch.stack([first + at // 1024, first + at // 32 % 32, first + at % 32]).to(torch.int32)
    return dict(qkv=qkv, pos=pos)


def _prompt_inputs(g, case: dict, seed: int) -> dict:
    lens = [n for n, _ in _lengths(case)]
    T, heads, dim = sum(lens), case["heads"], case["dim"]
    qkv = torch.randn(T, heads * (case["group"] + 2), dim, generator=g, device="cuda")
    qkv[:, :heads * case["group"]] *= 1.5
    keys, values = _vectors(g, case)
    qkv = qkv.to(_DT[case["dtype"]])
    qkv[:, heads * case["group"]:heads * (case["group"] + 1)] = keys(T)
    qkv[:, heads * (case["group"] + 1):] = values(T)
    return dict(qkv=qkv.view(T, -1), cu=_ints(_running(lens)))


def _batch_inputs(g, case: dict, seed: int) -> dict:
    """Sequences on pages in no order, and their cache."""
    lens = _lengths(case)
    count = [-(-n // case["page"]) for n, _ in lens]
    pages, width = sum(count) + 3, max(count)
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    col = torch.arange(width, device="cuda")
    first = torch.tensor(_running(count)[:-1], device="cuda")
    table = perm[(first[:, None] + col[None, :]).clamp_max(pages - 1)].contiguous()
    new = [w for _, w in lens]
    s = dict(table=table, lens=_ints([n for n, _ in lens]), cu=_ints(_running(new)), cache=_cache(g, case, pages))
    T = sum(new)
    if case["kind"] == "tree":
        s["q"] = (torch.randn(T, case["heads"] * case["group"], case["dim"], generator=g, device="cuda") * 1.5).to(
            _DT[case["dtype"]])
        rng = random.Random(seed)
        # a drafted token follows one of the six before it, some the context itself
        s["parents"] = _ints([-1 if i == 0 or rng.random() < 0.1 else rng.randrange(max(0, i - 6), i)
                              for n in new for i in range(n)])
    else:
        keys, values = _vectors(g, case)
        s["k_new"], s["v_new"] = keys(T), values(T)
        kept = _kept(case)
        s["keep"] = torch.zeros(len(lens), max(kept), dtype=torch.int32, device="cuda")
        for b, (n, m) in enumerate(zip(new, kept)):
            s["keep"][b, :m] = torch.randperm(n, generator=g, device="cuda")[:m].sort().values.to(torch.int32)
        s["kept"], s["cu_kept"] = _ints(kept), _ints(_running(kept))
    return s


def _copy_inputs(g, case: dict, seed: int) -> dict:
    n, page = case["pages"], case["page"]
    total = 2 * n + 5
    perm = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    src = perm[:n][torch.randint(0, n, (n,), generator=g, device="cuda")].contiguous()  # some are forked more than once
    cu = torch.arange(0, (n + 1) * page, page, dtype=torch.int32, device="cuda")
    return dict(src=src, dst=perm[n:2 * n].contiguous(), cu=cu,
                lens=torch.full((n,), page, dtype=torch.int32, device="cuda"),
                caches=[_cache(g, case, total) for _ in range(case["layers"])])


def _inputs(case: dict, seed: int) -> dict:
    make = {"rotate": _rotate_inputs, "prompt": _prompt_inputs, "copy": _copy_inputs}.get(case["kind"], _batch_inputs)
    return dict(make(_gen(seed), case, seed), case=case)


def prepare(case: dict, seed: int) -> dict:
    s = _inputs(case, seed)
    if case["kind"] in ("tree", "keep"):  # what a scheduler knows of its batch on the host
        s["host"] = dict(lens=_lengths(case), max_q=max(w for _, w in _lengths(case)), max_kv=case["most"])
        if case["kind"] == "keep":
            s["host"]["kept"] = _kept(case)
    if own:
        if case["kind"] == "rotate":
            rotary = importlib.import_module(_PKG + ".layers.rotary")
            s["rotary"] = rotary.Rotary(case["dim"], base=_BASE, rotary_dim=case["rotary"],
                                        sections=_sections(case) if case["axes"] > 1 else None,
                                        interleaved=case["interleaved"] and case["axes"] > 1, adjacent=case["adjacent"],
                                        device="cuda")
        elif case["kind"] == "prompt":
            s["attention"] = importlib.import_module(_PKG + ".layers.attention")
        else:
            s["kv4"] = importlib.import_module(_PKG + ".quant.kv4")
            if case["kind"] == "copy":
                s["caches"] = [s["kv4"].KV4Cache.from_tensors(**c) for c in s["caches"]]
            else:
                s["cache"] = s["kv4"].KV4Cache.from_tensors(**s["cache"])
    return s


# ------------------------------------------------------------------------------------------------
# one pass: the framework's calls, or the plain forms
# ------------------------------------------------------------------------------------------------
def _split(s: dict) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """A merged projection's output -> q, k and v, (tokens, heads, dim) views of it."""
    case = s["case"]
    kv = case["heads"] * case["dim"]
    q, k, v = s["qkv"].split([kv * case["group"], kv, kv], dim=1)
    return tuple(t.view(t.shape[0], -1, case["dim"]) for t in (q, k, v))


def run(state: dict):
    case = state["case"]
    if not own:
        return {"rotate": _plain_rotate, "prompt": _plain_prompt, "tree": _plain_tree, "copy": _plain_copy,
                "keep": _plain_keep}[case["kind"]](state)
    if case["kind"] == "rotate":
        q, k, _ = _split(state)
        return state["rotary"].forward(q, k, state["pos"])
    if case["kind"] == "prompt":
        return state["attention"].prompt_attention(*_split(state), state["cu"], max_q=case["most"], window=case["window"])
    kv4 = state["kv4"]
    if case["kind"] == "copy":
        kv4.kv4_copy_pages(state["caches"], state["src"], state["dst"])
        rows = case["pages"] * case["page"]
        return [kv4.kv4_read(c, state["dst"].view(-1, 1), state["cu"], state["lens"], rows) for c in state["caches"]]
    cache, table, cu, lens, host = state["cache"], state["table"], state["cu"], state["lens"], state["host"]
    if case["kind"] == "tree":
        tree = kv4.kv4_tree(state["parents"], cu, lens, max_q=host["max_q"])
        out = kv4.kv4_attention(state["q"], cache, table, cu, lens, max_q=host["max_q"], max_kv=host["max_kv"], tree=tree)
        return tree.mask, tree.positions, out
    kv4.kv4_append(cache, state["k_new"], state["v_new"], table, cu, lens)
    now = kv4.kv4_keep(cache, table, cu, lens, state["keep"], state["kept"])
    k, v = kv4.kv4_read(cache, table, state["cu_kept"], now, sum(host["kept"]))
    return now, k, v


def _axis_of_pair(case: dict) -> list[int]:
    sec = _sections(case)
    if case["axes"] > 1 and case["interleaved"]:
        return [i % 3 if i < 3 * sec[i % 3] else 0 for i in range(case["rotary"] // 2)]
    return [a for a, n in enumerate(sec) for _ in range(n)]


def _plain_rotate(s: dict):
    case = s["case"]
    half = case["rotary"] // 2
    freq = _BASE ** (torch.arange(half, dtype=torch.float64, device="cuda") * (-2.0 / case["rotary"]))
    pos = s["pos"].double().view(case["axes"], -1)[torch.tensor(_axis_of_pair(case), device="cuda")].t()
    angle = (pos * freq).unsqueeze(1)
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    out = []
    for x in _split(s)[:2]:
        f = x.float()
        r = f[..., :case["rotary"]]
        if case["adjacent"]:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        else:
            a, b = r[..., :half], r[..., half:]
            r = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        out.append(torch.cat([r, f[..., case["rotary"]:]], -1).to(x.dtype))
    return tuple(out)


def _softmax_of(x: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """Masked scores (heads, rows, keys) and values (heads, keys, dim); rows that see nothing are 0."""
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = x.sum(-1, keepdim=True)
    return torch.matmul(x, v) / torch.where(total == 0, 1.0, total)


def _plain_prompt(s: dict) -> torch.Tensor:
    case = s["case"]
    q, k, v = _split(s)
    heads, grp, dim = case["heads"], case["group"], case["dim"]
    out = torch.empty(q.shape, dtype=q.dtype, device="cuda")
    row = 0
    for n, _ in _lengths(case):
        at = torch.arange(n, device="cuda")
        hidden = at > at.unsqueeze(1)
        if case["window"]:
            hidden |= at <= at.unsqueeze(1) - case["window"]
        together = heads if heads * grp * n * n <= 1 << 28 else 1
        for h in range(0, heads, together):
            hs = slice(h, h + together)
            qh = q[row:row + n].view(n, heads, grp, dim)[:, hs].permute(1, 2, 0, 3).float().reshape(together, grp * n, dim)
            kh = k[row:row + n, hs].permute(1, 2, 0).float().contiguous()
            vh = v[row:row + n, hs].permute(1, 0, 2).float().contiguous()
            x = (torch.matmul(qh, kh) / math.sqrt(dim)).view(together, grp, n, n).masked_fill_(hidden, -math.inf)
            o = _softmax_of(x.view(together, grp * n, n), vh).view(together, grp, n, dim)
            out[row:row + n].view(n, heads, grp, dim)[:, hs] = o.permute(2, 0, 1, 3).to(out.dtype)
        row += n
    return out


def _values(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """Codes (..., D) and (step, least) (..., 2) -> what they stand for, in f32."""
    f = scale.float()
    return codes.float() * f[..., :1] + f[..., 1:]


def _plain_pages(cache: dict, pages: torch.Tensor, hs: slice) -> tuple[torch.Tensor, torch.Tensor]:
    """Values of whole pages, (pages, heads, tokens, dim) each."""
    k = _values(_unpack8(cache["k"][pages, hs].view(torch.int32)), cache["k_scale"][pages, hs])
    v = _unpack8(cache["v"][pages, hs].unsqueeze(-1)).transpose(-1, -2)
    return k, _values(v.reshape(k.shape), cache["v_scale"][pages, hs])


def _plain_tree(s: dict):
    case, cache, host = s["case"], s["cache"], s["host"]
    heads, grp, dim = case["heads"], case["group"], case["dim"]
    words = -(-host["max_q"] // 32)
    mask = torch.zeros(s["parents"].shape[0], words, dtype=torch.int32, device="cuda")
    pos = torch.empty_like(s["parents"])
    out = torch.empty_like(s["q"])
    row = 0
    for b, (n, new) in enumerate(host["lens"]):
        parent = s["parents"][row:row + new].long()
        see = torch.eye(new, dtype=torch.bool, device="cuda")
        up = parent.clone()
        for _ in range(new - 1):  # an ancestor more a step
            see |= torch.arange(new, device="cuda") == up.unsqueeze(1)
            up = torch.where(up < 0, up, parent[up.clamp_min(0)])
        pos[row:row + new] = n - new + see.sum(1).to(torch.int32) - 1
        bits = torch.zeros(new, words * 32, dtype=torch.int64, device="cuda")
        bits[:, :new] = see.long()
        bits = (bits.view(new, words, 32) << torch.arange(32, device="cuda")).sum(-1)
        mask[row:row + new] = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32)
        hidden = torch.cat([torch.zeros(new, n - new, dtype=torch.bool, device="cuda"), ~see], 1).unsqueeze(1)
        table = s["table"][b, :-(-n // case["page"])].long()
        together = heads if heads * grp * new * n <= 1 << 28 else 1
        for h in range(0, heads, together):
            hs = slice(h, h + together)
            k, v = (t.transpose(0, 1).reshape(together, -1, dim)[:, :n] for t in _plain_pages(cache, table, hs))
            q = s["q"][row:row + new].view(new, heads, grp, dim)[:, hs].float().permute(1, 0, 2, 3)
            x = torch.matmul(q.reshape(together, new * grp, dim), k.transpose(1, 2).contiguous()) / math.sqrt(dim)
            x = x.view(together, new, grp, n).masked_fill_(hidden, -math.inf).view(together, new * grp, n)
            o = _softmax_of(x, v).view(together, new, grp, dim)
            out[row:row + new].view(new, heads, grp, dim)[:, hs] = o.permute(1, 0, 2, 3).to(out.dtype)
        row += new
    return mask, pos, out


def _plain_copy(s: dict):
    src, dst, out = s["src"].long(), s["dst"].long(), []
    for cache in s["caches"]:
        for t in cache.values():
            t[dst] = t[src]
        k, v = _plain_pages(cache, dst, slice(None))
        out.append(tuple(t.transpose(1, 2).flatten(0, 1).to(cache["k_scale"].dtype) for t in (k, v)))
    return out


def _plain_keep(s: dict):
    case, cache, host = s["case"], s["cache"], s["host"]
    page, dt = case["page"], _DT[case["dtype"]]
    base = torch.tensor([n - new for n, new in host["lens"]], device="cuda")
    first = torch.tensor(_running([new for _, new in host["lens"]])[:-1], device="cuda")

    def place(counts):
        """(sequence, number of its tokens before it) of each of so many tokens."""
        total = sum(counts)
        seq = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), torch.tensor(counts, device="cuda"),
                                      output_size=total)
        return seq, torch.arange(total, device="cuda") - torch.tensor(_running(counts)[:-1], device="cuda")[seq]

    def slots(seq, j):
        pos = base[seq] + j
        return s["table"][seq, pos // page].long(), pos % page

    def nibbles(p, t, codes):
        for j in range(8):  # the 8 tokens of a word one after another
            at = torch.where(t % 8 == j)[0]
            w = (p[at], slice(None), t[at] // 8)
            cache["v"][w] = (cache["v"][w] & ~(15 << (4 * j))) | (codes[at] << (4 * j))

    def fetch(p, t):
        return (cache["v"][p, :, t // 8] >> (4 * (t % 8)).to(torch.int32)[:, None, None]) & 15

    p, t = slots(*place([new for _, new in host["lens"]]))
    kc, ks = _quantize(s["k_new"])
    vc, vs = _quantize(s["v_new"])
    cache["k"][p, :, t] = _pack8(kc).view(torch.uint8)
    cache["k_scale"][p, :, t], cache["v_scale"][p, :, t] = ks, vs
    nibbles(p, t, vc)
    seq, j = place(host["kept"])
    sp, st = slots(seq, s["keep"][seq, j].long())
    p, t = slots(seq, j)
    moved = cache["k"][sp, :, st], cache["k_scale"][sp, :, st], cache["v_scale"][sp, :, st], fetch(sp, st)
    cache["k"][p, :, t], cache["k_scale"][p, :, t], cache["v_scale"][p, :, t] = moved[:3]
    nibbles(p, t, moved[3])
    k = _values(_unpack8(cache["k"][p, :, t].view(torch.int32)), cache["k_scale"][p, :, t]).to(dt)
    v = _values(fetch(p, t), cache["v_scale"][p, :, t]).to(dt)
    return (base + s["kept"]).to(torch.int32), k, v


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without, and what it gives in 64 bits
# ------------------------------------------------------------------------------------------------
def work(case: dict) -> dict:
    heads, dim = case["heads"], case["dim"]
    vector = dim // 2 + 4  # codes, step and least value
    if case["kind"] == "rotate":
        rows = case["tokens"] * heads * (case["group"] + 1)
        return dict(bytes=4 * rows * dim + 4 * case["tokens"] * case["axes"], flops=3.0 * rows * case["rotary"])
    if case["kind"] == "copy":  # read, written, read and given as values
        rows = case["layers"] * case["pages"] * case["page"] * heads
        return dict(bytes=rows * 2 * (3 * vector + 2 * dim) + 8 * case["pages"], flops=4.0 * rows * dim)
    tokens = sum(new for _, new in _lengths(case))
    if case["kind"] == "prompt":
        return dict(bytes=4 * tokens * heads * (case["group"] + 1) * dim,
                    flops=4.0 * _pairs(case) * heads * case["group"] * dim)
    if case["kind"] == "keep":  # in, into the cache, the kept ones read, written, read and given as values
        return dict(bytes=2 * heads * (tokens * (2 * dim + vector) + sum(_kept(case)) * (3 * vector + 2 * dim)),
                    flops=heads * dim * (8.0 * tokens + 4.0 * sum(_kept(case))))
    # every drafted token is counted with its whole context and half of its tree
    keys = sum(n for n, _ in _lengths(case))
    pairs = sum(new * (n - new + (new + 1) // 2) for n, new in _lengths(case))
    return dict(bytes=4 * tokens * heads * case["group"] * dim + 2 * keys * heads * vector + 12 * tokens,
                flops=4.0 * pairs * heads * case["group"] * dim)


def exact(case: dict, seed: int):
    s = _inputs(case, seed)
    return {"rotate": _exact_rotate, "prompt": _exact_prompt, "tree": _exact_tree, "copy": _exact_copy,
            "keep": _exact_keep}[case["kind"]](case, s)


def _exact_rotate(case: dict, s: dict):
    R, heads, dim = case["rotary"], case["heads"], case["dim"]
    axis = []
    if case["axes"] == 3 and case["interleaved"]:  # time, height, width, time, ...
        third = (R // 2) // 3
        axis = [(0, 1, 2)[i % 3] if i // 3 < third else 0 for i in range(R // 2)]
    else:
        for a, n in enumerate(_sections(case)):
            axis += [a] * n
    x = s["qkv"].double().view(case["tokens"], -1, dim)[:, :heads * (case["group"] + 1)]
    out = x.clone()
    pos = s["pos"].double().view(case["axes"], -1)
    for i in range(R // 2):
        angle = pos[axis[i]] * _BASE ** (-2.0 * i / R)
        turn = torch.polar(torch.ones_like(angle), angle)
        a, b = (2 * i, 2 * i + 1) if case["adjacent"] else (i, i + R // 2)
        z = torch.complex(x[..., a], x[..., b]) * turn[:, None]
        out[..., a], out[..., b] = z.real, z.imag
    return out[:, :heads * case["group"]].contiguous(), out[:, heads * case["group"]:].contiguous()


def _attend64(q, k, v, seen):
    """q (rows, group, dim), k and v (keys, dim), seen (rows, keys) -> (rows, group, dim)."""
    x = (q.reshape(-1, q.shape[-1]) @ k.t()).view(*q.shape[:2], -1) * q.shape[-1] ** -0.5
    p = torch.softmax(torch.where(seen.unsqueeze(1), x, -torch.inf), dim=-1)
    return (p.reshape(-1, k.shape[0]) @ v).view(q.shape)


def _exact_prompt(case: dict, s: dict):
    heads, dim, grp = case["heads"], case["dim"], case["group"]
    T = s["qkv"].shape[0]
    qkv = s["qkv"].view(T, -1, dim)
    out = torch.empty(T, heads * grp, dim, dtype=torch.float64, device="cuda")
    start = 0
    for n, _ in _lengths(case):
        for h in range(heads):
            k = qkv[start:start + n, heads * grp + h].double()
            v = qkv[start:start + n, heads * (grp + 1) + h].double()
            for a in range(0, n, 1024):
                b = min(n, a + 1024)
                lo = max(0, a + 1 - case["window"]) if case["window"] else 0
                i, j = torch.arange(a, b, device="cuda")[:, None], torch.arange(lo, b, device="cuda")
                seen = (j <= i) & (j > i - case["window"]) if case["window"] else j <= i
                q = qkv[start + a:start + b, h * grp:(h + 1) * grp].double()
                out[start + a:start + b, h * grp:(h + 1) * grp] = _attend64(q, k[lo:b], v[lo:b], seen)
        start += n
    return out


def _cached64(cache: dict, ids: torch.Tensor, h) -> tuple[torch.Tensor, torch.Tensor]:
    """One head's cached keys and values on pages ids, in order, in 64 bits."""
    dim = cache["v"].shape[-1]
    k = torch.stack([cache["k"][ids, h] & 15, cache["k"][ids, h] >> 4], -1).reshape(-1, dim).double()
    nib = torch.arange(8, device="cuda", dtype=torch.int32).view(1, 1, 8, 1) * 4
    v = ((cache["v"][ids, h].unsqueeze(2) >> nib) & 15).reshape(-1, dim).double()
    ks, vs = cache["k_scale"][ids, h].reshape(-1, 2).double(), cache["v_scale"][ids, h].reshape(-1, 2).double()
    return k * ks[:, :1] + ks[:, 1:], v * vs[:, :1] + vs[:, 1:]


def _exact_tree(case: dict, s: dict):
    lens = _lengths(case)
    words = -(-max(new for _, new in lens) // 32)
    parents = s["parents"].tolist()
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    masks, pos, row, grp = [], [], 0, case["group"]
    for b, (n, new) in enumerate(lens):
        above = []  # each node's line of ancestors, itself last
        for i in range(new):
            p = parents[row + i]
            above.append((above[p] if p >= 0 else []) + [i])
            bits = sum(1 << j for j in above[i])
            part = [(bits >> (32 * w)) & 0xffffffff for w in range(words)]
            masks.append([w - (1 << 32) if w >> 31 else w for w in part])
            pos.append(n - new + len(above[i]) - 1)
        seen = torch.zeros(new, n, dtype=torch.bool)
        seen[:, :n - new] = True
        for i, line in enumerate(above):
            seen[i, [n - new + j for j in line]] = True
        seen = seen.cuda()
        for h in range(case["heads"]):
            k, v = _cached64(s["cache"], s["table"][b].long()[:-(-n // case["page"])], h)
            q = s["q"][row:row + new, h * grp:(h + 1) * grp].double()
            out[row:row + new, h * grp:(h + 1) * grp] = _attend64(q, k[:n], v[:n], seen)
        row += new
    return _ints(masks), _ints(pos), out


def _exact_copy(case: dict, s: dict):
    out = []
    for c in s["caches"]:
        kv = [_cached64(c, s["src"].long(), h) for h in range(case["heads"])]
        out.append(tuple(torch.stack([x[i] for x in kv], 1) for i in (0, 1)))
    return out


def _exact_keep(case: dict, s: dict):
    rows, at = [], 0
    for b, ((_, new), m) in enumerate(zip(_lengths(case), _kept(case))):
        rows += [at + j for j in s["keep"][b, :m].tolist()]
        at += new
    now = _ints([n - new + m for (n, new), m in zip(_lengths(case), _kept(case))])
    out = []
    for x in (s["k_new"], s["v_new"]):
        x = x[torch.tensor(rows, dtype=torch.int64, device="cuda")]
        least = 2.0 ** -24 if x.dtype == torch.float16 else 2.0 ** -126
        f = x.double()
        lo, hi = f.min(dim=-1).values, f.max(dim=-1).values
        step = torch.maximum((hi - lo) / 15.0, f.abs().max(dim=-1).values / 16384.0).to(x.dtype).double()
        step = torch.clamp(step, min=least).unsqueeze(-1)
        out.append(lo.unsqueeze(-1) + step * torch.clamp(torch.round((f - lo.unsqueeze(-1)) / step), 0.0, 15.0))
    return (now, *out)
