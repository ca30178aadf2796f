"""The host extension's calls for prompts, trees, rotary positions and what moves in the cache: they leave what they do not
take to the Python path, and both give the same tensors, bit for bit."""
import pytest
import torch

from conftest import pkg
from test_host_operators import _same

NEW = {"kv4_tree": 5, "kv4_tree_attention": 16, "kv4_copy_pages": 3, "kv4_keep": 6, "prompt_attention": 10, "rotary": 11}


def test_cpu_tensors_and_wrong_counts_are_left_alone():
    m = pkg("_host").load()
    t = torch.zeros(4, 4)
    for name, n in NEW.items():
        assert getattr(m, name)(*[t] * n) is None
        assert getattr(m, name)(*[None] * n) is None
        with pytest.raises(TypeError):
            getattr(m, name)(t)
        assert getattr(pkg("_host")._Absent, name)(*range(n)) is None


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
        mp.setattr(host, "_mod", host._Absent)
        b = fn()
    torch.cuda.synchronize()
    return a, b


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_calls(monkeypatch, dev, dtype):
    kv4, att, rotary = pkg("quant.kv4"), pkg("layers.attention"), pkg("layers.rotary")
    H, G, D, page = 2, 4, 128, 16
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    table, cu, seq = i32([3, 1, 0], [2, 4, 5]), i32(0, 3, 8), i32(40, 33)
    qkv = torch.randn(8, (G * H + 2 * H) * D, device=dev).to(dtype)
    q, k, v = (t.view(8, -1, D) for t in qkv.split([G * H * D, H * D, H * D], dim=1))
    for kw in ({}, dict(return_lse=True, window=3), dict(max_q=5, sm_scale=0.5), dict(causal=False)):
        _same(*_both(monkeypatch, "prompt_attention", lambda: att.prompt_attention(q, k, v, cu, **kw)))
    buf = torch.zeros(8, 3 * G * H, D, dtype=dtype, device=dev)
    got = _both(monkeypatch, "prompt_attention", lambda: att.prompt_attention(q, k, v, cu, out=buf[:, :G * H]))
    assert got[0].data_ptr() == buf.data_ptr() and (buf[:, G * H:] == 0).all()
    for r, pos in ((rotary.Rotary(D, device=dev), torch.arange(8, device=dev)), (rotary.Rotary(D, device=dev), i32(*range(8)).view(1, 8)),
                   (rotary.Rotary(D, sections=(16, 24, 24), adjacent=True, scale=0.5, device=dev), i32(*range(24)).view(3, 8))):
        _same(*_both(monkeypatch, "rotary", lambda: r.forward(q, k, pos)))

        def inplace():
            x = qkv.clone()
            a, b, _ = (t.view(8, -1, D) for t in x.split([G * H * D, H * D, H * D], dim=1))
            r.forward_inplace(a, b, pos)
            return x

        _same(*_both(monkeypatch, "rotary", inplace))
    c = kv4.KV4Cache(8, page, H, D, dtype, dev)
    kv4.kv4_append(c, k, v, table, cu, seq)
    parents = i32(-1, 0, 0, -1, 0, 1, 1, 2)
    _same(*_both(monkeypatch, "kv4_tree", lambda: tuple(kv4.kv4_tree(parents, cu, seq, max_q=5, window=2))))
    tree = kv4.kv4_tree(parents, cu, seq, max_q=5)
    for kw in ({}, dict(return_lse=True, window=7), dict(max_q=5, max_kv=40, sm_scale=0.5)):
        _same(*_both(monkeypatch, "kv4_tree_attention", lambda: kv4.kv4_attention(q, c, table, cu, seq, tree=tree, **kw)))

    def moved(many, call):
        cs = [kv4.KV4Cache.from_tensors(*(t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale))) for _ in range(many)]
        r = call(cs if many > 1 else cs[0])
        return tuple(t for x in cs for t in (x.k, x.v, x.k_scale, x.v_scale)) + (() if r is None else (r,))

    for many in (1, 3):
        _same(*_both(monkeypatch, "kv4_copy_pages", lambda: moved(many, lambda cs: kv4.kv4_copy_pages(cs, i32(3, 4), i32(6, 7)))))
        _same(*_both(monkeypatch, "kv4_keep", lambda: moved(many, lambda cs: kv4.kv4_keep(cs, table, cu, seq, i32([1, 2], [0, 4]), i32(1, 2)))))
    with pytest.raises(ValueError, match="window"):
        kv4.kv4_attention(q, c, table, cu, seq, window=-1, tree=tree)
    with pytest.raises(ValueError, match="window"):
        att.prompt_attention(q, k, v, cu, window=-1)
