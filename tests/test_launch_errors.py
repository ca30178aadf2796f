"""What an entry point says when HIP reports an error with its launch: the error's own text, once. An error that the host
raises itself, a device that does not exist, stands for a failed launch, since HIP keeps one last error per thread."""
import ctypes

import pytest
import torch

from conftest import pkg


@pytest.mark.gpu
def test_a_failed_launch_keeps_its_text(dev):
    lib = pkg("_abi").load()
    hip = ctypes.CDLL("libamdhip64.so")
    M, D, page = 4, 64, 16
    x = torch.randn(M, 1, D, device=dev).bfloat16()
    codes, vcodes = torch.zeros(1, 1, page, D // 2, dtype=torch.uint8, device=dev), torch.zeros(1, 1, 2, D, dtype=torch.int32, device=dev)
    ks, vs = (torch.zeros(1, 1, page, 2, dtype=torch.bfloat16, device=dev) for _ in range(2))
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    table, cu, seq, ids = i32(0), i32(0, M), i32(M), i32(0, -1, 1, 0)
    out, fp8, scales = torch.zeros_like(x), torch.empty(M, D, dtype=torch.uint8, device=dev), torch.empty(M, device=dev)
    a, b, s = torch.randn(2, 8, D, device=dev).bfloat16(), torch.randn(2, 16, 8, device=dev).bfloat16(), torch.ones(2, device=dev)
    y, ws = torch.zeros(M, 16, device=dev).bfloat16(), torch.empty(1 << 16, dtype=torch.uint8, device=dev)
    cols = (ctypes.c_int64 * 1)(16)
    cache = tuple(t.data_ptr() for t in (codes, vcodes, ks, vs))
    p = {k: v.data_ptr() for k, v in dict(x=x, table=table, cu=cu, seq=seq, ids=ids, out=out, fp8=fp8, scales=scales, a=a, b=b, s=s,
                                          y=y, ws=ws).items()}
    st = torch.cuda.current_stream().cuda_stream
    calls = {
        "w4a8_kv4_append": lambda: lib.w4a8_kv4_append(p["x"], D, D, p["x"], D, D, 0, M, 1, D, *cache, 1, page, p["table"], 1, 1, p["cu"],
                                                       p["seq"], 1, st),
        "w4a8_kv4_read": lambda: lib.w4a8_kv4_read(*cache, 0, 1, page, 1, D, p["table"], 1, 1, p["cu"], p["seq"], 1, M, p["x"], p["out"],
                                                   st),
        "w4a8_kv4_attention": lambda: lib.w4a8_kv4_attention(p["x"], 0, D, D, M, 1, 1, D, *cache, 1, page, p["table"], 1, 1, p["cu"],
                                                             p["seq"], 1, 1.0, 1, 0, M, page, p["out"], D, D, None, None, 0, st),
        "w4a8_lora_add": lambda: lib.w4a8_lora_add(p["x"], 0, M, D, D, p["a"], p["b"], p["s"], 2, 8, ctypes.addressof(cols), 1, p["ids"],
                                                   p["y"], 0, 16, p["y"], 16, p["ws"], 1 << 16, st),
        "act_quant": lambda: lib.w4a8_act_quant(p["x"], 0, M, D, D, p["fp8"], D, p["scales"], None, st),
    }
    torch.cuda.synchronize()
    for who, call in calls.items():
        assert call() == 0, who
        assert hip.hipSetDevice(1 << 20) != 0
        assert call() == 3, who
        text = lib.w4a8_last_error().decode()
        assert who in text and "invalid device" in text, text
        assert call() == 0, f"{who}: reported twice"
    torch.cuda.synchronize()
