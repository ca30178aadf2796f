"""What w4a8_kv4_keep refuses of its output's place, on the CPU: pointers that are never read."""
import ctypes

import pytest
import torch

from conftest import pkg


def test_new_lengths_beside_what_is_read():
    """Every workgroup reads the lists while one writes a sequence's new length."""
    if torch.cuda.is_available():
        pytest.skip("the pointers are not real")
    lib = pkg("_abi").load()
    F = 1 << 20
    arrays = (ctypes.c_void_p * 8)(*[P * F for P in (20, 21, 22, 23)], *[0] * 4)
    table, cu, lens, keep, kept, away = (P * F for P in (1, 2, 3, 4, 5, 6))
    B, ldt, width, ldk, most = 7, 9, 6, 11, 5

    def call(now, **kw):
        a = dict(width=width, most=most)
        a.update(kw)
        # the second cache's arrays are null: what passes the checks of the lists ends there, before a launch
        rc = lib.w4a8_kv4_keep(ctypes.addressof(arrays), 2, 4, 16, 1, 64, table, ldt, a["width"], cu, lens, B, keep, ldk, a["most"], kept, now,
                               None)
        return rc, lib.w4a8_last_error().decode()

    for start, entries, name in ((lens, B, "seq_lens"), (cu, B + 1, "cu"), (kept, B, "kept"), (keep, (B - 1) * ldk + most, "keep"),
                                 (table, (B - 1) * ldt + width, "page table")):
        for now in (start, start - 4 * (B - 1), start + 4 * (entries - 1)):
            rc, msg = call(now)
            assert rc == 1 and "overlaps" in msg and name in msg, (name, now - start, rc, msg)
        for now in (start - 4 * B, start + 4 * entries):
            rc, msg = call(now)
            assert rc == 1 and "16-byte" in msg, (name, now - start, rc, msg)
    for kw, now in ((dict(most=0), keep), (dict(width=0), table), ({}, None), ({}, away)):
        rc, msg = call(now, **kw)
        assert rc == 1 and "16-byte" in msg, (kw, rc, msg)
