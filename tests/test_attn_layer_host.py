"""What the C host side of the attention half refuses (r-mda_b200/host/moe_attn.c), without a GPU: nothing is enqueued then, so a
context that cannot work does no harm, and the pointers are never followed."""
import ctypes as C

import pytest


class Attn(C.Structure):
    _fields_ = ([("c", C.c_void_p)] + [(n, C.c_uint32) for n in ("d", "heads", "kv_heads", "hd", "rot")] + [("theta", C.c_float)]
                + [(n, C.c_uint32) for n in ("cols", "rows", "keys")] + [(n, C.c_void_p) for n in ("p", "p16", "o16", "k16", "v16")])


class Rows(C.Structure):
    _fields_ = [("rows", C.c_uint32), ("seqs", C.c_uint32), ("a16", C.c_void_p), ("amax", C.c_void_p), ("sa", C.c_uint32), ("pos", C.c_void_p),
                ("slot", C.c_void_p), ("table", C.c_void_p), ("table_stride", C.c_uint32), ("out", C.c_void_p)]


@pytest.fixture()
def layer(pkg, mc):
    pkg.build.build_host()
    L = C.CDLL(pkg.build.HOST_LIB)
    for f in (L.moe_attn_prompt, L.moe_attn_step):
        f.restype = C.c_bool
    c = mc.Ctx(0)
    yield L, Attn(c=c.p, d=256, heads=2, kv_heads=1, hd=64, rot=64, theta=1e4, cols=256, rows=8, keys=16)
    c.close()


@pytest.mark.parametrize("rows,keys", [(9, None), (0xFFFFFFFF, None), (8, 17), (9, 17)])
def test_prompts_that_do_not_fit(layer, rows, keys, capfd):
    L, q = layer
    r = Rows(rows=rows, seqs=1)
    assert L.moe_attn_prompt(C.byref(q), None, None, C.byref(r), None, None if keys is None else C.c_void_p(16), keys or 0) is False
    assert "room for" in capfd.readouterr().err


@pytest.mark.parametrize("rows,seqs", [(3, 2), (2, 3), (9, 9)])
def test_steps_that_do_not_fit(layer, rows, seqs, capfd):
    L, q = layer
    assert L.moe_attn_step(C.byref(q), None, None, C.byref(Rows(rows=rows, seqs=seqs)), None, 16) is False
    assert "moe_attn:" in capfd.readouterr().err
