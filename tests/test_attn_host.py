"""What the attention calls refuse (r-mda_b200/csrc/moe_attn_args.h, plain C), checked without a GPU: a copy of the header's
functions is compiled with gcc and called through ctypes.  Also the layouts of the argument structs."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
AT = 0x10000   # an address that is never followed


@pytest.fixture(scope="module")
def args(tmp_path_factory):
    d = tmp_path_factory.mktemp("args")
    src = d / "args.c"
    src.write_text('#include "%s/r-mda_b200/csrc/moe_attn_args.h"\n' % ROOT + '''
const char *rope(const void *x, const void *pos, const void *out, struct moe_pc_rope_t pc) { return moe_rope_refusal(x, pos, out, pc); }
const char *kv(const moe_cuda_kv_t *kv) { return moe_kv_refusal(kv); }
const char *kv_write(const moe_cuda_kv_t *kv, const void *k, const void *v, const void *s, struct moe_pc_kv_write_t pc) { return moe_kv_write_refusal(kv, k, v, s, pc); }
const char *kv_read(const moe_cuda_kv_t *kv, const void *t, const void *cu, const void *k, const void *v, struct moe_pc_kv_read_t pc) { return moe_kv_read_refusal(kv, t, cu, k, v, pc); }
const char *attn(const void *q, const void *k, const void *v, const void *cq, const void *ck, const void *o, struct moe_pc_attn_t pc) { return moe_attn_refusal(q, k, v, cq, ck, o, pc); }
const char *decode(const moe_cuda_kv_t *kv, const void *q, const void *t, const void *l, const void *o, struct moe_pc_attn_decode_t pc) { return moe_attn_decode_refusal(kv, q, t, l, o, pc); }
unsigned sizes(int i) {
    unsigned s[] = {sizeof(struct moe_pc_rope_t), sizeof(moe_cuda_kv_t), sizeof(struct moe_pc_kv_write_t), sizeof(struct moe_pc_kv_read_t),
                    sizeof(struct moe_pc_attn_t), sizeof(struct moe_pc_attn_decode_t)};
    return s[i];
}
''')
    so = d / "args.so"
    r = subprocess.run(["gcc", "-std=gnu17", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-o", str(so), str(src)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    lib = C.CDLL(str(so))
    for n in ("rope", "kv", "kv_write", "kv_read", "attn", "decode"):
        getattr(lib, n).restype = C.c_char_p
    return lib


def test_struct_layouts(args, mc):
    for i, t in enumerate((mc.PcRope, mc.Kv, mc.PcKvWrite, mc.PcKvRead, mc.PcAttn, mc.PcAttnDecode)):
        assert args.sizes(i) == C.sizeof(t)


def _vp(*a):
    return [C.c_void_p(x) for x in a]


ROPE = dict(rows=5, heads=6, rot_heads=4, hd=64, rot=64, stride=384, out_stride=384, theta=1e4)


@pytest.mark.parametrize("change,at", [
    (dict(heads=0), None), (dict(hd=60), None), (dict(rot_heads=7), None), (dict(rot=12), None), (dict(rot=72), None), (dict(rot=0), None),
    (dict(hd=1024, rot=520, stride=6144, out_stride=6144), None), (dict(theta=0.0), None), (dict(theta=-1.0), None), (dict(theta=float("nan")), None),
    (dict(theta=float("inf")), None), (dict(stride=380), None), (dict(stride=386), None), (dict(out_stride=388), None), (dict(out_stride=376), None),
    ({}, (AT + 4, AT, AT)), ({}, (AT, AT, AT + 8)), ({}, (AT, None, AT)), ({}, (None, AT, AT)), ({}, (AT, AT + 2, AT))])
def test_rope_refusals(args, mc, change, at):
    assert args.rope(*_vp(AT, AT, AT), mc.PcRope(**ROPE)) is None
    assert args.rope(*_vp(*(at or (AT, AT, AT))), mc.PcRope(**{**ROPE, **change})) is not None


def test_rope_accepts(args, mc):
    assert args.rope(*_vp(AT, None, AT), mc.PcRope(**{**ROPE, "rot_heads": 0, "rot": 0, "theta": 0.0})) is None
    assert args.rope(*_vp(None, None, None), mc.PcRope(**{**ROPE, "rows": 0})) is None


KV = dict(k=AT, v=AT, k_scale=None, v_scale=None, pages=10, page=16, kv_heads=2, hd=64, type=0)


@pytest.mark.parametrize("change", [
    dict(type=2), dict(hd=96), dict(hd=256), dict(page=8), dict(page=48), dict(page=512), dict(pages=0), dict(pages=2 ** 28, page=16), dict(kv_heads=0),
    dict(kv_heads=1025), dict(k=None), dict(v=AT + 8), dict(type=1), dict(type=1, k_scale=AT, v_scale=AT + 4), dict(type=1, k_scale=AT)])
def test_cache_refusals(args, mc, change):
    assert args.kv(C.byref(mc.Kv(**KV))) is None and args.kv(C.byref(mc.Kv(**{**KV, "type": 1, "k_scale": AT, "v_scale": AT}))) is None
    assert args.kv(C.byref(mc.Kv(**{**KV, **change}))) is not None
    assert args.kv(None) is not None


def test_cache_takes_all_but_the_last_slots(args, mc):
    assert args.kv(C.byref(mc.Kv(**{**KV, "pages": 2 ** 27 - 1, "page": 16, "kv_heads": 1}))) is None
    assert args.kv(C.byref(mc.Kv(**{**KV, "pages": 2 ** 26, "page": 16, "kv_heads": 2}))) is not None


@pytest.mark.parametrize("rows,stride,at", [(3, 120, (AT, AT, AT)), (3, 132, (AT, AT, AT)), (2 ** 29, 128, (AT, AT, AT)), (3, 128, (None, AT, AT)),
                                             (3, 128, (AT, AT + 2, AT)), (3, 128, (AT, AT, None)), (3, 128, (AT, AT, AT + 1))])
def test_kv_write_refusals(args, mc, rows, stride, at):
    kv = mc.Kv(**KV)
    assert args.kv_write(C.byref(kv), *_vp(AT, AT, AT), mc.PcKvWrite(3, 128)) is None
    assert args.kv_write(C.byref(kv), *_vp(*at), mc.PcKvWrite(rows, stride)) is not None


@pytest.mark.parametrize("pc,at", [((1, 3, 1, 120), (AT,) * 4), ((1, 2 ** 31, 1, 128), (AT,) * 4), ((2 ** 20, 3, 1, 128), (AT,) * 4),
                                    ((1, 3, 1, 128), (None, AT, AT, AT)), ((1, 3, 1, 128), (AT, AT + 2, AT, AT)), ((1, 3, 1, 128), (AT, AT, AT + 8, AT)),
                                    ((1, 3, 1, 128), (AT, AT, AT, None))])
def test_kv_read_refusals(args, mc, pc, at):
    kv = mc.Kv(**KV)
    assert args.kv_read(C.byref(kv), *_vp(AT, AT, AT, AT), mc.PcKvRead(1, 3, 1, 128)) is None
    assert args.kv_read(C.byref(kv), *_vp(*at), mc.PcKvRead(*pc)) is not None


ATTN = dict(seqs=2, rows_q=10, rows_k=20, heads=4, kv_heads=2, hd=64, q_stride=256, kv_stride=128, o_stride=256, scale=0.125)


@pytest.mark.parametrize("change,at", [
    (dict(heads=0), None), (dict(kv_heads=0), None), (dict(heads=3), None), (dict(heads=34, q_stride=4096, o_stride=4096), None), (dict(hd=80), None),
    (dict(q_stride=248), None), (dict(kv_stride=120), None), (dict(o_stride=260), None), (dict(rows_q=2 ** 31), None), (dict(rows_k=2 ** 31), None),
    (dict(seqs=2 ** 20), None), (dict(scale=0.0), None), (dict(scale=float("nan")), None), (dict(scale=2e4), None),
    ({}, (AT + 2, AT, AT, AT, AT, AT)), ({}, (AT, None, AT, AT, AT, AT)), ({}, (AT, AT, AT + 8, AT, AT, AT)), ({}, (AT, AT, AT, None, AT, AT)),
    ({}, (AT, AT, AT, AT, AT + 1, AT)), ({}, (AT, AT, AT, AT, AT, None))])
def test_attn_refusals(args, mc, change, at):
    assert args.attn(*_vp(AT, AT, AT, AT, AT, AT), mc.PcAttn(**ATTN)) is None
    assert args.attn(*_vp(*(at or (AT,) * 6)), mc.PcAttn(**{**ATTN, **change})) is not None


def test_attn_accepts_nothing_to_do(args, mc):
    assert args.attn(*_vp(*(None,) * 6), mc.PcAttn(**{**ATTN, "rows_q": 0})) is None
    assert args.attn(*_vp(*(None,) * 6), mc.PcAttn(**{**ATTN, "seqs": 0})) is None
    assert args.attn(*_vp(AT, None, None, AT, AT, AT), mc.PcAttn(**{**ATTN, "rows_k": 0})) is None


DECODE = dict(seqs=2, heads=4, max_len=40, table_stride=3, q_stride=256, o_stride=256, scale=0.125)


@pytest.mark.parametrize("change,at", [
    (dict(heads=0), None), (dict(heads=5), None), (dict(heads=34), None), (dict(max_len=49), None), (dict(max_len=2 ** 31, table_stride=2 ** 30), None),
    (dict(table_stride=0), None), (dict(q_stride=250), None), (dict(o_stride=128), None), (dict(seqs=2 ** 20), None), (dict(scale=-1.0), None),
    ({}, (None, AT, AT, AT)), ({}, (AT, None, AT, AT)), ({}, (AT, AT, AT + 3, AT)), ({}, (AT, AT, AT, AT + 8))])
def test_decode_refusals(args, mc, change, at):
    kv = mc.Kv(**KV)
    assert args.decode(C.byref(kv), *_vp(AT, AT, AT, AT), mc.PcAttnDecode(**DECODE)) is None
    assert args.decode(C.byref(kv), *_vp(*(at or (AT,) * 4)), mc.PcAttnDecode(**{**DECODE, **change})) is not None


def test_decode_accepts_nothing_to_do(args, mc):
    kv = mc.Kv(**KV)
    assert args.decode(C.byref(kv), *_vp(*(None,) * 4), mc.PcAttnDecode(**{**DECODE, "seqs": 0})) is None
    assert args.decode(C.byref(kv), *_vp(AT, None, AT, AT), mc.PcAttnDecode(**{**DECODE, "max_len": 0})) is None
