"""Calls of the attention half that lie at the edge of what is allowed: flags of masked blocks under many short items, refusals with
nothing else to do, values at the end of a type's range, scores far beyond fp32's whole numbers, offsets that leave rows out."""
import ctypes as C

import numpy as np
import pytest
import torch

from . import attn_ref as R
from .test_gpu_attn import NO_SLOT, Attn, AttnRows, AttnW, Cache, _attn, _f16, _gen, _refused, _starts, _u32, on  # noqa: F401

pytestmark = pytest.mark.gpu


# ---- values that a masked block hides from some rows ------------------------------------------------
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_attn_infinity_before_many_unmasked_items(on, hd, value):
    """One query over 200 keys with a value that is not finite in its last, masked block, and several hundred queries over whole
    blocks, which mask nothing: the value reaches the row that sees it, whatever number of items stands behind it."""
    g, heads, kv_heads, short = _gen(hd), 8, 8, 400
    lk = [200] + [128] * short
    q, k, v = _f16(g, short + 1, heads, hd), _f16(g, sum(lk), kv_heads, hd), _f16(g, sum(lk), kv_heads, hd)
    v[150, :, 5] = value
    out = torch.full_like(q, 7.0)
    cu_q, cu_k = _starts([1] * (short + 1)), _starts(lk)
    on.attn(q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(), out.data_ptr(), short + 1, short + 1, sum(lk), heads, kv_heads, hd)
    on.flush()
    seen = out[0, :, 5]
    assert torch.isnan(seen).all() if np.isnan(value) else (seen == value).all()
    out[0, :, 5] = 0
    v[150, :, 5] = 0
    at = 0
    for i, n in enumerate(lk):
        o, mass, size = R.attention(q[i:i + 1].double(), k[at:at + n].double(), v[at:at + n].double(), hd ** -0.5, n - 1)
        if i == 0:
            o[:, :, 5] = 0
        R.check(out[i:i + 1], o, mass, size, hd, n)
        at += n


# ---- refusals that only the device can see --------------------------------------------------------
@pytest.mark.parametrize("lengths", [[33], [0xFFFFFFFF], [0xFFFFFFFF, 0], [0, 33, 0, 0x80000000]])
def test_lengths_beyond_the_bound_with_nothing_else_to_do(mc, lengths):
    """Every sequence refused or empty: zeros, and the status says so."""
    seqs = len(lengths)
    kv = Cache(mc, _gen(3), 4, 16, 1, 64, False)
    table, length = torch.zeros(seqs, 2, device="cuda", dtype=torch.int32), _u32(lengths)
    q, out = _f16(_gen(4), seqs, 64), torch.full((seqs + 1, 64), 7.0, device="cuda", dtype=torch.float16)
    _refused(mc, lambda c: c.attn_decode(kv.c, q.data_ptr(), table.data_ptr(), length.data_ptr(), out.data_ptr(), seqs, 1, 32, 2), "length")
    assert (out[:seqs] == 0).all() and (out[seqs:] == 7).all()


@pytest.mark.parametrize("cu,rows,read,left", [([0, 20, 50], 40, (0, 20), (20, 40)), ([0, 41], 40, None, (0, 40)), ([0, 30, 10, 40], 40, None, None),
                                               ([50, 60], 40, None, (0, 40)), ([0xFFFFFFF0, 5], 40, None, (0, 40))])
def test_kv_read_ranges_outside_the_rows(mc, cu, rows, read, left):
    """Offsets that fall or pass the rows: the status says so, rows of such a sequence are left, nothing behind the rows is written."""
    kv = Cache(mc, _gen(5), 5, 16, 2, 64, False)
    table = torch.arange(5, device="cuda", dtype=torch.int32).repeat(len(cu) - 1, 1).contiguous()
    k, v = (torch.full((rows + 3, 128), 7.0, device="cuda", dtype=torch.float16) for _ in range(2))
    at = _u32(cu)
    _refused(mc, lambda c: c.kv_read(kv.c, table.data_ptr(), at.data_ptr(), k.data_ptr(), v.data_ptr(), len(cu) - 1, rows, 5), "row range")
    assert (k[rows:] == 7).all() and (v[rows:] == 7).all()
    if left is not None:
        assert (k[left[0]:left[1]] == 7).all() and (v[left[0]:left[1]] == 7).all()
    if read is not None:
        want = kv.rows(torch.arange(5, device="cuda"), read[1])
        for t, w in zip((k, v), want):
            assert torch.equal(t[read[0]:read[1]].view(-1, 2, 64), w.half())


def test_kv_read_rows_before_the_first_sequence(on, mc):
    """Offsets that begin behind 0, as moe_cuda_attn takes them: the rows before are left, and nothing is wrong."""
    kv = Cache(mc, _gen(6), 3, 16, 2, 64, True)
    table = torch.tensor([[2, 0, 1]], device="cuda", dtype=torch.int32)
    k, v = (torch.full((50, 128), 7.0, device="cuda", dtype=torch.float16) for _ in range(2))
    cu = _u32([9, 49])
    on.kv_read(kv.c, table.data_ptr(), cu.data_ptr(), k.data_ptr(), v.data_ptr(), 1, 50, 3)
    on.flush()
    for t, w in zip((k, v), kv.rows(table[0].long(), 40)):
        assert torch.equal(t[9:49].view(40, 2, 64), w.half())
        assert (t[:9] == 7).all() and (t[49:] == 7).all()


# ---- the ends of the types ---------------------------------------------------------------------------
@pytest.mark.parametrize("hd", [64, 128])
def test_largest_values_through_an_e4m3_cache(on, mc, hd):
    """fp16 values up to 65504 come back finite: those that are kept as 256 * 256 as 65504.  Infinities come back as infinities."""
    x = torch.zeros(6, hd, device="cuda", dtype=torch.float16)
    x[0, :8] = torch.tensor([65504.0, -65504.0, 63488.0, 63456.0, 61440.0, 57376.0, 57344.0, 1.0], device="cuda")
    x[1, :2] = torch.tensor([57344.0, -57344.0], device="cuda")      # the largest that scale 128 holds
    x[2, 0], x[2, 1] = float("inf"), 65504.0
    x[3, 0] = -float("inf")
    x[4] = 65504.0
    x[5, 3] = 2.0 ** -14
    kv = Cache(mc, _gen(1), 1, 16, 1, hd, True)
    slot, cu, table = _u32(range(6)), _u32([0, 6]), _u32([0])
    k, v = torch.empty_like(x), torch.empty_like(x)
    on.kv_write(kv.c, x.data_ptr(), x.data_ptr(), slot.data_ptr(), 6)
    on.kv_read(kv.c, table.data_ptr(), cu.data_ptr(), k.data_ptr(), v.data_ptr(), 1, 6, 1)
    on.flush()
    assert torch.equal(k, v)
    assert torch.equal(torch.isinf(k), torch.isinf(x)) and torch.equal(k[torch.isinf(x)], x[torch.isinf(x)])
    code, scale = R.e4m3(x)
    want = (code.double() * scale.double()[..., None])
    want = torch.where(want.abs() == 65536, want.sign() * 65504, want)[~torch.isinf(x)]
    assert torch.equal(k[~torch.isinf(x)].double(), want)
    assert k[0, 0] == 65504 and k[0, 1] == -65504 and k[0, 2] == 65504 and k[0, 3] == 61440 and (k[4] == 65504).all()


@pytest.mark.parametrize("scale", [256.0, 300.0, 2.0 ** 15, 146.2857])
def test_read_of_products_beyond_the_type(on, mc, scale):
    """Codes and scales of any origin: a product rounds to fp16, what lies beyond 65536 is infinite, up to there the largest value."""
    kv = Cache(mc, _gen(2), 16, 16, 1, 64, True)
    kv.k.view(torch.uint8).copy_(torch.arange(256, device="cuda", dtype=torch.uint8).repeat(64).view(16, 1, 16, 64))
    kv.v.copy_(kv.k)
    for t in kv.scales:
        t[:] = scale
    cu, table = _u32([0, 256]), _u32(range(16))
    k, v = (torch.empty(256, 64, device="cuda", dtype=torch.float16) for _ in range(2))
    on.kv_read(kv.c, table.data_ptr(), cu.data_ptr(), k.data_ptr(), v.data_ptr(), 1, 256, 16)
    on.flush()
    y = kv.k.view(256, 64).double() * float(np.float32(scale))
    want = torch.where((y.abs() >= 65504) & (y.abs() <= 65536), y.sign() * 65504, y).float().half()   # y has 4 + 24 bits: float is one rounding early only for 146.2857
    got = k.clone()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    ok = ~torch.isnan(want)
    assert torch.equal(torch.isinf(got[ok]), torch.isinf(want[ok]))
    fin = ok & ~torch.isinf(want)
    assert ((got[fin].double() - want[fin].double()).abs() <= want[fin].double().abs() * 2.0 ** -10).all()   # one step: the early rounding may fall on a tie
    assert torch.equal(torch.nan_to_num(k), torch.nan_to_num(v))


# ---- scores far beyond fp32's whole numbers -----------------------------------------------------------
def _whole(g, most, *shape):
    return torch.randint(-most, most + 1, shape, device="cuda", generator=g).half()


def _check_sharp(got, q, k, v, offset, scale):
    """Whole queries and keys: scores are exact, and two that differ, differ by the scale at least.  With 2^-scale far below every
    rounding a row is the mean of the values at its largest score.  Weights of the largest are equal but for 2^-20 (the two ways
    of taking 2^x) and round to fp16 for the product, their sum does not: 2^-11 of the mean of |v|; the output rounds by 2^-11."""
    h, g = q.shape[1], k.shape[1]
    seen = torch.arange(k.shape[0], device="cuda")[None] <= torch.arange(q.shape[0], device="cuda")[:, None] + offset
    assert torch.isfinite(got).all()
    for a in range(h):
        b = a // (h // g)
        x = (q[:, a].double() @ k[:, b].double().T).masked_fill(~seen, -float("inf"))
        p = (x == x.amax(-1, keepdim=True)).double()
        p = p / p.sum(-1, keepdim=True)
        o = p @ v[:, b].double()
        tol = 2.0 ** -11 * o.abs() + 2.0 ** -25 + (2.0 ** -11 + 2.0 ** -19) * (p @ v[:, b].double().abs())
        assert ((got[:, a].double() - o).abs() <= tol).all()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,scale", [(8, 64.0), (8, 4096.0), (20, 1e4), (2, 3000.0)])
def test_decode_scores_beyond_whole_numbers(on, mc, e4m3, hd, heads, scale):
    g, kv_heads, page, lengths = _gen(int(scale) + heads), 2, 16, [1, 700, 33, 5000, 128]
    need = [-(-n // page) for n in lengths]
    kv = Cache(mc, g, sum(need), page, kv_heads, hd, e4m3)
    order, at = torch.arange(sum(need), device="cuda", dtype=torch.int32), 0
    table = torch.zeros(len(need), max(need), device="cuda", dtype=torch.int32)
    for i, m in enumerate(need):
        table[i, :m] = order[at:at + m]
        at += m
    total = sum(need) * page
    k = _whole(g, 16, total, kv_heads, hd) * (4 if e4m3 else 5)   # 16 and below are e4m3 values at any power of two
    v = _f16(g, total, kv_heads, hd).clamp_(-3.5, 3.5)
    v[..., 0] = 4.0   # one scale for all values: rows of equal scores keep equal weights
    slot = torch.arange(total, device="cuda", dtype=torch.int32)
    on.kv_write(kv.c, k.data_ptr(), v.data_ptr(), slot.data_ptr(), total)
    q, length = _whole(g, 64, len(lengths), heads, hd), _u32(lengths)
    out = torch.full_like(q, 7.0)
    on.attn_decode(kv.c, q.data_ptr(), table.data_ptr(), length.data_ptr(), out.data_ptr(), len(lengths), heads, max(lengths), max(need), scale=scale)
    on.flush()
    at = 0
    for i, n in enumerate(lengths):
        _, vv = kv.rows(table[i, :need[i]].long(), n)
        _check_sharp(out[i:i + 1], q[i:i + 1], k[at * page:at * page + n], vv, n - 1, scale)
        at += need[i]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("scale", [64.0, 1000.0, 4096.0, 1e4])
def test_attn_scores_beyond_whole_numbers(on, hd, scale):
    """Logits of 10^8 and more: no weight overflows, none that counts is lost, and the maximum of a row is found across its blocks."""
    g, heads, kv_heads, lq, lk = _gen(int(scale)), 6, 2, [300, 5, 1], [700, 5, 384]
    q, k, v = _whole(g, 64, sum(lq), heads, hd), _whole(g, 64, sum(lk), kv_heads, hd), _f16(g, sum(lk), kv_heads, hd)
    q[200:230] = 0   # rows of equal scores beside them in the same tile
    out = torch.full_like(q, 7.0)
    cu_q, cu_k = _starts(lq), _starts(lk)
    on.attn(q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(), out.data_ptr(), len(lq), sum(lq), sum(lk), heads, kv_heads, hd, scale=scale)
    on.flush()
    a = b = 0
    for m, n in zip(lq, lk):
        rows = [i for i in range(a, a + m) if not 200 <= i < 230]
        lo, hi = (0, 200) if a == 0 else (0, m)
        _check_sharp(out[a + lo:a + hi], q[a + lo:a + hi], k[b:b + n], v[b:b + n], n - m + lo, scale)
        if a == 0:
            _check_sharp(out[230:300], q[230:300], k[:n], v[:n], n - m + 230, scale)
            o, mass, size = R.attention(q[200:230].double(), k[:n].double(), v[:n].double(), scale, n - m + 200)
            R.check(out[200:230], o, mass, size, hd, n)
        assert rows
        a, b = a + m, b + n


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("scale", [1e-30, 1e-38, 1e-42])
def test_attn_scales_next_to_zero(on, hd, scale):
    """All visible keys weigh the same, masked ones nothing, down to scales below the normal numbers."""
    _attn(on, _gen(7), [200, 3, 130], [200, 300, 130], 4, 2, hd, scale=scale)


# ---- one slot, two rows ------------------------------------------------------------------------------
@pytest.mark.parametrize("e4m3", [False, True])
def test_one_slot_twice_touches_no_other(on, mc, e4m3):
    g = _gen(8)
    kv = Cache(mc, g, 8, 16, 4, 128, e4m3)
    rows = 100
    x, y = _f16(g, rows, 512), _f16(g, rows, 512)
    slot = torch.randperm(128, device="cuda", generator=g)[:rows].int()
    slot[50:60] = slot[40]
    slot[99] = slot[40]
    before = [t.clone().view(torch.uint8) for t in (kv.k, kv.v)]
    on.kv_write(kv.c, x.data_ptr(), y.data_ptr(), slot.data_ptr(), rows)
    on.flush()
    single = [i for i in range(rows) if int((slot == slot[i]).sum()) == 1]
    for t, b, s in zip((kv.k, kv.v), before, (x, y)):
        code = R.e4m3(s.view(rows, 4, 128))[0].view(torch.uint8) if e4m3 else s.view(rows, 4, 128).view(torch.uint8)
        got = t.view(torch.uint8)
        for i in single:
            b[int(slot[i]) // 16, :, int(slot[i]) % 16] = code[i]
        b[int(slot[40]) // 16, :, int(slot[40]) % 16] = got[int(slot[40]) // 16, :, int(slot[40]) % 16]
        assert torch.equal(got, b)


# ---- the C host side ---------------------------------------------------------------------------------
def _host(pkg, mc):
    pkg.build.build_host()
    L = C.CDLL(pkg.build.HOST_LIB)
    L.moe_attn_open.restype = L.moe_attn_prompt.restype = L.moe_attn_step.restype = C.c_bool
    L.moe_attn_open.argtypes = [C.POINTER(Attn), C.c_void_p] + [C.c_uint32] * 5 + [C.c_float, C.c_uint32, C.c_uint32]
    L.moe_attn_close.argtypes = [C.POINTER(Attn)]
    L.moe_attn_prompt.argtypes = [C.POINTER(Attn), C.POINTER(mc.Kv), C.POINTER(AttnW), C.POINTER(AttnRows), C.c_void_p, C.c_void_p, C.c_uint32]
    L.moe_attn_step.argtypes = [C.POINTER(Attn), C.POINTER(mc.Kv), C.POINTER(AttnW), C.POINTER(AttnRows), C.c_void_p, C.c_uint32]
    return L


class _Layer:
    """A layer's attention of 2 x 64 columns over 256, with a cache of one sequence."""

    def __init__(self, on, pkg, mc, rot, rows, keys, seed=71):
        self.L, self.d, self.h, self.g, self.hd, self.seed = _host(pkg, mc), 256, 2, 1, 64, seed
        gen = _gen(seed)
        self.q = Attn()
        self.opened = self.L.moe_attn_open(C.byref(self.q), on.p, self.d, self.h, self.g, self.hd, rot, 1e4, rows, keys)
        self.qkv, self.wo = _f16(gen, self.q.cols, self.d) * 0.06, _f16(gen, self.d, self.h * self.hd) * 0.05
        self.w = AttnW(self.qkv.data_ptr(), self.wo.data_ptr())
        self.kv = Cache(mc, gen, 16, 16, self.g, self.hd, False)
        self.table = torch.arange(16, device="cuda", dtype=torch.int32)

    def rows(self, rows, kept, seqs=1, value=7.0):
        gen = _gen(self.seed + rows)
        self.x, self.pos = _f16(gen, rows, self.d), torch.arange(rows, device="cuda", dtype=torch.int32)
        self.slot = torch.where(self.pos < kept, self.pos, -1).int()
        self.out = torch.full((rows, self.d), value, device="cuda")
        return AttnRows(rows, seqs, self.x.data_ptr(), None, NO_SLOT, self.pos.data_ptr(), self.slot.data_ptr(), self.table.data_ptr(), 16, self.out.data_ptr())

    def close(self):
        self.L.moe_attn_close(C.byref(self.q))


def test_host_attention_says_what_it_refuses(on, mc, pkg):
    """Too many rows, too many keys, a step of other rows than sequences: false, nothing written, and the context goes on."""
    y = _Layer(on, pkg, mc, 64, 8, 8)
    assert y.opened
    cu, length = _u32([0, 8]), _u32([8])
    for run in (lambda r: y.L.moe_attn_prompt(C.byref(y.q), C.byref(y.kv.c), C.byref(y.w), C.byref(r), cu.data_ptr(), None, 0),
                lambda r: y.L.moe_attn_step(C.byref(y.q), C.byref(y.kv.c), C.byref(y.w), C.byref(r), length.data_ptr(), 16)):
        assert run(y.rows(9, 9, 9)) is False and (y.out == 7).all()
    r = y.rows(8, 8)
    assert y.L.moe_attn_prompt(C.byref(y.q), C.byref(y.kv.c), C.byref(y.w), C.byref(r), cu.data_ptr(), cu.data_ptr(), 9) is False
    assert y.L.moe_attn_step(C.byref(y.q), C.byref(y.kv.c), C.byref(y.w), C.byref(r), length.data_ptr(), 16) is False
    on.flush()
    assert (y.out == 7).all()
    assert y.L.moe_attn_prompt(C.byref(y.q), C.byref(y.kv.c), C.byref(y.w), C.byref(r), cu.data_ptr(), None, 0) is True
    on.flush()
    assert not (y.out == 7).any()
    r0 = y.rows(0, 0)
    assert y.L.moe_attn_prompt(C.byref(y.q), C.byref(y.kv.c), C.byref(y.w), C.byref(r0), cu.data_ptr(), None, 0) is True   # nothing to do
    y.close()


def test_host_attention_without_rotation(on, mc, pkg):
    """rot 0: queries and keys stay as projected."""
    y = _Layer(on, pkg, mc, 0, 8, 0)
    cu = _u32([0, 8])
    r = y.rows(8, 8)
    y.L.moe_attn_prompt(C.byref(y.q), C.byref(y.kv.c), C.byref(y.w), C.byref(r), cu.data_ptr(), None, 0)
    on.flush()
    p = (y.x.double() @ y.qkv.double().T)[:, :4 * 64].view(8, 4, 64)
    o, mass, size = R.attention(p[:, :2], p[:, 2:3], p[:, 3:], 0.125, 0)
    # half a step of fp16 in queries, keys and values and in the weights of the second product; sums of 256 fp32 products
    e = R.bound(o, mass, size, 64, 8) + mass * (2 * 2.0 ** -10 * size[..., None] * 1.1 + 2.0 ** -10)
    assert ((y.out.double() - o.view(8, -1) @ y.wo.double().T).abs() <= e.view(8, -1) @ y.wo.double().abs().T * 1.01 + 1e-5).all()
    y.close()


def test_host_attention_of_a_padded_batch(on, mc, pkg):
    """Rows behind the last sequence: their output is zero, whatever an earlier call has left in the buffers."""
    y = _Layer(on, pkg, mc, 64, 40, 0)
    whole, cu = _u32([0, 40]), _u32([0, 27])
    r = y.rows(40, 40)
    y.L.moe_attn_prompt(C.byref(y.q), C.byref(y.kv.c), C.byref(y.w), C.byref(r), whole.data_ptr(), None, 0)
    on.flush()
    full = y.out.clone()
    r = y.rows(40, 27)
    y.L.moe_attn_prompt(C.byref(y.q), C.byref(y.kv.c), C.byref(y.w), C.byref(r), cu.data_ptr(), None, 0)
    on.flush()
    assert torch.equal(y.out[:27], full[:27])   # causal: the same rows
    assert (y.out[27:] == 0).all()
    y.close()


def test_host_attention_of_no_sequence(on, mc, pkg):
    """Rows, but no sequence, and no offsets: all of the output is zero."""
    y = _Layer(on, pkg, mc, 64, 40, 0)
    r = y.rows(40, 40)
    cu = _u32([0, 40])
    assert y.L.moe_attn_prompt(C.byref(y.q), C.byref(y.kv.c), C.byref(y.w), C.byref(r), cu.data_ptr(), None, 0)
    r = y.rows(40, 0, seqs=0)
    assert y.L.moe_attn_prompt(C.byref(y.q), C.byref(y.kv.c), C.byref(y.w), C.byref(r), None, None, 0)
    on.flush()
    assert (y.out == 0).all()
    y.close()


@pytest.mark.parametrize("rows,row,first", [(1, 16, 0), (40, 4096, 27), (40, 4096, 40), (40, 48, 41), (40, 48, 0xFFFFFFFF), (3000, 2048, 1)])
def test_clear_behind(on, rows, row, first):
    """Rows from *first on, none where that passes the rows, nothing behind them."""
    out, at = torch.full((rows + 1, row), 7, device="cuda", dtype=torch.uint8), _u32([first])
    on.clear_behind(out.data_ptr(), at.data_ptr(), rows, row)
    on.flush()
    assert (out[:min(first, rows)] == 7).all() and (out[min(first, rows):rows] == 0).all() and (out[rows] == 7).all()


# ---- waits ----------------------------------------------------------------------------------------------
def test_attn_longer_than_the_wait_limit(on, mc):
    """The limit is for a pipeline that does not move: a tile over two million keys takes many times it and ends in order."""
    mc.lib().moe_cuda_set_wait_ns(on.p, 1_000_000)
    g, n, hd = _gen(9), 2_000_000, 64
    q, k, v = _f16(g, 8, 1, hd), _f16(g, n, 1, hd), _f16(g, n, 1, hd)
    out = torch.full_like(q, 7.0)
    cu_q, cu_k = _u32([0, 8]), _u32([0, n])
    on.attn(q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(), out.data_ptr(), 1, 8, n, 1, 1, hd)
    on.flush()
    o, mass, size = R.attention(q.double(), k.double(), v.double(), hd ** -0.5, n - 8)
    R.check(out, o, mass, size, hd, n)


# ---- offsets that pass 32 bits ---------------------------------------------------------------------------
def test_rows_far_apart(on, mc):
    """Columns of rows 2^23 elements apart: projection, positions, cache and prompt attention beyond 2^32 elements."""
    g, rows, h, kv_heads, hd, stride = _gen(12), 600, 4, 2, 64, 2 ** 23 + 8
    cols = (h + 2 * kv_heads) * hd
    x = torch.empty(rows, stride, device="cuda")
    x[:, :cols] = torch.randn(rows, cols, device="cuda", generator=g)
    p = torch.empty(rows, stride, device="cuda", dtype=torch.float16)
    p[:, cols:cols + 8] = 7.0
    out = torch.empty(rows, stride, device="cuda", dtype=torch.float16)
    out[:, h * hd:h * hd + 8] = 7.0
    pos, cu = torch.zeros(rows, device="cuda", dtype=torch.int32), _u32([0, rows])
    on.rope(x.data_ptr(), pos.data_ptr(), p.data_ptr(), rows, h + 2 * kv_heads, h + kv_heads, hd, hd, 1e4, stride, stride)
    at = p.data_ptr()
    on.attn(at, at + 2 * h * hd, at + 2 * (h + kv_heads) * hd, cu.data_ptr(), cu.data_ptr(), out.data_ptr(), 1, rows, rows, h, kv_heads, hd, stride, stride, stride)
    kv = Cache(mc, g, -(-rows // 16), 16, kv_heads, hd, False)
    slot = torch.arange(rows, device="cuda", dtype=torch.int32)
    on.kv_write(kv.c, at + 2 * h * hd, at + 2 * (h + kv_heads) * hd, slot.data_ptr(), rows, stride)
    table, back = torch.arange(-(-rows // 16), device="cuda", dtype=torch.int32), [out[:, 1024:], out[:, 2048:]]
    on.kv_read(kv.c, table.data_ptr(), cu.data_ptr(), back[0].data_ptr(), back[1].data_ptr(), 1, rows, table.numel(), stride)
    on.flush()
    y = x[:, :cols].half()   # position 0 turns nothing
    assert torch.equal(p[:, :cols], y) and (p[:, cols:cols + 8] == 7).all() and (out[:, h * hd:h * hd + 8] == 7).all()
    q, k, v = (y[:, a * hd:b * hd].reshape(rows, -1, hd) for a, b in ((0, h), (h, h + kv_heads), (h + kv_heads, h + 2 * kv_heads)))
    for t, w in zip(back, (k, v)):
        assert torch.equal(t[:, :kv_heads * hd], w.reshape(rows, -1))
    R.check(out[:, :h * hd].reshape(rows, h, hd), *R.attention(q.double(), k.double(), v.double(), hd ** -0.5, 0), hd, rows)
