"""The attention half of a layer against plain 64-bit forms: rotary positions, the paged key-value cache (fp16 and e4m3),
attention over packed prompts and of one new token over the cache, alone and together."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from . import attn_ref as R

pytestmark = pytest.mark.gpu
NO_SLOT = 0xFFFFFFFF


@pytest.fixture()
def on(mc):
    """A context on a torch stream that is current for the test."""
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        c = mc.Ctx(0, stream.cuda_stream)
        c.check()
        yield c
        torch.cuda.synchronize()
        c.close()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _f16(gen, *shape):
    return torch.randn(shape, device="cuda", generator=gen).half()


def _u32(values):
    return torch.from_numpy(np.asarray(values, dtype=np.uint32).view(np.int32)).cuda()


def _starts(lengths):
    return _u32(np.concatenate([[0], np.cumsum(lengths)]))


# ---- rotary positions ---------------------------------------------------------------------------
@pytest.mark.parametrize("rows,heads,rot_heads,hd,rot,theta,gap", [
    (1, 1, 1, 64, 64, 1e4, 0), (37, 6, 4, 128, 128, 1e6, 8), (5, 40, 36, 128, 64, 1e6, 0), (300, 20, 16, 64, 48, 5e5, 16),
    (1201, 3, 3, 8, 8, 1e4, 0), (3, 5, 0, 64, 0, 0.0, 0), (9, 2, 1, 512, 512, 1e7, 8)])
def test_rope(on, rows, heads, rot_heads, hd, rot, theta, gap):
    g = _gen(rows)
    n = heads * hd
    x = torch.randn(rows, n + gap, device="cuda", generator=g) * 3
    pos = torch.randint(0, 2 ** 20, (rows,), device="cuda", generator=g, dtype=torch.int32)
    pos[0] = 0
    if rows > 4:
        pos[3], pos[4] = -1, 2 ** 31 - 1   # the largest unsigned position
    out = torch.full((rows + 1, n + 2 * gap), 7.0, device="cuda", dtype=torch.float16)
    on.rope(x.data_ptr(), pos.data_ptr() if rot_heads else None, out.data_ptr(), rows, heads, rot_heads, hd, rot, theta, n + gap, n + 2 * gap)
    on.flush()
    z = x[:, :n].double().view(rows, heads, hd)
    ref, err = z.clone(), torch.zeros_like(z)
    if rot_heads:
        half = rot // 2
        a = (pos.long() & 0xFFFFFFFF).double()[:, None] * torch.tensor([float(np.float32(theta)) ** (-i / half) for i in range(half)], device="cuda", dtype=torch.float64)
        c, s = a.cos()[:, None], a.sin()[:, None]
        lo, hi = z[:, :rot_heads, :half], z[:, :rot_heads, half:rot]
        ref[:, :rot_heads, :half], ref[:, :rot_heads, half:rot] = lo * c - hi * s, hi * c + lo * s
        # sines: the turn's fraction rounds to 24 bits (pi * 2^-24 of angle), 64-bit products of positions up to 2^32 and
        # frequencies with some steps of 2^-53 each (2^32 * 2^-50 * 2 pi), two steps of the function itself; three fp32 roundings
        err[:, :rot_heads, :half] = err[:, :rot_heads, half:rot] = (lo.abs() + hi.abs()) * (math.pi * 2.0 ** -24 + math.pi * 2.0 ** -17 * 0.5 + 5 * 2.0 ** -24)
    got = out[:rows, :n].double().view(rows, heads, hd)
    assert ((got - ref).abs() <= ref.abs() * 2.0 ** -11 + 2.0 ** -25 + err * 1.01).all()
    assert (out[rows:] == 7).all() and (out[:, n:] == 7).all()


def test_rope_far_positions_are_exact_to_fp16(on):
    """Positions up to 2^20 with the plain bound (no allowance for a position times a frequency)."""
    rows, hd = 512, 128
    g = _gen(1)
    x = torch.randn(rows, hd, device="cuda", generator=g)
    pos = torch.randint(2 ** 19, 2 ** 20, (rows,), device="cuda", generator=g, dtype=torch.int32)
    out = torch.empty(rows, hd, device="cuda", dtype=torch.float16)
    on.rope(x.data_ptr(), pos.data_ptr(), out.data_ptr(), rows, 1, 1, hd, hd, 10000.0)
    on.flush()
    a = pos.double()[:, None] * torch.tensor([10000.0 ** (-i / 64) for i in range(64)], device="cuda", dtype=torch.float64)
    lo, hi = x[:, :64].double(), x[:, 64:].double()
    ref = torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin()], 1)
    far = (lo.abs() + hi.abs()).repeat(1, 2)
    assert ((out.double() - ref).abs() <= ref.abs() * 2.0 ** -11 + 2.0 ** -25 + far * 1e-6).all()


# ---- the cache ----------------------------------------------------------------------------------
class Cache:
    def __init__(self, mc, gen, pages, page, heads, hd, e4m3, fill=None):
        self.page, self.heads, self.hd, self.e4m3 = page, heads, hd, e4m3
        shape = (pages, heads, page, hd)
        x = [_f16(gen, *shape) for _ in range(2)] if fill is None else [torch.full(shape, fill, device="cuda", dtype=torch.float16) for _ in range(2)]
        self.scales = None
        if e4m3:
            (self.k, ks), (self.v, vs) = (R.e4m3(t * torch.exp2(torch.randint(-6, 6, t.shape[:3], device="cuda", generator=gen).float())[..., None].half()) for t in x)
            self.scales = [ks.contiguous(), vs.contiguous()]
        else:
            self.k, self.v = x
        at = [t.data_ptr() for t in self.scales] if e4m3 else [None, None]
        self.c = mc.Kv(k=self.k.data_ptr(), v=self.v.data_ptr(), k_scale=at[0], v_scale=at[1], pages=pages, page=page, kv_heads=heads, hd=hd,
                       type=mc.KV_E4M3 if e4m3 else mc.KV_F16)

    def rows(self, pages, n):
        """The first n tokens on these pages, [n, heads, hd] in float64."""
        out = []
        for i, t in enumerate((self.k, self.v)):
            x = t.view(torch.uint8)[pages].view(torch.float8_e4m3fn).double() if self.e4m3 else t[pages].double()
            if self.e4m3:
                x = x * self.scales[i][pages].double()[..., None]
            out.append(x.transpose(1, 2).reshape(-1, self.heads, self.hd)[:n])
        return out


def _table(gen, lengths, page, pages, stride):
    order = torch.randperm(pages, device="cuda", generator=gen).int()
    table = torch.full((len(lengths), stride), 0x7FFFFFFF, device="cuda", dtype=torch.int32)   # unused entries are never looked at
    at = 0
    for i, n in enumerate(lengths):
        m = -(-n // page)
        table[i, :m] = order[at:at + m]
        at += m
    return table


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("rows,heads,hd,page,gap", [(1, 1, 64, 16, 0), (7, 4, 128, 64, 640), (129, 3, 128, 16, 0), (1000, 2, 64, 256, 8), (4099, 16, 128, 32, 8)])
def test_kv_write(on, mc, e4m3, rows, heads, hd, page, gap):
    g = _gen(rows + heads)
    pages = -(-rows // page) + 2
    kv = Cache(mc, g, pages, page, heads, hd, e4m3)
    stride = heads * hd + gap
    k, v = _f16(g, rows, stride), _f16(g, rows, stride)
    for t in (k, v):
        t *= torch.exp2(torch.randint(-14, 9, (rows, 1), device="cuda", generator=g).float()).half()
    k[0, :hd] = 0
    v[0, 0] = 65504
    k[rows // 2, 1] = 448 * 2.0 ** -12   # exactly a scale's largest value
    slot = torch.randperm(pages * page, device="cuda", generator=g)[:rows].int()
    if rows > 2:
        slot[1] = -1   # not kept
    want = [t.clone().view(torch.uint8 if e4m3 else torch.float16) for t in (kv.k, kv.v)]
    scales = [t.clone() for t in kv.scales] if e4m3 else None
    on.kv_write(kv.c, k.data_ptr(), v.data_ptr(), slot.data_ptr(), rows, stride)
    on.flush()
    kept = slot >= 0
    at = slot[kept].long()
    for i, t in enumerate((k, v)):
        x = t[kept, :heads * hd].view(-1, heads, hd)
        if e4m3:
            code, scale = R.e4m3(x)
            want[i][at // page, :, at % page] = code.view(torch.uint8)
            scales[i][at // page, :, at % page] = scale
            assert torch.equal(kv.scales[i], scales[i])
            assert torch.equal((kv.k, kv.v)[i].view(torch.uint8), want[i])
        else:
            want[i][at // page, :, at % page] = x
            assert torch.equal((kv.k, kv.v)[i], want[i])


def test_kv_write_special_values_and_back(on, mc):
    """NaN, infinities, zeros and subnormals through an e4m3 cache and back."""
    g = _gen(3)
    kv = Cache(mc, g, 1, 16, 1, 64, True)
    x = torch.zeros(6, 64, device="cuda", dtype=torch.float16)
    x[0, 3], x[0, 4] = float("nan"), 1.5
    x[1, 0], x[1, 1], x[1, 2] = float("inf"), -float("inf"), 300.0
    x[2, 5] = 2.0 ** -24
    x[3] = -0.0
    x[4, :3] = torch.tensor([448.0, 17.0, 2.0 ** -9], device="cuda")
    x[5, :] = float("nan")
    slot, cu, table = _u32(range(6)), _u32([0, 6]), _u32([0])
    k, v = torch.empty_like(x), torch.empty_like(x)
    on.kv_write(kv.c, x.data_ptr(), x.data_ptr(), slot.data_ptr(), 6)
    on.kv_read(kv.c, table.data_ptr(), cu.data_ptr(), k.data_ptr(), v.data_ptr(), 1, 6, 1)
    on.flush()
    assert torch.equal(k.view(torch.int16), v.view(torch.int16))
    assert torch.isnan(k[0, 3]) and k[0, 4] == 1.5 and k[0, 0] == 0
    assert k[1, 0] == float("inf") and k[1, 1] == -float("inf") and k[1, 2] == 288   # 300 / 256 = 1.171875 to four bits: 1.125
    assert k[2, 5] == 2.0 ** -24 and (k[3] == 0).all() and torch.isnan(k[5]).all()
    assert k[4, 0] == 448 and k[4, 1] == 16   # 17 lies half way between 16 and 18: the even one
    code, scale = R.e4m3(x)
    want = (code.float() * scale[..., None]).half()
    assert torch.equal(torch.nan_to_num(k, nan=7.0)[2:], torch.nan_to_num(want, nan=7.0)[2:])


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lengths,heads,hd,page,gap", [([1], 1, 64, 16, 0), ([0, 5, 0, 33, 16, 0], 4, 128, 16, 8), ([513, 1, 700], 2, 64, 256, 0),
                                                        ([64] * 40, 16, 128, 64, 0), ([3000], 8, 128, 32, 24)])
def test_kv_read(on, mc, e4m3, lengths, heads, hd, page, gap):
    g = _gen(sum(lengths))
    need = sum(-(-n // page) for n in lengths)
    kv = Cache(mc, g, need + 1, page, heads, hd, e4m3)
    per = max(1, max(-(-n // page) for n in lengths))
    table = _table(g, lengths, page, need + 1, per)
    total, stride = sum(lengths), heads * hd + gap
    k, v = (torch.full((total + 2, stride), 7.0, device="cuda", dtype=torch.float16) for _ in range(2))
    cu = _starts(lengths)
    on.kv_read(kv.c, table.data_ptr(), cu.data_ptr(), k.data_ptr(), v.data_ptr(), len(lengths), total + 2, per, stride)
    on.flush()
    at = 0
    for i, n in enumerate(lengths):
        rk, rv = kv.rows(table[i, :-(-n // page)].long(), n)
        assert torch.equal(k[at:at + n, :heads * hd].view(n, heads, hd), rk.half())
        assert torch.equal(v[at:at + n, :heads * hd].view(n, heads, hd), rv.half())
        at += n
    assert (k[total:] == 7).all() and (k[:, heads * hd:] == 7).all() and (v[total:] == 7).all()


# ---- one new token over the cache ----------------------------------------------------------------
def _decode(on, mc, g, lengths, heads, kv_heads, hd, page, e4m3, gap=0, poison=True, max_len=None):
    need = sum(-(-n // page) for n in lengths)
    kv = Cache(mc, g, need + 1, page, kv_heads, hd, e4m3)
    per = max(1, max(-(-n // page) for n in lengths))
    table = _table(g, lengths, page, need + 1, per)
    rows = [kv.rows(table[i, :-(-n // page)].long(), n) for i, n in enumerate(lengths)]
    if poison:   # what lies behind a sequence's last token on its last page is nobody's
        for i, n in enumerate(lengths):
            if n % page:
                last = int(table[i, n // page])
                for j, t in enumerate((kv.k, kv.v)):
                    t[last, :, n % page:] = float("nan")
                    if e4m3:
                        kv.scales[j][last, :, n % page:] = float("inf") if j else float("nan")
    seqs, length = len(lengths), _u32(lengths)
    q = _f16(g, seqs, heads * hd + gap)
    out = torch.full((seqs + 1, heads * hd + 2 * gap), 7.0, device="cuda", dtype=torch.float16)
    on.attn_decode(kv.c, q.data_ptr(), table.data_ptr(), length.data_ptr(), out.data_ptr(), seqs, heads,
                   max(lengths) if max_len is None else max_len, per, heads * hd + gap, heads * hd + 2 * gap)
    on.flush()
    assert (out[seqs:] == 7).all() and (out[:, heads * hd:] == 7).all()
    for i, n in enumerate(lengths):
        got = out[i:i + 1, :heads * hd].view(1, heads, hd)
        if n == 0:
            assert (got == 0).all()
            continue
        o, mass, size = R.attention(q[i:i + 1, :heads * hd].double().view(1, heads, hd), *rows[i], hd ** -0.5, n - 1)
        R.check(got, o, mass, size, hd, n)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lengths,heads,kv_heads,page", [
    ([1], 1, 1, 16), ([0, 1, 0], 8, 1, 16), ([15, 16, 17, 31, 32, 33, 0, 63, 64, 65], 8, 2, 16), ([777], 32, 4, 64),
    ([5, 1000, 3, 129, 0, 0, 512], 14, 2, 32), ([2049] * 3, 16, 1, 128), ([100, 3000], 10, 10, 256), ([33] * 300, 6, 2, 16)])
def test_decode(on, mc, e4m3, hd, lengths, heads, kv_heads, page):
    _decode(on, mc, _gen(len(lengths) + heads), lengths, heads, kv_heads, hd, page, e4m3)


def test_decode_strides_and_a_loose_bound(on, mc):
    _decode(on, mc, _gen(9), [40, 7, 100], 12, 4, 64, 16, False, gap=24, max_len=112)


@pytest.mark.parametrize("e4m3", [False, True])
def test_decode_long(on, mc, e4m3):
    """One long sequence on the whole chip, several pieces to every head."""
    _decode(on, mc, _gen(4), [100003, 3], 8, 1, 128, 64, e4m3)


def test_decode_far_offsets(on, mc):
    """Pages beyond 2^32 elements of the pool."""
    pages, page, heads, hd = 34000, 256, 4, 128   # 4.46e9 elements each
    k = torch.empty(pages, heads, page, hd, device="cuda", dtype=torch.float16)
    v = torch.empty_like(k)
    g = _gen(5)
    table = torch.tensor([[33999, 3, 33000]], device="cuda", dtype=torch.int32)
    for t in (k, v):
        for p in table[0].tolist():
            t[p] = _f16(g, heads, page, hd)
    kv = mc.Kv(k=k.data_ptr(), v=v.data_ptr(), k_scale=None, v_scale=None, pages=pages, page=page, kv_heads=heads, hd=hd, type=mc.KV_F16)
    n = 700
    row = _f16(g, 2, heads * hd)
    slot = _u32([33000 * 256 + 187, 33999 * 256])   # places 699 and 0
    length, cu = _u32([n]), _u32([0, n])
    on.kv_write(kv, row.data_ptr(), row.data_ptr(), slot.data_ptr(), 2)
    q, out = _f16(g, 1, 8 * hd), torch.empty(1, 8 * hd, device="cuda", dtype=torch.float16)
    on.attn_decode(kv, q.data_ptr(), table.data_ptr(), length.data_ptr(), out.data_ptr(), 1, 8, n, 3)
    kr, vr = torch.empty(n, heads, hd, device="cuda", dtype=torch.float16), torch.empty(n, heads, hd, device="cuda", dtype=torch.float16)
    on.kv_read(kv, table.data_ptr(), cu.data_ptr(), kr.data_ptr(), vr.data_ptr(), 1, n, 3)
    on.flush()
    x = [t[table[0].long()].transpose(1, 2).reshape(-1, heads, hd)[:n] for t in (k, v)]
    assert torch.equal(x[0][699].flatten(), row[0]) and torch.equal(x[0][0].flatten(), row[1])
    assert torch.equal(kr, x[0]) and torch.equal(vr, x[1])
    o, mass, size = R.attention(q.double().view(1, 8, hd), x[0].double(), x[1].double(), hd ** -0.5, n - 1)
    R.check(out.view(1, 8, hd), o, mass, size, hd, n)


def test_decode_large_logits_and_wide_scales(on, mc):
    """Logits far apart, V scales from 2^-20 to 2^6: the rows that carry the weight are the small ones."""
    g = _gen(6)
    n, hd = 200, 64
    kv = Cache(mc, g, 13, 16, 1, hd, True)
    order = torch.arange(13, device="cuda", dtype=torch.int32)[None].contiguous()
    kv.scales[1][:] = 2.0 ** -20
    kv.scales[1][0, 0, 3] = 2.0 ** 6
    kv.scales[0][:] = 2.0 ** -4
    q, length = _f16(g, 1, 4 * hd) * 8, _u32([n])
    rows = kv.rows(order[0].long(), n)
    out = torch.empty(1, 4 * hd, device="cuda", dtype=torch.float16)
    on.attn_decode(kv.c, q.data_ptr(), order.data_ptr(), length.data_ptr(), out.data_ptr(), 1, 4, n, 13)
    on.flush()
    o, mass, size = R.attention(q.double().view(1, 4, hd), *rows, hd ** -0.5, n - 1)
    R.check(out.view(1, 4, hd), o, mass, size, hd, n)


# ---- whole prompts --------------------------------------------------------------------------------
def _attn(on, g, lq, lk, heads, kv_heads, hd, gap=0, poison=False, scale=None):
    nq, nk = sum(lq), sum(lk)
    q, k, v = _f16(g, nq + 1, heads * hd + gap), _f16(g, nk + 1, kv_heads * hd + gap), _f16(g, nk + 1, kv_heads * hd + gap)
    out = torch.full((nq + 1, heads * hd + 2 * gap), 7.0, device="cuda", dtype=torch.float16)
    cq, ck = np.concatenate([[0], np.cumsum(lq)]), np.concatenate([[0], np.cumsum(lk)])
    if poison:
        # the last third of every other sequence's keys and values is NaN or infinite: rows before it must not notice
        for i in range(0, len(lq), 2):
            a, b = ck[i] + lk[i] - lk[i] // 3, ck[i + 1]
            k[a:b] = float("nan")
            v[a:b:2] = float("inf")
            v[a + 1:b:2] = float("nan")
    k[nk], v[nk] = float("nan"), float("nan")   # behind the last sequence
    scale = hd ** -0.5 if scale is None else scale
    cu_q, cu_k = _u32(cq), _u32(ck)
    on.attn(q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(), out.data_ptr(), len(lq), nq, nk, heads, kv_heads,
            hd, heads * hd + gap, kv_heads * hd + gap, heads * hd + 2 * gap, scale)
    on.flush()
    assert (out[nq:] == 7).all() and (out[:, heads * hd:] == 7).all()
    for i in range(len(lq)):
        m = lq[i]
        clean = m
        if poison and i % 2 == 0:
            clean = max(0, min(m, m - lk[i] // 3))   # query r sees keys up to r + lk - lq
        got = out[cq[i]:cq[i] + m, :heads * hd].view(m, heads, hd)
        qq = q[cq[i]:cq[i] + m, :heads * hd].double().view(m, heads, hd)
        kk, vv = (t[ck[i]:ck[i + 1], :kv_heads * hd].double().view(lk[i], kv_heads, hd) for t in (k, v))
        if poison and i % 2 == 0 and clean < m:
            assert torch.isnan(got[clean:]).any(-1).all()
        if clean:
            cut = clean + lk[i] - m   # keys that any clean query sees
            o, mass, size = R.attention(qq[:clean], kk[:max(cut, 0)], vv[:max(cut, 0)], scale, lk[i] - m)
            empty = max(0, min(clean, m - lk[i]))
            assert (got[:empty] == 0).all()
            if empty < clean:
                R.check(got[empty:clean], o[empty:], mass[empty:], size[empty:], hd, lk[i])


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lq,lk,heads,kv_heads", [
    ([1], [1], 1, 1), ([5], [5], 8, 1), ([128], [128], 4, 4), ([129, 1, 127], [129, 1, 127], 6, 2), ([300], [300], 16, 1),
    ([0, 3, 0, 200, 0], [0, 3, 0, 200, 0], 14, 2), ([64, 65], [500, 1065], 8, 8), ([7, 1, 1], [1000, 1, 513], 12, 4),
    ([40, 200, 10], [0, 13, 9], 4, 2), ([384] * 5, [384] * 5, 16, 2), ([1100], [1100], 5, 1), ([513, 2, 1000], [600, 300, 1000], 10, 2)])
def test_attn(on, hd, lq, lk, heads, kv_heads):
    _attn(on, _gen(sum(lq) + heads), lq, lk, heads, kv_heads, hd)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(8, 1), (4, 4), (14, 2)])
def test_attn_masked_places_may_hold_anything(on, hd, heads, kv_heads):
    _attn(on, _gen(heads), [200, 33, 400, 64, 7], [200, 33, 777, 64, 300], heads, kv_heads, hd, poison=True)


def test_attn_strides(on):
    _attn(on, _gen(1), [50, 129], [70, 129], 6, 3, 64, gap=40)
    _attn(on, _gen(2), [50, 129], [70, 129], 4, 1, 128, gap=8)


@pytest.mark.parametrize("scale", [4.0, 1e-3])
def test_attn_scales(on, scale):
    """Logits up to several hundred apart, and next to equal ones."""
    _attn(on, _gen(3), [300], [300], 4, 2, 64, scale=scale)


def test_attn_many_sequences(on):
    rng = np.random.default_rng(0)
    lq = rng.integers(0, 40, 700).tolist()
    _attn(on, _gen(4), lq, [n + int(e) for n, e in zip(lq, rng.integers(0, 30, 700))], 4, 2, 64)


def test_attn_long(on):
    _attn(on, _gen(5), [5000], [6001], 8, 2, 128)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,lq,lk", [(16, 2, [384] * 32, [384] * 32), (12, 4, [700] * 9, [1100] * 9), (1, 1, [20000], [20000]),
                                                  (16, 1, [900, 3, 1500], [900, 3, 1500])])
def test_attn_several_items_to_every_sm_and_call_after_call(on, hd, heads, kv_heads, lq, lk):
    """More tile pairs than SMs, of one key block and of many, and calls one behind the other without a wait between."""
    g = _gen(heads)
    nq, nk = sum(lq), sum(lk)
    q, k, v = _f16(g, nq, heads, hd), _f16(g, nk, kv_heads, hd), _f16(g, nk, kv_heads, hd)
    cq, ck = _starts(lq), _starts(lk)
    outs = [torch.full_like(q, 7.0) for _ in range(4)]
    for out in outs:
        on.attn(q.data_ptr(), k.data_ptr(), v.data_ptr(), cq.data_ptr(), ck.data_ptr(), out.data_ptr(), len(lq), nq, nk, heads, kv_heads, hd)
    on.flush()
    for out in outs[1:]:
        assert torch.equal(out, outs[0])
    a = b = 0
    for m, n in zip(lq, lk):
        for lo in range(0, m, 2500):   # query rows in pieces
            hi = min(m, lo + 2500)
            o, mass, size = R.attention(q[a + lo:a + hi].double(), k[b:b + n].double(), v[b:b + n].double(), hd ** -0.5, n - m + lo)
            R.check(outs[0][a + lo:a + hi], o, mass, size, hd, n)
        a, b = a + m, b + n


# ---- refusals that only the device can see --------------------------------------------------------
def _refused(mc, run, kind):
    """run(context) on a context of its own: MOE_ERR_ARG by the next flush, and later calls do nothing."""
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        c = mc.Ctx(0, stream.cuda_stream)
        c.check()
        run(c)
        with pytest.raises(mc.MoeCudaError, match=kind):
            c.flush()
        assert c.status() == mc.MOE_ERR_ARG
        torch.cuda.synchronize()
        c.close()


@pytest.mark.parametrize("e4m3", [False, True])
def test_slots_outside_the_cache(mc, e4m3):
    g = _gen(1)
    kv = Cache(mc, g, 3, 16, 2, 64, e4m3)
    before = [t.clone() for t in (kv.k.view(torch.uint8), kv.v.view(torch.uint8))]
    x = _f16(g, 4, 128)
    slot = _u32([5, 48, 0x7FFFFFFF, NO_SLOT])

    def run(c):
        c.kv_write(kv.c, x.data_ptr(), x.data_ptr(), slot.data_ptr(), 4)

    _refused(mc, run, "cache slot")
    for t, b in zip((kv.k.view(torch.uint8), kv.v.view(torch.uint8)), before):   # slot 5 alone is written
        same = (t == b).view(3, 2, 16, -1).all(-1).all(1)
        same[0, 5] = True
        assert same.all()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
def test_pages_outside_the_cache(mc, e4m3, hd):
    """Rows of bad pages are left, the others are read; a decode counts their tokens as not there."""
    g = _gen(2)
    kv = Cache(mc, g, 5, 16, 2, hd, e4m3)
    table = torch.tensor([[0, 0x7FFFFFF0, 2], [3, 5, 4]], device="cuda", dtype=torch.int32)
    cu, length = _u32([0, 48, 90]), _u32([48, 42])
    k, v = (torch.full((90, 2 * hd), 7.0, device="cuda", dtype=torch.float16) for _ in range(2))
    q, out = _f16(g, 2, 4 * hd), torch.full((2, 4 * hd), 7.0, device="cuda", dtype=torch.float16)

    def read(c):
        c.kv_read(kv.c, table.data_ptr(), cu.data_ptr(), k.data_ptr(), v.data_ptr(), 2, 90, 3)

    def decode(c):
        c.attn_decode(kv.c, q.data_ptr(), table.data_ptr(), length.data_ptr(), out.data_ptr(), 2, 4, 48, 3)

    _refused(mc, read, "page")
    assert (k[16:32] == 7).all() and (v[64:80] == 7).all()
    rk, _ = kv.rows(torch.tensor([0, 2], device="cuda"), 32)
    assert torch.equal(k[:16].view(16, 2, hd), rk[:16].half()) and torch.equal(k[32:48].view(16, 2, hd), rk[16:].half())
    _refused(mc, decode, "page")
    for i, (pages, n) in enumerate((([0, 2], 32), ([3, 4], 26))):
        x = kv.rows(torch.tensor(pages, device="cuda"), n)
        o, mass, size = R.attention(q[i:i + 1].double().view(1, 4, hd), *x, hd ** -0.5, n - 1)
        R.check(out[i:i + 1].view(1, 4, hd), o, mass, size, hd, n)


def test_lengths_beyond_the_bound(mc):
    g = _gen(3)
    kv = Cache(mc, g, 4, 16, 1, 64, False)
    table, length = torch.tensor([[0, 1], [2, 3]], device="cuda", dtype=torch.int32), _u32([0xFFFFFFFF, 20])
    q, out = _f16(g, 2, 64), torch.full((2, 64), 7.0, device="cuda", dtype=torch.float16)
    _refused(mc, lambda c: c.attn_decode(kv.c, q.data_ptr(), table.data_ptr(), length.data_ptr(), out.data_ptr(), 2, 1, 32, 2), "length")
    assert (out[0] == 0).all()
    x = kv.rows(table[1].long(), 20)
    R.check(out[1:].view(1, 1, 64), *R.attention(q[1:].double().view(1, 1, 64), *x, 0.125, 19), 64, 20)


@pytest.mark.parametrize("cu_q,cu_k", [([0, 9], [0, 40]), ([0, 300], [0, 40]), ([5, 2], [0, 40]), ([0, 9, 5], [0, 20, 40]), ([0, 5, 9], [0, 50, 40])])
def test_row_ranges_outside_the_tensors(mc, cu_q, cu_k):
    """Offsets that fall, or pass the tensors' rows, are refused without a read outside them (8 query rows, 40 key rows)."""
    g = _gen(4)
    q, k, out = _f16(g, 8, 64), _f16(g, 40, 64), torch.full((9, 64), 7.0, device="cuda", dtype=torch.float16)
    a, b = _u32(cu_q), _u32(cu_k)
    _refused(mc, lambda c: c.attn(q.data_ptr(), k.data_ptr(), k.data_ptr(), a.data_ptr(), b.data_ptr(), out.data_ptr(), len(cu_q) - 1, 8, 40, 1, 1, 64), "row range")
    assert (out[8] == 7).all()


def test_many_falling_offsets(mc):
    """Offsets that go to and fro cover the rows many times over: more tiles than the list has room for."""
    g = _gen(5)
    q, k, out = _f16(g, 4096, 16 * 64), _f16(g, 16, 64), torch.empty(4096, 16 * 64, device="cuda", dtype=torch.float16)
    a, b = _u32([0, 4096] * 200), _u32([0, 16] * 200)
    _refused(mc, lambda c: c.attn(q.data_ptr(), k.data_ptr(), k.data_ptr(), a.data_ptr(), b.data_ptr(), out.data_ptr(), 399, 4096, 16, 16, 1, 64), "row range")


def test_attn_without_keys(on):
    _attn(on, _gen(6), [5], [0], 4, 2, 64)
    _attn(on, _gen(6), [5, 300, 1], [0, 0, 0], 4, 2, 128)


def test_work_on_another_current_device(mc):
    """The calling thread's current device is left as it was, and the calls run on the context's."""
    s = _calls_state(mc, 71, [40, 9])
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    c = mc.Ctx(0, stream.cuda_stream)
    with torch.cuda.device(torch.cuda.device_count() - 1):
        _run_of_calls(c, s)
        c.flush()
        assert torch.cuda.current_device() == torch.cuda.device_count() - 1
    assert not (s["od"] == 7).all()
    c.close()


def test_host_refusals_are_sticky(mc):
    with mc.Ctx(0) as c:
        c.check()
        b = c.alloc(4096)
        c.attn(b, b, b, b, b, b, 1, 4, 4, 3, 2, 64)
        assert c.status() == mc.MOE_ERR_ARG and "query heads" in c.last_error()


def test_nothing_to_do(on, mc):
    """No rows, no sequences: no launch, no error."""
    kv = Cache(mc, _gen(1), 1, 16, 1, 64, False)
    n = on.launches()
    on.rope(None, None, None, 0, 1, 1, 64, 64, 1e4)
    on.kv_write(kv.c, None, None, None, 0)
    on.kv_read(kv.c, None, None, None, None, 0, 0, 1)
    on.attn(None, None, None, None, None, None, 0, 0, 0, 1, 1, 64)
    on.attn_decode(kv.c, None, None, None, None, 0, 1, 0, 1)
    on.flush()
    assert on.launches() == n


# ---- streams, graphs, contexts ----------------------------------------------------------------------
def _run_of_calls(c, s):
    """Rotary positions, cache, prompt attention, read-back and a decode step, one behind the other."""
    h, g, hd, rows = 8, 2, 64, s["rows"]
    cols = (h + 2 * g) * hd
    c.rope(s["x"].data_ptr(), s["pos"].data_ptr(), s["p"].data_ptr(), rows, h + 2 * g, h + g, hd, hd, 1e4)
    at = s["p"].data_ptr()
    c.kv_write(s["kv"].c, at + 2 * h * hd, at + 2 * (h + g) * hd, s["slot"].data_ptr(), rows, cols)
    c.attn(at, at + 2 * h * hd, at + 2 * (h + g) * hd, s["cu"].data_ptr(), s["cu"].data_ptr(), s["o"].data_ptr(), 2, rows, rows, h, g, hd, cols, cols)
    c.kv_read(s["kv"].c, s["table"].data_ptr(), s["cu"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), 2, rows, s["table"].shape[1])
    c.attn_decode(s["kv"].c, s["q"].data_ptr(), s["table"].data_ptr(), s["len"].data_ptr(), s["od"].data_ptr(), 2, h, max(s["lengths"]), s["table"].shape[1])


def _calls_state(mc, seed, lengths):
    gen = _gen(seed)
    h, g, hd, page, rows = 8, 2, 64, 16, sum(lengths)
    per = [-(-n // page) for n in lengths]
    kv = Cache(mc, gen, sum(per), page, g, hd, True)
    table = _table(gen, lengths, page, sum(per), max(per))
    place = torch.cat([torch.arange(n, device="cuda") for n in lengths])
    seq = torch.cat([torch.full((n,), i, device="cuda") for i, n in enumerate(lengths)])
    slot = (table[seq, place // page] * page + place % page).int()
    f = lambda *shape: torch.full(shape, 7.0, device="cuda", dtype=torch.float16)  # noqa: E731
    return {"rows": rows, "lengths": lengths, "x": torch.randn(rows, (h + 2 * g) * hd, device="cuda", generator=gen), "pos": place.int(), "slot": slot,
            "kv": kv, "table": table, "cu": _starts(lengths), "len": _u32(lengths), "q": _f16(gen, 2, h * hd), "p": f(rows, (h + 2 * g) * hd),
            "o": f(rows, h * hd), "k": f(rows, g * hd), "v": f(rows, g * hd), "od": f(2, h * hd)}


def test_run_together(on, mc):
    """Each step against the plain form of what the step before it left."""
    s = _calls_state(mc, 11, [75, 130])
    _run_of_calls(on, s)
    on.flush()
    h, g, hd = 8, 2, 64
    p = s["p"].view(-1, h + 2 * g, hd)
    kd, vd = (R.e4m3(p[:, a:a + g]) for a in (h, h + g))
    kd, vd = (c.double() * sc.double()[..., None] for c, sc in (kd, vd))
    assert torch.equal(s["k"].view(-1, g, hd), kd.half()) and torch.equal(s["v"].view(-1, g, hd), vd.half())
    at = 0
    for i, n in enumerate(s["lengths"]):
        q, k, v = (p[at:at + n, a:b].double() for a, b in ((0, h), (h, h + g), (h + g, h + 2 * g)))
        R.check(s["o"][at:at + n].view(n, h, hd), *R.attention(q, k, v, 0.125, 0), hd, n)
        R.check(s["od"][i:i + 1].view(1, h, hd), *R.attention(s["q"][i:i + 1].double().view(1, h, hd), kd[at:at + n], vd[at:at + n], 0.125, n - 1), hd, n)
        at += n


def test_captured_and_replayed(mc):
    """One graph of all calls, replayed on new values in the same buffers; then a second graph of the same context."""
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        c = mc.Ctx(0, stream.cuda_stream)
        c.check()
        a, b = _calls_state(mc, 21, [75, 130]), _calls_state(mc, 22, [300, 1])
        graphs = []
        for s in (a, b):
            _run_of_calls(c, s)   # kernels are loaded before a capture
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                _run_of_calls(c, s)
            graphs.append(graph)
        for s, graph, seed in ((a, graphs[0], 31), (b, graphs[1], 32), (a, graphs[0], 33)):
            s["x"].copy_(torch.randn(s["x"].shape, device="cuda", generator=_gen(seed)))
            for n in ("p", "o", "k", "v", "od"):
                s[n].fill_(7.0)
            graph.replay()
            torch.cuda.synchronize()
            got = {n: s[n].clone() for n in ("p", "o", "k", "v", "od")}
            for n in got:
                s[n].fill_(7.0)
            _run_of_calls(c, s)
            c.flush()
            for n in got:
                assert torch.equal(got[n], s[n]), n
        del graphs
        c.close()


def test_two_contexts_at_once(mc):
    """Two contexts on streams of their own, both at work: each has its own work area."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [mc.Ctx(0, s.cuda_stream) for s in streams]
    states = [_calls_state(mc, 41 + i, n) for i, n in enumerate(([700, 900], [1500, 64]))]
    torch.cuda.synchronize()
    want = []
    for c, s in zip(ctxs, states):
        _run_of_calls(c, s)
        c.flush()
        want.append({n: s[n].clone() for n in ("o", "od", "k")})
    torch.cuda.synchronize()
    for _ in range(5):
        for c, s in zip(ctxs, states):
            _run_of_calls(c, s)
    for c, s, w in zip(ctxs, states, want):
        c.flush()
        for n in w:
            assert torch.equal(s[n], w[n]), n
        c.close()


def test_calls_allocate_nothing(on, mc):
    s = _calls_state(mc, 51, [200, 77])
    _run_of_calls(on, s)
    on.flush()
    free0, _ = torch.cuda.mem_get_info(0)
    mc.lib().moe_cuda_fail_alloc_after(on.p, 1)
    _run_of_calls(on, s)
    on.flush()
    assert torch.cuda.mem_get_info(0)[0] == free0


# ---- the C host side ---------------------------------------------------------------------------------
class Attn(C.Structure):
    _fields_ = ([("c", C.c_void_p)] + [(n, C.c_uint32) for n in ("d", "heads", "kv_heads", "hd", "rot")] + [("theta", C.c_float)]
                + [(n, C.c_uint32) for n in ("cols", "rows", "keys")] + [(n, C.c_void_p) for n in ("p", "p16", "o16", "k16", "v16")])


class AttnW(C.Structure):
    _fields_ = [("qkv", C.c_void_p), ("out", C.c_void_p)]


class AttnRows(C.Structure):
    _fields_ = [("rows", C.c_uint32), ("seqs", C.c_uint32), ("a16", C.c_void_p), ("amax", C.c_void_p), ("sa", C.c_uint32), ("pos", C.c_void_p),
                ("slot", C.c_void_p), ("table", C.c_void_p), ("table_stride", C.c_uint32), ("out", C.c_void_p)]


@pytest.mark.parametrize("e4m3", [False, True])
def test_layer_attention_prompt_chunks_and_steps(on, mc, pkg, e4m3):
    """The C host side: a batch of prompts at once, the same in two chunks over the cache, and token by token: the three agree with
    the 64-bit form of the whole and so with one another."""
    pkg.build.build_host()
    L = C.CDLL(pkg.build.HOST_LIB)
    L.moe_attn_open.restype = C.c_bool
    L.moe_attn_open.argtypes = [C.POINTER(Attn), C.c_void_p] + [C.c_uint32] * 5 + [C.c_float, C.c_uint32, C.c_uint32]
    L.moe_attn_close.argtypes = [C.POINTER(Attn)]
    L.moe_attn_prompt.argtypes = [C.POINTER(Attn), C.POINTER(mc.Kv), C.POINTER(AttnW), C.POINTER(AttnRows), C.c_void_p, C.c_void_p, C.c_uint32]
    L.moe_attn_step.argtypes = [C.POINTER(Attn), C.POINTER(mc.Kv), C.POINTER(AttnW), C.POINTER(AttnRows), C.c_void_p, C.c_uint32]
    d, h, g, hd, rot, theta, page = 256, 6, 2, 64, 32, 1e4, 16
    gen, lengths = _gen(61), [40, 7, 65]
    seqs, rows = len(lengths), sum(lengths)
    cols = ((h + 2 * g) * hd + 127) // 128 * 128
    x = _f16(gen, rows, d)
    qkv, wo = torch.zeros(cols, d, device="cuda", dtype=torch.float16), _f16(gen, d, h * hd) * 0.05
    qkv[:(h + 2 * g) * hd] = _f16(gen, (h + 2 * g) * hd, d) * 0.06
    per = -(-max(lengths) // page)
    kv = Cache(mc, gen, seqs * per, page, g, hd, e4m3)
    table = torch.randperm(seqs * per, device="cuda", generator=gen).int().view(seqs, per)
    place = torch.cat([torch.arange(n, device="cuda") for n in lengths])
    seq = torch.cat([torch.full((n,), i, device="cuda") for i, n in enumerate(lengths)])
    slot = (table[seq, place // page] * page + place % page).int()
    q, w = Attn(), AttnW(qkv.data_ptr(), wo.data_ptr())
    assert L.moe_attn_open(C.byref(q), on.p, d, h, g, hd, rot, theta, rows, rows) and q.cols == cols

    # the 64-bit form; keys and values as the cache keeps them
    p = (x.double() @ qkv.double().T)[:, :(h + 2 * g) * hd].view(rows, h + 2 * g, hd)
    a = place.double()[:, None] * theta ** (-torch.arange(rot // 2, device="cuda", dtype=torch.float64) / (rot // 2))
    lo, hi, c, s = p[:, :h + g, :rot // 2].clone(), p[:, :h + g, rot // 2:rot].clone(), a.cos()[:, None], a.sin()[:, None]
    p[:, :h + g, :rot // 2], p[:, :h + g, rot // 2:rot] = lo * c - hi * s, hi * c + lo * s
    step = 2.0 ** -4 if e4m3 else 2.0 ** -11   # half a step of what the cache keeps, relative

    def rows_of(idx, out):
        t = {"x": x[idx].contiguous(), "pos": place[idx].int().contiguous(), "slot": slot[idx].contiguous()}
        r = AttnRows(len(idx), seqs, t["x"].data_ptr(), None, NO_SLOT, t["pos"].data_ptr(), t["slot"].data_ptr(), table.data_ptr(), per, out.data_ptr())
        return r, t

    def want(idx, cached):
        out, tol = torch.empty(len(idx), d, device="cuda", dtype=torch.float64), torch.empty(len(idx), d, device="cuda", dtype=torch.float64)
        for n, i in enumerate(idx.tolist()):
            b = i - int(place[i])
            o, mass, size = R.attention(p[i:i + 1, :h], p[b:i + 1, h:h + g], p[b:i + 1, h + g:], hd ** -0.5, i - b)
            out[n] = o.view(-1) @ wo.double().T
            # queries and keys off by half a step of fp16 (and the cache's) move a logit by that of sum |qk|, values theirs, the
            # products' sums 2^-20 of their size; then the kernel's own error, the output's rounding and the second product's
            rel = (step if cached else 2.0 ** -11) + 2.0 ** -11
            e = R.bound(o, mass, size, hd, i - b + 1) + mass * (2 * rel * size[..., None] * 1.1 + rel) + 2.0 ** -18 * mass
            tol[n] = e.view(-1) @ wo.double().abs().T * 1.01 + 1e-5
        return out, tol

    whole = torch.arange(rows, device="cuda")
    out = torch.full((rows, d), 7.0, device="cuda")
    r, keep = rows_of(whole, out)
    cu = _starts(lengths)
    L.moe_attn_prompt(C.byref(q), C.byref(kv.c), C.byref(w), C.byref(r), cu.data_ptr(), None, 0)
    on.flush()
    ref, tol = want(whole, False)
    assert ((out.double() - ref).abs() <= tol).all()

    # two chunks: the second one's keys come back out of the cache
    first = [n // 3 for n in lengths]
    for idx, lq, lk in ((whole[place < torch.tensor(first, device="cuda")[seq]], first, first),
                        (whole[place >= torch.tensor(first, device="cuda")[seq]], [n - f for n, f in zip(lengths, first)], lengths)):
        out = torch.full((len(idx), d), 7.0, device="cuda")
        r, keep = rows_of(idx, out)
        cu_q, cu_k = _starts(lq), _starts(lk)
        L.moe_attn_prompt(C.byref(q), C.byref(kv.c), C.byref(w), C.byref(r), cu_q.data_ptr(), cu_k.data_ptr(), sum(lk))
        on.flush()
        ref, tol = want(idx, True)
        assert ((out.double() - ref).abs() <= tol).all()

    # a token at a time, the last seven of every sequence
    for back in range(7, 0, -1):
        idx = torch.tensor([sum(lengths[:i + 1]) - back for i in range(seqs)], device="cuda")
        length = _u32([n - back + 1 for n in lengths])
        out = torch.full((seqs, d), 7.0, device="cuda")
        r, keep = rows_of(idx, out)
        L.moe_attn_step(C.byref(q), C.byref(kv.c), C.byref(w), C.byref(r), length.data_ptr(), max(lengths))
        on.flush()
        ref, tol = want(idx, True)
        assert ((out.double() - ref).abs() <= tol).all()
    L.moe_attn_close(C.byref(q))
