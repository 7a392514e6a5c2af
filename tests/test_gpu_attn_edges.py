"""Calls of the attention half that lie at the edge of what is allowed: flags of masked blocks under many short items, refusals with
nothing else to do, values at the end of a type's range, scores far beyond fp32's whole numbers, offsets that leave rows out."""
import ctypes as C

import numpy as np
import pytest
import torch

from . import attn_ref as R
from .test_gpu_attn import NO_SLOT, Attn, AttnRows, AttnW, Cache, _f16, _gen, _refused, _starts, _u32, on  # noqa: F401

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
