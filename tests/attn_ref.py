"""Plain 64-bit forms of the attention calls, and what their kernels may be off by."""
import math

import torch


def attention(q, k, v, scale, offset):
    """q [m, H, D], k and v [n, G, D] in float64; query i sees keys 0 .. i + offset.  Returns the output and, per row and
    head, what one part in one of the weights and logits is worth: sum of p |v|, and the largest sum of |q k| scale."""
    h, g = q.shape[1], k.shape[1]
    seen = (torch.arange(k.shape[0], device=q.device)[None] <= torch.arange(q.shape[0], device=q.device)[:, None] + offset)
    out, mass, size = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=q.dtype, device=q.device)
    for a in range(h):
        b = a // (h // g)
        x = (q[:, a] @ k[:, b].T * scale).masked_fill(~seen, -math.inf)
        top = x.amax(-1, keepdim=True) if k.shape[0] else torch.full((q.shape[0], 1), -math.inf, dtype=q.dtype, device=q.device)
        p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
        p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
        vis = seen.any(0)
        out[:, a] = p[:, vis] @ v[vis, b]
        mass[:, a] = p[:, vis] @ v[vis, b].abs()
        if k.shape[0]:
            size[:, a] = (q[:, a].abs() @ k[:, b].abs().T).masked_fill(~seen, 0.0).amax(-1) * scale
    return out, mass, size


def bound(out, mass, size, d, keys):
    """fp16 output: half a step of the value (2^-11, subnormals 2^-25).  Weights round to fp16: 2^-11 of sum p|v|, and below
    2^-14 of their shifted range absolutely: 2^-25 / 2^4 of the largest weight for every key.  Logits: d fp32 sums, at most
    2^-23 of sum |qk| each, some steps of the exponent's argument (three more of the logit's size) and of exp2 itself (2^-21).
    A weight's relative error enters numerator and sum."""
    logit = (d + 3) * 2.0 ** -23 * size[..., None] + 2.0 ** -20
    return 2.0 ** -11 * out.abs() + 2.0 ** -25 + mass * (2.0 ** -11 + 2.0 * logit) * 1.01 + keys * 2.0 ** -29 * mass.amax(-1, keepdim=True)


def check(got, out, mass, size, d, keys):
    assert torch.isfinite(got).all()
    far = (got.double() - out).abs() / bound(out, mass, size, d, keys)
    assert far.max() <= 1.0, f"{far.max():.3f} of the bound at {far.flatten().argmax()}"


def e4m3(x):
    """Codes of x [..., D] (fp16) and their power-of-two scales."""
    f = x.float()
    top = torch.where(torch.isnan(f), torch.zeros_like(f), f).abs().amax(-1).clamp(max=65504.0)
    m, e = torch.frexp(top)
    scale = torch.where(top == 0, 1.0, torch.ldexp(torch.ones_like(m), torch.where(m <= 0.875, e - 9, e - 8)))
    y = (f / scale[..., None]).clamp(-448.0, 448.0)   # clamp passes NaN on
    return y.to(torch.float8_e4m3fn), scale
