"""4-bit microscaled floating point in 64 bits, from the format's definition, and limits for sums of its products."""

import math

import torch

STEPS = 2.0 ** -23          # what a float32 sum may lose a time: one unit of its last place


def scales_of(x):
    """The blocks of 32 of the last axis (filled up with zeros) and each block's scale; NaN where a block is no number."""
    x = x.double()
    short = -x.shape[-1] % 32
    x = torch.cat([x, x.new_zeros((*x.shape[:-1], short))], -1).unflatten(-1, (-1, 32))
    top = x.abs().max(-1).values
    scale = torch.empty_like(top)
    flat, out = top.flatten(), scale.view(-1)
    for i, m in enumerate(flat.tolist()):
        if not math.isfinite(m):
            out[i] = math.nan
        elif m == 0.0:
            out[i] = 2.0 ** -127
        else:
            out[i] = 2.0 ** max(math.frexp(m)[1] - 3, -127)      # frexp's fraction is at least 1/2
    return x, scale


def nearest(x):
    """The nearest 4-bit values: quarters' steps below 2 scales, halves up to 4, wholes up to 6."""
    k = x.shape[-1]
    blocks, scale = scales_of(x)
    v = blocks / scale[..., None]
    size = v.abs()
    step = torch.full_like(v, 0.5)
    step[size >= 2] = 1.0
    step[size >= 4] = 2.0
    v = (torch.round(v / step) * step).clamp(-6.0, 6.0)          # round: ties to even, which is the even code
    return (v * scale[..., None]).flatten(-2)[..., :k]


def product(a, w):
    """a w^T and the most that float32 sums of it may be off: every instruction of 64 products and every rounding
    behind them loses at most two units of the last place of what has been added up."""
    want = a @ w.transpose(-1, -2)
    size = a.abs() @ w.abs().transpose(-1, -2)
    return want, size * STEPS * 2 * (-(-a.shape[-1] // 64) + 2)


def unit(gate, up, off_gate, off_up, alpha=1.0, limit=0.0):
    """The gated unit, and the most it may be off: the slope of g * sigmoid(alpha g) is at most 1.1, the exponential's and
    the quotient's roundings cost a few units of float32's last place."""
    if limit > 0:
        gate, up = gate.clamp(max=limit), up.clamp(-limit, limit) + 1
        s = gate * torch.sigmoid(alpha * gate)
    else:
        s = gate * torch.sigmoid(gate)
    off = 1.1 * up.abs() * off_gate + s.abs() * off_up + 1.1 * off_gate * off_up
    return s * up, off + (s * up).abs() * 16 * STEPS


def rounding(dtype, want):
    """Half a step of the type, and half its smallest one."""
    info = torch.finfo(dtype)
    return want.abs() * info.eps / 2 + info.smallest_normal * info.eps
