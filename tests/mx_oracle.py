"""The block-scaled operators in 64 bits on the CPU, from their definitions (OCP Microscaling v1.0 element formats)."""
import torch

#: largest exponent, smallest exponent, digits behind the point, largest value
FORMATS = {"mxfp8": (8, -6, 3, 448.0), "mxfp4": (2, 0, 1, 6.0)}


def power(e):
    """2^e in float64, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def scale_exponents(x, fmt):
    """The exponents of the blocks' scales of float64 x [R, K] -> int64 [R, blocks]; a block with NaN or infinity has 128."""
    r, k = x.shape
    b = torch.zeros(r, -(-k // 32) * 32, dtype=torch.float64)
    b[:, :k] = x
    top = b.reshape(r, -1, 32).abs().amax(dim=2)
    e = (torch.frexp(top)[1] - 1 - FORMATS[fmt][0]).clamp(min=-127).long()
    e[top == 0] = -127
    e[~torch.isfinite(b.reshape(r, -1, 32)).all(dim=2)] = 128
    return e


def values(x, fmt, exponents=None):
    """The values that the block-scaled form of float64 x [R, K] stands for."""
    emax, emin, digits, most = FORMATS[fmt]
    e = scale_exponents(x, fmt) if exponents is None else exponents
    e = e.repeat_interleave(32, dim=1)[:, :x.shape[1]]
    scale = power(e.clamp(max=127))
    v = x / scale
    v = torch.where(torch.isfinite(v), v, 0.0)
    step = power((torch.frexp(v)[1] - 1).clamp(min=emin) - digits)
    v = (torch.round(v / step) * step).clamp(-most, most) * scale
    return torch.where(e == 128, torch.nan, v)


def held_within(got, want, rel, fmt):
    """Whether `got` is the block-scaled form of values that are each within `rel` (relative, in whole blocks) of float64
    `want`: between the forms of want (1 - rel) and want (1 + rel).  A block whose largest value lies within `rel` of a power
    of two may have either scale: there an element may be one step of the larger scale off."""
    lo, hi = want * (1 - rel), want * (1 + rel)
    elo, ehi = scale_exponents(lo, fmt), scale_exponents(hi, fmt)
    a, b = values(lo, fmt), values(hi, fmt)
    inside = (got >= torch.minimum(a, b)) & (got <= torch.maximum(a, b))
    either = (elo != ehi).repeat_interleave(32, dim=1)[:, :want.shape[1]]
    step = power(ehi.clamp(max=127)).repeat_interleave(32, dim=1)[:, :want.shape[1]] * 2.0 ** (FORMATS[fmt][0] - FORMATS[fmt][2])
    near = (got - want).abs() <= step
    both_nan = torch.isnan(got) & torch.isnan(a)
    return bool((inside | (either & near) | both_nan).all())


def gate(b, act):
    # (ndtr is 1 + erf, which cancels on the left)
    return b * torch.special.erfc(b * -0.5 ** 0.5) * 0.5 if act == "gelu" else b * torch.sigmoid(b)


def rmsnorm(x, gamma, eps):
    return x / torch.sqrt((x * x).mean(dim=-1, keepdim=True) + eps) * gamma
