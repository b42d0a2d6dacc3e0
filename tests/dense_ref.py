"""Plain 64-bit formulas of the dense operators and the 8-bit formats, for the tests (torch, CPU or GPU)."""
import math

import torch

EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # half a step, relative
# below the smallest normal number the spacing is fixed (2^-24 in float16): a rounding there is off by up to half of it
LOW = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def act(z, name):
    """act(z), act'(z)"""
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z)), (z > 0).to(z.dtype)
    if name == "gelu":
        cdf = 0.5 * torch.special.erfc(-z * math.sqrt(0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


def two_to(n):
    """2^n in 64 bits from the exponent's bits (library powers may be a bit off)"""
    return ((n.to(torch.int64) + 1023) << 52).view(torch.float64)


def mx8(x):
    """what a matrix reads back as after quantize_mx8, in 64 bits, block by block"""
    top = 15 if x.dtype == torch.float16 else 127
    M, K = x.shape
    pad = (K + 31) // 32 * 32 - K
    b = torch.nn.functional.pad(x.double(), (0, pad)).view(M, -1, 32)
    fin = torch.isfinite(b)
    a = torch.where(fin, b.abs(), torch.zeros_like(b)).amax(2, keepdim=True)
    m, e = torch.frexp(a)                                   # a = m 2^e, m in [0.5, 1)
    E = torch.where(a > 0, e - 9 + (m > 0.875), torch.full_like(e, -126)).clamp(min=-126)
    s = two_to(E)
    lim = torch.where(e - 1 >= top, 240.0, 448.0).to(a)
    v = torch.maximum(torch.minimum(b / s, lim), -lim)
    step = two_to((torch.frexp(v.abs())[1] - 4).clamp(min=-9))
    q = torch.where(fin, torch.round(v / step) * step * s, torch.full_like(v, math.nan))
    return q.view(M, -1)[:, :K], (E + 127).view(M, -1)
