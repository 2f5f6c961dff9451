"""The AdamW step and its float8 states from their definition, in 64 bits (torch on the device of its arguments)."""
from __future__ import annotations

import torch

BLOCK = 256
FORMATS = {"m": (7, 20, None, -6, 3, torch.float8_e4m3fn), "v": (14, 21, 2.0 ** -16, -14, 2, torch.float8_e5m2)}
# largest exponent a block is scaled to, mantissa bits cut off, least value, exponent of the least normal, mantissa bits kept, type


def moments(m, v, g, betas):
    """(m', v') and the magnitudes their roundings are relative to."""
    a, b = m * betas[0], g * (1.0 - betas[0])
    c, d = v * betas[1], g * g * (1.0 - betas[1])
    return a + b, c + d, a.abs() + b.abs(), c + d


def param(p, m, v, t, lr, betas, eps, wd):
    """(p', the update that was taken off)."""
    upd = lr / (1.0 - betas[0] ** t) * m / (v.sqrt() / (1.0 - betas[1] ** t) ** 0.5 + eps)
    return p * (1.0 - lr * wd) - upd, upd


def param_bound(p, upd, dtype):
    """p', rounded to dtype: half a step, three fp32 roundings of p', and of the update 16 (moments 6, half of the 4 of v, root 2,
    product and sum in the denominator 2, quotient 3, factor 1)."""
    f = torch.finfo(dtype)
    tiny = 0.0 if dtype == torch.float32 else f.smallest_normal * f.eps / 2
    return (f.eps / 2 * (dtype != torch.float32) + 3 * 2.0 ** -24) * p.abs() + 16 * 2.0 ** -24 * upd.abs() * 1.02 + tiny + 1e-44


def _mix(x):
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def random_bits(n, t, device="cpu"):
    e = torch.arange(n, dtype=torch.int64, device=device)
    h = _mix(((e >> 3) + _mix(torch.tensor(t, dtype=torch.int64, device=device))) & 0xFFFFFFFF)
    return (h * ((0x9E3779B1 * (2 * (e & 7) + 1)) & 0xFFFFFFFF)) & 0xFFFFFFFF


def blocks(x, fill=0.0):
    x = x.reshape(-1)
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK), value=fill).view(-1, BLOCK)


def encode(x, which, t):
    """(values the codes stand for before the scale, scales as fp32) of an fp32 tensor, blockwise, at step count t: y = x / scale
    becomes sign(y) floor(|y| / u + r / 2^drop) u, u the format's spacing at y, that of its subnormals below the least normal
    number.  In 64 bits from the definition; every operation is exact."""
    top, drop, least, _, _, dtype = FORMATS[which]
    n = x.numel()
    h = random_bits(n, t, x.device)
    r = (h & 0xFFFFF) if which == "m" else h >> 11
    b = blocks(x).double()
    a = b.abs().amax(1, keepdim=True)
    e = (torch.frexp(a)[1] - 1 - top).clamp(-126, 127)
    scale = torch.where(a > 0, torch.ldexp(torch.ones_like(a), e), torch.full_like(a, 2.0 ** -126))
    y = b / scale
    if least is not None:
        y = torch.where(a > 0, y.clamp(min=least), y)
    u = spacing(y, which)
    q = torch.floor(y.abs() / u + blocks(r).double() / 2.0 ** drop) * u * torch.sign(y)
    return q.to(dtype).reshape(-1)[:n].view(x.shape), scale[:, 0].float()


def decode(codes, scale):
    n = codes.numel()
    return (blocks(codes.float()) * scale.float()[:, None]).reshape(-1)[:n].view(codes.shape)


def spacing(y, which):
    """Distance of neighbouring codes at y (the scaled value)."""
    _, _, _, low, bits, _ = FORMATS[which]
    e = (torch.frexp(y.abs())[1] - 1).clamp(min=low)
    return torch.ldexp(torch.ones_like(y), e - bits)
