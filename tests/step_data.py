"""The definitions in 64 bits of what a serving step does around its paged cache: microscaled 4-bit floating point, the norm and
rotation of heads, log probabilities. On the CPU."""
from __future__ import annotations

import math

import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a step, relative
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}  # half the smallest step
GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def quantised(x):
    """(codes [rows, cols], one to an element, scale bytes [rows, cols / 32]) of x, block by block from the definition."""
    rows, cols = x.shape
    d = x.double().view(rows, cols // 32, 32)
    finite = torch.isfinite(d).all(-1)
    d = torch.where(finite[..., None], d, 0.0)
    most = d.abs().amax(-1)
    field = torch.where(most >= 2.0 ** -126, torch.frexp(most).exponent - 1 + 127, 0)   # fp32's exponent field
    byte = (field - 2).clamp(min=0)
    a = (d * torch.ldexp(torch.ones_like(most), 127 - byte)[..., None]).abs()
    grid = torch.tensor(GRID, dtype=torch.float64)
    gap = (a[..., None] - grid).abs()
    # the nearest; of two equally near the even code, which the second key puts first
    code = (gap + 1e-9 * (torch.arange(8) % 2)).argmin(-1)
    code = code + 8 * (torch.signbit(x.view(d.shape)) & finite[..., None])
    return code.view(rows, cols), torch.where(finite, byte, 255)


def packed(code):
    return (code[:, 0::2] | code[:, 1::2] << 4).to(torch.uint8)


def values_of(code, byte):
    grid = torch.tensor(GRID + [-g for g in GRID], dtype=torch.float64)
    scale = torch.where(byte == 255, math.nan, torch.ldexp(torch.ones(byte.shape, dtype=torch.float64), byte.int() - 127))
    return grid[code] * scale.repeat_interleave(32, 1)


def random_codes(g, rows, cols, low=127, spread=2):
    code = torch.randint(0, 16, (rows, cols), generator=g)
    return code, low + torch.randint(0, spread, (rows, cols // 32), generator=g)


def table(positions, rot, theta=10000.0):
    half = rot // 2
    a = torch.arange(positions, dtype=torch.float64)[:, None] * theta ** (-torch.arange(half, dtype=torch.float64) / half)
    return torch.cat([a.cos(), a.sin()], 1).float()


def rotated(x, gamma, tab, pos, hd, eps):
    """(y, the error that fp32 steps allow before the rounding) of rows x at positions pos: [rows, heads, hd] in 64 bits. A
    term is x / sqrt(.) gamma cos: the sum of squares (hd fp32 steps at most, in a square root), and ten steps more."""
    half = tab.shape[1] // 2
    u = x.double().view(len(pos), -1, hd)
    if gamma is not None:
        u = u / torch.sqrt(u.square().mean(-1, keepdim=True) + eps) * gamma.double()
    t = tab[pos].double()[:, None]
    c, s = t[..., :half], t[..., half:]
    a, b, rest = u[..., :half], u[..., half:2 * half], u[..., 2 * half:]
    y = torch.cat([a * c - b * s, b * c + a * s, rest], -1)
    size = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs(), rest.abs()], -1)
    return y, (hd / 2 + 10) * 2.0 ** -24 * size


def logprobs(x, tokens, top):
    """(logprobs, entropy, top values, top ids) of one row, in 64 bits; tokens outside: -infinity."""
    x = x.double()
    vocab = x.numel()
    if (x == -math.inf).all():
        lp, h = torch.full((vocab,), -math.inf, dtype=torch.float64), 0.0
    else:
        lp = torch.log_softmax(x, 0)
        p = lp.exp()
        h = float(-torch.where(p > 0, p * lp, p).sum())
    # NaN above all, then by value, then by place
    order = sorted(range(vocab), key=lambda i: (not math.isnan(x[i]), 0.0 if math.isnan(x[i]) else -float(x[i]), i))[:top]
    given = [float(lp[t]) if 0 <= t < vocab else -math.inf for t in tokens]
    return given, h, [float(lp[i]) for i in order], order
