"""64-bit oracle and error bounds of the linear operators with activation and residual."""
import math

import torch


def act(z, name):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * torch.special.erfc(-z / math.sqrt(2.0)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s + z * s * (1 - s)
    return torch.ones_like(z)


HALF = 2.0 ** -8                   # half a step of bf16, relative


def sum_bound(x, y, terms):
    """Error of an fp32 product x @ y: a running sum of one addition per 32 terms, each off by at most 2^-23 of what the
    absolute values sum to, and 32-term sums inside an instruction."""
    return (terms / 32 + 32) * 2.0 ** -23 * (x.abs() @ y.abs())


def fwd(a, w, bias, name, residual):
    """(y, z, bound on y, bound on z)"""
    a, w = a.double(), w.double()
    z = a @ w.t()
    dz = sum_bound(a, w.t(), a.shape[1])
    if bias is not None:
        z = z + bias.double()
        dz = dz + 2.0 ** -23 * (z.abs() + bias.double().abs())
    y = act(z, name)
    # no activation here is steeper than 1.13; their own fp32 evaluation: 2e-7 |z| (Abramowitz-Stegun's Phi), 1e-6 relative
    dy = 1.13 * dz + (2e-7 * z.abs() + 1e-6 * y.abs() if name in ("gelu", "silu") else 0.0)
    if residual is not None:
        y = y + residual.double()
        dy = dy + 2.0 ** -23 * y.abs()
    return y, z, dy * 1.01 + HALF * y.abs(), dz * 1.01 + HALF * z.abs()


def bwd(a, w, dy, z, name):
    """(da, dw, dbias, their bounds); the products' operand dz is rounded to bf16 where there is an activation"""
    a, w, g = a.double(), w.double(), dy.double()
    off = torch.zeros_like(g)
    if name != "none":
        s = slope(z.double(), name)
        off = g.abs() * (4e-7 + 2e-6 * s.abs())
        g = g * s
    rounded = off + (HALF * 1.01 * g.abs() if name != "none" else 0.0)
    da, dw, db = g @ w, g.t() @ a, g.sum(0)
    b_da = rounded @ w.abs() + sum_bound(g, w, g.shape[1]) * 1.01
    b_dw = rounded.t() @ a.abs() + sum_bound(g.t(), a, g.shape[0]) * 1.01
    b_db = off.sum(0) + g.shape[0] * 2.0 ** -24 * g.abs().sum(0)
    return (da, dw, db), (b_da + HALF * (da.abs() + b_da), b_dw + HALF * (dw.abs() + b_dw), b_db + 2.0 ** -24 * db.abs())


def rows(shape, gen, dtype=torch.bfloat16, scale=1.0, wide=0, skip=0, device="cpu"):
    """A random matrix; ``wide`` / ``skip``: a window of a wider one that starts ``skip`` columns in (NaN around it)."""
    x = (torch.randn(*shape, generator=gen) * scale).to(dtype)
    if wide or skip:
        big = torch.full((shape[0], shape[1] + wide + skip), math.nan, dtype=dtype)
        big[:, skip:skip + shape[1]] = x
        return big.to(device)[:, skip:skip + shape[1]]
    return x.to(device)
