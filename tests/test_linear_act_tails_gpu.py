"""GPU tier: gelu and its slope far below zero, where they are small but no less exact, relative to their own value."""
import math

import pytest
import torch

import _linear_oracle as oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    from pytorch_distributed_training_amd.ops import hip as hip_ops
    return hip_ops


def every_bf16(low, high, device):
    """All bf16 numbers of [-high, -low]."""
    bits = torch.arange(0x8000, 0xff80, dtype=torch.int32)
    z = (bits << 16).view(torch.float32)
    return z[(z <= -low) & (z >= -high)].to(torch.bfloat16).to(device)


# fp32 arithmetic: exp(-z^2 / 2) has an argument of up to z^2 / 2 log2(e) = 104 at z = -12 with three roundings of 2^-24 each
# on the way, 1.3e-5; approximation and polynomial: below 4e-6
RELATIVE = 2e-5


@pytest.mark.parametrize("rows", [64, None])
def test_gelu_tail(hip, device, rows):
    """Both forward kernels: few rows, tiles."""
    z = every_bf16(0.25, 12.0, device)
    assert z.numel() > 600
    one = torch.ones(1, 1, dtype=torch.bfloat16, device=device)
    for part in z.split(rows or z.numel()):
        y, _ = hip.linear_act_fwd(part[:, None].contiguous(), one, act="gelu")
        want = oracle.act(part.double(), "gelu")
        off = (y[:, 0].double() - want).abs()
        bound = want.abs() * (RELATIVE + oracle.HALF * (1 + RELATIVE))
        assert (off <= bound).all(), (part[off > bound][:5].tolist(), (off / want.abs()).max().item())


def test_slope_tail(hip, device):
    """dbias sums the unrounded slope: here of one row per column."""
    z = every_bf16(0.25, 12.0, device)
    n = z.numel()
    zs = torch.zeros(n, n, dtype=torch.bfloat16, device=device)
    zs.diagonal().copy_(z)
    eye = torch.eye(n, device=device).bfloat16()
    thin = torch.zeros(n, 8, dtype=torch.bfloat16, device=device)
    _, _, db = hip.linear_act_bwd(thin, thin, eye, zs, "gelu", need_da=False)
    zd = z.double()
    tail, density = 0.5 * torch.special.erfc(-zd / math.sqrt(2.0)), torch.exp(-zd * zd / 2) / math.sqrt(2 * math.pi)
    off = (db.double() - (tail + zd * density)).abs()
    bound = RELATIVE * (tail + zd.abs() * density)             # the two parts nearly cancel at z = -0.75
    assert (off <= bound).all(), (z[off > bound][:5].tolist(), (off / bound).max().item())
