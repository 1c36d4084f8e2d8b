"""CPU tier: the reference linear operators against the 64-bit oracle, differences and autograd, and every refusal."""
import math

import pytest
import torch

import _linear_oracle as oracle
from pytorch_distributed_training_amd.ops import ref

ACTS = ["none", "relu", "gelu", "silu"]


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (5, 7, 3), (16, 33, 20), (0, 4, 5)])
def test_forward_and_backward(act, dtype, M, N, K):
    gen = torch.Generator().manual_seed(M + N + K)
    a, w = oracle.rows((M, K), gen, dtype, wide=3), oracle.rows((N, K), gen, dtype, K ** -0.5)
    bias, res = torch.randn(N, generator=gen), oracle.rows((M, N), gen, dtype, wide=1)
    y, z = ref.linear_act_fwd(a, w, bias, act, res, save=True)
    want_y, want_z, by, bz = oracle.fwd(a, w, bias, act, res)
    assert y.dtype == dtype and ((y.double() - want_y).abs() <= by).all()
    assert (z is None) == (act == "none")
    if z is not None:
        assert ((z.double() - want_z).abs() <= bz).all()
    dy = oracle.rows((M, N), gen, dtype)
    got = ref.linear_act_bwd(a, w, dy, z, act)
    want, bounds = oracle.bwd(a, w, dy, z, act)
    for g, x, b in zip(got, want, bounds):
        assert ((g.double() - x).abs() <= b).all()
    dw, db = torch.ones(N, K), torch.ones(N)
    _, dw2, db2 = ref.linear_act_bwd(a, w, dy, z, act, dw, db, need_da=False)
    assert dw2 is dw and db2 is db and _ is None
    assert torch.allclose(dw - 1, (want[1]).float(), atol=1e-4, rtol=1e-2)


@pytest.mark.parametrize("act", ACTS)
def test_slope_against_differences(act):
    z = torch.tensor([-6.0, -3.0, -1.0, -0.25, 0.3, 0.8, 2.0, 5.0], dtype=torch.float64)
    h = 1e-5
    moved = (oracle.act(z + h, act) - oracle.act(z - h, act)) / (2 * h)
    assert (oracle.slope(z, act) - moved).abs().max() < 1e-9      # h^2 / 6 f''' (below 2) + 1e-16 / h
    if act != "none":
        assert (ref._act_slope(z, act) - oracle.slope(z, act)).abs().max() < 1e-12
        assert (ref._act_value(z, act) - oracle.act(z, act)).abs().max() < 1e-12


def test_backward_is_the_gradient_of_forward():
    gen = torch.Generator().manual_seed(3)
    a, w, b = (torch.randn(*s, generator=gen).requires_grad_(True) for s in ((6, 5), (4, 5), (4,)))
    dy = torch.randn(6, 4, generator=gen)
    for act in ACTS:
        y, z = ref.linear_act_fwd(a, w, b, act, save=True)
        want = torch.autograd.grad(y, (a, w, b), dy)
        with torch.no_grad():
            got = ref.linear_act_bwd(a.detach(), w.detach(), dy, None if z is None else z.detach(), act)
        for g, x in zip(got, want):
            assert torch.allclose(g, x, atol=1e-5)


@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
def test_infinities_and_nan(act):
    z = torch.tensor([-math.inf, math.inf, math.nan])
    v, s = ref._act_value(z, act), ref._act_slope(z, act)
    assert v[0] == 0 and v[1] == math.inf and v[2].isnan() and s[0] == 0 and s[1] == 1 and s[2].isnan()


def test_refusals():
    a, w, b, r = torch.randn(6, 5), torch.randn(4, 5), torch.randn(4), torch.randn(6, 4)

    def fwd(error, **other):
        args = dict(a=a, w=w, bias=b, act="relu", residual=r)
        args.update(other)
        with pytest.raises(error):
            ref.linear_act_fwd(**args)

    def bwd(error, **other):
        args = dict(a=a, w=w, dy=r, z=r, act="relu")
        args.update(other)
        with pytest.raises(error):
            ref.linear_act_bwd(**args)

    fwd(ValueError, act="tanh")
    fwd(ValueError, w=torch.randn(4, 6))
    fwd(ValueError, a=torch.randn(6))
    fwd(ValueError, a=torch.randn(6, 0), w=torch.randn(4, 0))
    fwd(ValueError, w=torch.randn(0, 5), bias=torch.randn(0), residual=torch.randn(6, 0))
    fwd(ValueError, a=torch.randn(5, 6).t())
    fwd(ValueError, w=torch.randn(5, 4).t())
    fwd(TypeError, a=a.double())
    fwd(TypeError, w=w.half())
    fwd(TypeError, bias=b.bfloat16())
    fwd(ValueError, bias=torch.randn(5))
    fwd(ValueError, bias=torch.randn(8)[::2])
    fwd(ValueError, residual=torch.randn(4))
    fwd(ValueError, residual=torch.randn(4, 6).t())
    bwd(ValueError, z=None)
    bwd(ValueError, dy=torch.randn(6, 5))
    bwd(ValueError, z=torch.randn(5, 4))
    bwd(ValueError, z=torch.randn(4, 6).t())
    bwd(TypeError, dw=torch.zeros(4, 5, dtype=torch.bfloat16))
    bwd(ValueError, dw=torch.zeros(5, 4))
    bwd(ValueError, dw=torch.zeros(1, 5).expand(4, 5))
    bwd(ValueError, dbias=torch.zeros(3))
    bwd(TypeError, dbias=torch.zeros(4).double())


def test_widths_beyond_32_bit_offsets_are_refused():
    wide, one = torch.zeros(1, ref.MAX_WIDTH + 1), torch.zeros(1, 1)
    with pytest.raises(ValueError):
        ref.linear_act_fwd(wide, wide)
    with pytest.raises(ValueError):
        ref.linear_act_fwd(one, wide.t().contiguous())
    with pytest.raises(ValueError):
        ref.linear_act_bwd(wide, wide, one)
    y, _ = ref.linear_act_fwd(wide[:, 1:], wide[:, 1:])
    assert y.shape == (1, 1)
