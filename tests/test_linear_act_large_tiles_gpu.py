"""GPU tier: the 256-row tiles of the three products, with remainders in rows, columns and reduction."""
import math

import pytest
import torch

import _linear_oracle as oracle

pytestmark = pytest.mark.gpu

SIZES = [(4000, 4001, 4010), (4000, 4008, 4024)]               # (the second needs no copies)
LAYOUTS = [(0, 0), (8, 8), (3, 1)]                             # contiguous, aligned window, unaligned window


@pytest.fixture(scope="module")
def hip():
    from pytorch_distributed_training_amd.ops import hip as hip_ops
    for size in SIZES:                                         # the cost rule may move: these tests are about this kernel
        assert [hip_ops._real.pdt_linear_tile_rows(*size, product) for product in range(3)] == [256] * 3
    return hip_ops


def within(got, want, bound):
    off = (got.double() - want).abs()
    assert (off <= bound).all(), ((off - bound).max().item(), torch.nonzero(~(off <= bound))[:4].tolist())


def padding_is_zero(t, columns):
    assert not t.as_strided((t.shape[0], t.stride(0)), (t.stride(0), 1))[:, columns:].any()


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("wide,skip", LAYOUTS)
@pytest.mark.parametrize("act", ["none", "gelu", "silu"])
def test_forward(hip, device, M, N, K, wide, skip, act):
    gen = torch.Generator().manual_seed(M + N + K)
    a = oracle.rows((M, K), gen, wide=wide, skip=skip, device=device)
    w = oracle.rows((N, K), gen, scale=K ** -0.5, wide=wide, skip=skip, device=device)
    bias = torch.randn(N, generator=gen).to(device)
    res = oracle.rows((M, N), gen, wide=wide, skip=skip, device=device) if act != "none" else None
    y, z = hip.linear_act_fwd(a, w, bias, act, res, save=True)
    want_y, want_z, by, bz = oracle.fwd(a, w, bias, act, res)
    within(y, want_y, by)
    padding_is_zero(y, N)
    assert (z is None) == (act == "none")
    if z is not None:
        within(z, want_z, bz)
        padding_is_zero(z, N)


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("wide,skip", LAYOUTS)
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_backward(hip, device, M, N, K, wide, skip, act):
    gen = torch.Generator().manual_seed(M + N + K)
    a = oracle.rows((M, K), gen, wide=wide, skip=skip, device=device)
    w = oracle.rows((N, K), gen, scale=K ** -0.5, wide=wide, skip=skip, device=device)
    dy = oracle.rows((M, N), gen, wide=wide, skip=skip, device=device)
    z = oracle.rows((M, N), gen, scale=2.0, wide=wide, skip=skip, device=device) if act != "none" else None
    want, bounds = oracle.bwd(a, w, dy, z, act)
    got = hip.linear_act_bwd(a, w, dy, z, act)
    for g, x, b in zip(got, want, bounds):
        within(g, x, b)
    buf = torch.full((N, K + wide), 7.0, device=device)
    dw, db = buf[:, :K], torch.full((N,), 3.0, device=device)
    da, _, _ = hip.linear_act_bwd(a, w, dy, z, act, dw, db)
    assert torch.equal(da, got[0])
    within(dw - 7.0, want[1], bounds[1] + 2.0 ** -21 + 2.0 ** -23 * want[1].abs())
    within(db - 3.0, want[2], bounds[2] + 2.0 ** -21 + 2.0 ** -23 * want[2].abs())
    assert (buf[:, K:] == 7.0).all()


@pytest.mark.parametrize("M,N,K", SIZES)
def test_nan_stays_in_its_row(hip, device, M, N, K):
    gen = torch.Generator().manual_seed(1)
    a, w = oracle.rows((M, K), gen, device=device), oracle.rows((N, K), gen, device=device)
    dy = oracle.rows((M, N), gen, device=device)
    a[M - 1], w[N // 3] = math.nan, math.inf
    y, _ = hip.linear_act_fwd(a, w)
    bad = y.isnan() | y.isinf()
    want = torch.zeros_like(bad)
    want[M - 1], want[:, N // 3] = True, True
    assert torch.equal(bad, want)
    a[M - 1], w[N // 3] = 1.0, 1.0
    dy[M // 2] = math.nan
    da, dw, db = hip.linear_act_bwd(a, w, dy)
    bad = da.isnan()
    assert bad[M // 2].all() and not bad[:M // 2].any() and not bad[M // 2 + 1:].any() and dw.isnan().all() and db.isnan().all()
    dy[M // 2], dy[:, N - 1] = 0.0, math.nan
    w[:, 5] = 0.0
    da, dw, _ = hip.linear_act_bwd(a, w, dy)
    assert da.isnan().all() and dw[N - 1].isnan().all() and not dw[:N - 1].isnan().any()


def test_gradients_are_the_products_of_dz_as_it_is_rounded(hip, device):
    """dz is rounded to bf16 once, and that is all that gradients through an activation lose beside their own rounding: they are
    as far from the products of the rounded dz as those are when they are rounded themselves (2 %: a dz next to a border)."""
    M, N, K = SIZES[1]
    gen = torch.Generator().manual_seed(3)
    a, w = oracle.rows((M, K), gen, device=device), oracle.rows((N, K), gen, scale=K ** -0.5, device=device)
    dy, z = oracle.rows((M, N), gen, device=device), oracle.rows((M, N), gen, device=device)
    da, dw, db = hip.linear_act_bwd(a, w, dy, z, "gelu")
    exact = dy.double() * oracle.slope(z.double(), "gelu")
    dz = exact.to(torch.bfloat16).double()
    for got, want in ((da, dz @ w.double()), (dw, dz.t() @ a.double())):
        off, own = (got.double() - want).norm(), (want.to(torch.bfloat16).double() - want).norm()
        assert off <= 1.02 * own, (off / own).item()
    # dbias has the unrounded ones: a sum of 500 per thread, of 8 and of 125 parts, each addition off by half a step of 2^-23
    assert ((db.double() - exact.sum(0)).abs() <= (4e-6 + 633 * 2.0 ** -24) * exact.abs().sum(0) + 4e-7 * dy.double().abs().sum(0)).all()
