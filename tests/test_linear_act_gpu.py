"""GPU tier: linear_act_fwd / linear_act_bwd against the 64-bit oracle, and the head with the distillation loss."""
import math

import pytest
import torch

import _distill_oracle
import _linear_oracle as oracle
from pytorch_distributed_training_amd.engine.graphs import ListProgram

pytestmark = pytest.mark.gpu

ACTS = ["none", "relu", "gelu", "silu"]
SIZES = [(1, 1, 1), (1, 1000, 2048), (3, 17, 33), (16, 64, 64), (17, 100, 40), (31, 130, 1021), (33, 10, 8), (33, 1000, 2048),
         (50, 70, 300), (65, 129, 72), (100, 64, 7), (128, 128, 64), (200, 300, 1000), (257, 513, 200), (333, 777, 1021),
         (1000, 1000, 512), (3900, 4001, 72)]


@pytest.fixture(scope="module")
def hip():
    from pytorch_distributed_training_amd.ops import hip as hip_ops
    return hip_ops


def within(got, want, bound):
    off = (got.double() - want).abs()
    assert (off <= bound).all(), ((off - bound).max().item(), torch.nonzero(~(off <= bound))[:4].tolist())


def padding_is_zero(t, columns):
    assert t.stride(0) % 64 == 0
    assert not t.as_strided((t.shape[0], t.stride(0)), (t.stride(0), 1))[:, columns:].any()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,N,K", SIZES)
def test_forward(hip, device, act, M, N, K):
    gen = torch.Generator().manual_seed(M + N + K)
    for wide, skip in ((0, 0), (8, 8), (3, 1)):                # contiguous, aligned window, unaligned window
        a = oracle.rows((M, K), gen, wide=wide, skip=skip, device=device)
        w = oracle.rows((N, K), gen, scale=K ** -0.5, wide=wide, skip=skip, device=device)
        bias = torch.randn(N, generator=gen).to(device) if wide != 8 else None
        res = oracle.rows((M, N), gen, wide=wide, skip=skip, device=device) if wide else None
        y, z = hip.linear_act_fwd(a, w, bias, act, res, save=wide != 3)
        want_y, want_z, by, bz = oracle.fwd(a, w, bias, act, res)
        assert y.shape == (M, N) and y.dtype == torch.bfloat16
        within(y, want_y, by)
        padding_is_zero(y, N)
        assert (z is not None) == (act != "none" and wide != 3)
        if z is not None:
            within(z, want_z, bz)
            padding_is_zero(z, N)


@pytest.mark.parametrize("M", [1, 5, 16, 17, 32, 33, 64])
def test_few_rows_of_many_lengths(hip, device, M):
    """Waves with no, one, an odd number and a partial turn of K."""
    gen = torch.Generator().manual_seed(M)
    for K in (8, 31, 32, 40, 127, 128, 256, 288, 1024, 1056, 1216, 2040, 2176, 3200, 4608):
        for N in (10, 100, 300):
            a, w = oracle.rows((M, K), gen, device=device), oracle.rows((N, K), gen, scale=K ** -0.5, device=device)
            y, _ = hip.linear_act_fwd(a, w)
            want, _, bound, _ = oracle.fwd(a, w, None, "none", None)
            within(y, want, bound)


@pytest.mark.parametrize("M,N,K", [(64, 30, 4000), (2000, 40, 60), (40, 3000, 50), (700, 2100, 1900), (2200, 2304, 2100), (60, 5000, 5000), (4096, 4096, 4096)])
def test_gradients_in_one_launch_and_apart(hip, device, M, N, K):
    gen = torch.Generator().manual_seed(N)
    a, w = oracle.rows((M, K), gen, device=device), oracle.rows((N, K), gen, scale=K ** -0.5, device=device)
    dy = oracle.rows((M, N), gen, device=device)
    want, bounds = oracle.bwd(a, w, dy, None, "none")
    for need_da in (True, False):
        got = hip.linear_act_bwd(a, w, dy, need_da=need_da)
        assert (got[0] is None) == (not need_da)
        for g, x, b in zip(got, want, bounds):
            if g is not None:
                within(g, x, b)
        buf, vec = torch.full((N, K), 7.0, device=device), torch.full((N,), 3.0, device=device)
        hip.linear_act_bwd(a, w, dy, dw=buf, dbias=vec, need_da=need_da)
        within(buf - 7.0, want[1], bounds[1] + 2.0 ** -21 + 2.0 ** -23 * want[1].abs())
        within(vec - 3.0, want[2], bounds[2] + 2.0 ** -22 + 2.0 ** -23 * want[2].abs())


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,N,K", SIZES)
def test_backward(hip, device, act, M, N, K):
    gen = torch.Generator().manual_seed(M + N + K)
    for wide, skip in ((0, 0), (8, 8), (3, 1)):
        a = oracle.rows((M, K), gen, wide=wide, skip=skip, device=device)
        w = oracle.rows((N, K), gen, scale=K ** -0.5, wide=wide, skip=skip, device=device)
        dy = oracle.rows((M, N), gen, wide=wide, skip=skip, device=device)
        z = oracle.rows((M, N), gen, scale=2.0, wide=wide, skip=skip, device=device) if act != "none" else None
        got = hip.linear_act_bwd(a, w, dy, z, act)
        want, bounds = oracle.bwd(a, w, dy, z, act)
        assert [g.dtype for g in got] == [torch.bfloat16, torch.bfloat16, torch.float32]
        for g, x, b in zip(got, want, bounds):
            assert g.shape == x.shape
            within(g, x, b)
        # gradient buffers: added to, and nothing around them touched
        buf = torch.full((N, K + wide), 7.0, device=device)
        dw, db = buf[:, :K], torch.full((N,), 3.0, device=device)
        da, dw2, db2 = hip.linear_act_bwd(a, w, dy, z, act, dw, db, need_da=False)
        assert da is None and dw2 is dw and db2 is db
        within(dw - 7.0, want[1], bounds[1] + 2.0 ** -21 + 2.0 ** -23 * want[1].abs())
        within(db - 3.0, want[2], bounds[2] + 2.0 ** -21 + 2.0 ** -23 * want[2].abs())
        assert (buf[:, K:] == 7.0).all()


@pytest.mark.parametrize("M,N,K", [(2, 40, 64), (40, 70, 72), (300, 200, 136), (300, 203, 131), (4000, 4100, 72)])
def test_nan_stays_in_its_row(hip, device, M, N, K):
    """A row of a (or w) that is NaN reaches its own row (column) of the product only: nothing read past the end of a row
    takes part, in any of the three products."""
    gen = torch.Generator().manual_seed(1)
    a, w = oracle.rows((M, K), gen, device=device), oracle.rows((N, K), gen, device=device)
    a[M // 2] = math.nan
    w[N // 3] = math.inf
    y, _ = hip.linear_act_fwd(a, w)
    bad = y.isnan() | y.isinf()
    want = torch.zeros_like(bad)
    want[M // 2], want[:, N // 3] = True, True
    assert torch.equal(bad, want)
    a, w = oracle.rows((M, K), gen, device=device), oracle.rows((N, K), gen, device=device)
    dy = oracle.rows((M, N), gen, device=device)
    dy[M - 1] = math.nan
    a[0, K - 1] = math.nan
    da, dw, db = hip.linear_act_bwd(a, w, dy)
    assert da[M - 1].isnan().all() and not da[:M - 1].isnan().any()
    assert dw.isnan().all() and db.isnan().all()
    dy[M - 1] = 0.0
    _, dw, _ = hip.linear_act_bwd(a, w, dy)
    assert dw[:, K - 1].isnan().all() and not dw[:, :K - 1].isnan().any()


def test_activations_at_the_ends(hip, device):
    z = torch.tensor([-math.inf, -3e38, -50.0, -9.0, -1e-30, -0.0, 0.0, 1e-30, 9.0, 50.0, 3e38, math.inf, math.nan],
                     device=device).bfloat16()
    one = torch.ones(1, 1, dtype=torch.bfloat16, device=device)
    a = z[:, None].contiguous()
    from pytorch_distributed_training_amd.ops import ref
    for act in ("relu", "gelu", "silu"):
        y, _ = hip.linear_act_fwd(a, one, act=act)
        want = ref._act_value(z.double(), act)
        assert torch.allclose(y[:, 0].double(), want, rtol=2.0 ** -8 * 1.01, atol=1e-9, equal_nan=True), act
        _, _, db = hip.linear_act_bwd(a[:1], one, one, a[3:4], act)
        assert abs(float(db) - float(ref._act_slope(z[3:4].double(), act))) < 1e-6
        dy = torch.eye(13, device=device).bfloat16()
        zs = torch.zeros(13, 13, dtype=torch.bfloat16, device=device)
        zs.diagonal().copy_(z)
        w = torch.zeros(13, 13, dtype=torch.bfloat16, device=device)
        _, _, db = hip.linear_act_bwd(torch.zeros_like(w), w, dy, zs, act)
        want = ref._act_slope(z.double(), act)
        assert torch.allclose(db.double(), want, rtol=1e-5, atol=1e-6, equal_nan=True), act


def test_no_rows(hip, device):
    a, w = torch.zeros(0, 24, dtype=torch.bfloat16, device=device), torch.ones(10, 24, dtype=torch.bfloat16, device=device)
    y, z = hip.linear_act_fwd(a, w, act="relu", save=True)
    assert y.shape == (0, 10) and z.shape == (0, 10)
    da, dw, db = hip.linear_act_bwd(a, w, y, z, "relu")
    assert da.shape == (0, 24) and not dw.any() and not db.any() and dw.shape == (10, 24)
    buf, vec = torch.ones(10, 24, device=device), torch.ones(10, device=device)
    hip.linear_act_bwd(a, w, y, z, "relu", buf, vec)
    assert (buf == 1).all() and (vec == 1).all()


def test_single_rows_whose_stride_says_nothing(hip, device):
    """[1, K] views may have any stride between their (no) rows."""
    gen = torch.Generator().manual_seed(8)
    K, N = 72, 40
    lone = [oracle.rows((1, n), gen, device=device).as_strided((1, n), (s, 1)) for n, s in ((K, 1), (N, 3), (K, 0), (1, 5))]
    a, dy, w1, dy1 = lone
    w = oracle.rows((N, K), gen, device=device)
    assert torch.equal(hip.linear_act_fwd(a, w)[0], hip.linear_act_fwd(a.clone().reshape(1, K), w)[0])
    for got, want in zip(hip.linear_act_bwd(a, w, dy), hip.linear_act_bwd(a.reshape(K).clone()[None], w, dy.reshape(N).clone()[None])):
        assert torch.equal(got, want)
    buf = torch.ones(K, device=device).as_strided((1, K), (1, 1))
    da, dw, db = hip.linear_act_bwd(a, w1, dy1, dw=buf)
    assert dw is buf and torch.allclose(buf.double(), 1 + dy1.double() * a.double(), rtol=1e-6)
    assert torch.allclose(da.double(), dy1.double() * w1.double(), rtol=2.0 ** -8) and float(db) == float(dy1)


def test_beyond_two_gigabytes(hip, device):
    """Offsets of operands and results pass 32 bits: the last rows against the same rows alone."""
    gen = torch.Generator().manual_seed(2)
    M, N, K = 140000, 16384, 64
    a = torch.randn(M, K, device=device).bfloat16()
    w, res = oracle.rows((N, K), gen, device=device), torch.zeros(1, N, dtype=torch.bfloat16, device=device).expand(M, N)
    y, _ = hip.linear_act_fwd(a, w, residual=res)
    small, _ = hip.linear_act_fwd(a[-300:].clone(), w)
    assert torch.equal(y[-300:], small)
    da, dw, db = hip.linear_act_bwd(a, w, y)
    want, _, _ = hip.linear_act_bwd(a[-300:].clone(), w, small)
    assert (da[-300:].float() - want.float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()
    del y, da
    big = torch.zeros(1100, 1 << 21, dtype=torch.bfloat16, device=device)
    big[:, :K] = a[:1100]
    y, _ = hip.linear_act_fwd(big[:, :K], w[:500])
    small, _ = hip.linear_act_fwd(a[:1100], w[:500])
    assert torch.equal(y, small)
    _, dw, _ = hip.linear_act_bwd(big[:, :K], w[:500], small)
    _, want, _ = hip.linear_act_bwd(a[:1100].contiguous(), w[:500], small)
    assert torch.equal(dw, want)


def test_results_repeat_and_inputs_stay(hip, device):
    gen = torch.Generator().manual_seed(4)
    a, w = oracle.rows((700, 512), gen, device=device), oracle.rows((300, 512), gen, device=device)
    dy, z = oracle.rows((700, 300), gen, device=device), oracle.rows((700, 300), gen, device=device)
    kept = [t.clone() for t in (a, w, dy, z)]
    first = hip.linear_act_fwd(a, w, None, "silu", dy, True) + hip.linear_act_bwd(a, w, dy, z, "silu")
    for _ in range(3):
        again = hip.linear_act_fwd(a, w, None, "silu", dy, True) + hip.linear_act_bwd(a, w, dy, z, "silu")
        assert all(torch.equal(x, y) for x, y in zip(first, again))
    assert all(torch.equal(x, y) for x, y in zip(kept, (a, w, dy, z)))


def test_refusals(hip, device):
    a, w = torch.randn(6, 8, device=device).bfloat16(), torch.randn(4, 8, device=device).bfloat16()
    with pytest.raises(TypeError):
        hip.linear_act_fwd(a.float(), w)
    with pytest.raises(ValueError):
        hip.linear_act_fwd(a, w.cpu())
    with pytest.raises(ValueError):
        hip.linear_act_fwd(a, w, act="tanh")
    with pytest.raises(ValueError):
        hip.linear_act_bwd(a, w, torch.zeros(6, 4, device=device).bfloat16(), act="gelu")
    fn, n = hip._real.pdt_linear_fwd, None
    good = [n] * 7 + [0, 4, 8, 8, 8, 0, 64, 0, n]
    assert fn(*good) == 0
    for at, bad in ((7, -1), (8, 0), (9, 0), (13, 3), (13, 63), (13, 128), (14, 4), (14, -1)):
        args = list(good)
        args[at] = bad
        assert fn(*args) == -1, (at, bad)
    many = list(good)
    many[7], many[9], many[10], many[11] = 100, 7, 7, 7         # copies of both operands, and no workspace for them
    assert fn(*many) == -3
    assert hip._real.pdt_linear_fwd_workspace(n, n, 100, 4, 7, 7, 7) >= 104 * 16
    fn = hip._real.pdt_linear_bwd
    good = [n] * 8 + [6, 4, 7, 4, 4, 7, 7, 7, 0, 0, 0, n]
    assert fn(*good) == -3
    for at, bad in ((8, 0), (9, 0), (10, 0), (15, 6), (16, 4), (16, -1), (16, 2)):   # (an activation without z)
        args = list(good)
        args[at] = bad
        assert fn(*args) == -1, (at, bad)


# ------------------------------------------------------------------------------------------------ a head that is distilled
def head_step(hip, ops, x, labels, teacher, p, temperature, alpha):
    """Two-layer head: h = x + gelu(x w1 + b1) (the residual), logits = h w2 + b2, distilled; gradients into p's buffers."""
    values, indices, lse = ops.top_logits(teacher, 10, temperature)
    h, z = ops.linear_act_fwd(x, p["w1"], p["b1"], "gelu", x, True)
    logits, _ = ops.linear_act_fwd(h, p["w2"], p["b2"])
    loss, dlogits = ops.distill_ce(logits, labels, values, indices, temperature, alpha, lse)
    dh, _, _ = ops.linear_act_bwd(h, p["w2"], dlogits, dw=p["dw2"], dbias=p["db2"])
    dx, _, _ = ops.linear_act_bwd(x, p["w1"], dh, z, "gelu", p["dw1"], p["db1"])
    return loss, logits, dx, dh                                 # the gradient of x: dx through the product, dh through the residual


def head(device, rows=96, width=200, classes=1000):
    gen = torch.Generator().manual_seed(8)
    p = {"w1": oracle.rows((width, width), gen, scale=width ** -0.5, device=device), "b1": torch.randn(width, generator=gen).to(device) * 0.1,
         "w2": oracle.rows((classes, width), gen, scale=width ** -0.5, device=device), "b2": torch.randn(classes, generator=gen).to(device) * 0.1}
    for n in ("1", "2"):
        p["dw" + n], p["db" + n] = torch.zeros_like(p["w" + n], dtype=torch.float32), torch.zeros_like(p["b" + n])
    x = oracle.rows((rows, width), gen, device=device)
    teacher = oracle.rows((rows, classes), gen, scale=3.0, device=device)
    labels = torch.randint(0, classes, (rows,), generator=gen).to(device)
    return p, x, labels, teacher


def test_head_against_the_oracle(hip, device):
    p, x, labels, teacher = head(device, rows=20)
    loss, logits, dx, dh = head_step(hip, hip, x, labels, teacher, p, 2.0, 0.6)
    names = ("w1", "b1", "w2", "b2")
    q = {n: p[n].double().cpu().requires_grad_(True) for n in names}
    xd = x.double().cpu().requires_grad_(True)
    hid = xd + oracle.act(xd @ q["w1"].t() + q["b1"], "gelu")
    want_logits = hid @ q["w2"].t() + q["b2"]
    v, i, lse = _distill_oracle.top_logits(teacher.cpu(), 10, 2.0)
    want = sum(_distill_oracle.row_loss(want_logits[b], int(labels[b]), list(zip(i[b].tolist(), v[b].tolist())), 2.0, 0.6,
                                        float(lse[b])) for b in range(20)) / 20
    grads = torch.autograd.grad(want, [xd] + [q[n] for n in names])
    # bf16 steps on the way: h, logits, dlogits, dh, dz and the results, each 2^-8 at most: six of them in the 2-norm
    rel = lambda g, t: ((g.double().cpu() - t).norm() / t.norm()).item()  # noqa: E731
    assert rel(logits, want_logits.detach()) < 2 * 2.0 ** -8 and abs(float(loss) - float(want.detach())) < 2.0 ** -6 * float(want.detach())
    for got, t in zip((dx.float() + dh.float(), p["dw1"], p["db1"], p["dw2"], p["db2"]), grads):
        assert rel(got, t) < 6 * 2.0 ** -8


def test_head_captured_recorded_and_on_another_stream(hip, device):
    p, x, labels, teacher = head(device)

    def step():
        for n in ("dw1", "db1", "dw2", "db2"):
            hip._lib.pdt_zero_f32(p[n].data_ptr(), p[n].numel(), hip._stream())
        return head_step(hip, hip, x, labels, teacher, p, 2.0, 0.6)

    def everything(out):
        return [t.clone() for t in out] + [p[n].clone() for n in ("dw1", "db1", "dw2", "db2")]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alone = everything(step())
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(s, t) for s, t in zip(alone, everything(step())))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    program = ListProgram(device, hip)
    with torch.cuda.use_mem_pool(program.pool):
        program.begin()
        recorded = step()
        program.finish()
    for seed in range(4):
        gen = torch.Generator(device=device).manual_seed(seed)
        x.copy_(torch.randn(x.shape, device=device, generator=gen))
        teacher.copy_(torch.randn(teacher.shape, device=device, generator=gen) * 3)
        want = everything(step())
        graph.replay()
        assert all(torch.equal(s, t) for s, t in zip(everything(captured), want))
        torch.cuda.synchronize()
        program.replay()
        assert all(torch.equal(s, t) for s, t in zip(everything(recorded), want))


def test_two_streams_at_once(hip, device):
    """Workspaces belong to a call: layers whose partial sums and copies live in them, on two streams at a time."""
    jobs = []
    for seed, (M, N, K) in enumerate([(333, 777, 1021), (100, 96, 4000)]):
        gen = torch.Generator().manual_seed(seed)
        a, w = oracle.rows((M, K), gen, device=device), oracle.rows((N, K), gen, scale=K ** -0.5, device=device)
        jobs.append((a, w, oracle.rows((M, N), gen, device=device)))

    def layer(a, w, dy):
        y, z = hip.linear_act_fwd(a, w, act="silu", save=True)
        return (y, z) + hip.linear_act_bwd(a, w, dy, z, "silu")

    want = [layer(*job) for job in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(10):
        for n, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[n].append(layer(*jobs[n]))
    torch.cuda.synchronize()
    for n in range(2):
        for out in got[n]:
            assert all(torch.equal(x, y) for x, y in zip(out, want[n]))


@pytest.mark.parametrize("act", ["none", "silu"])
def test_the_largest_widths(hip, device, act):
    """K, then N, of MAX_WIDTH: 32-bit offsets of a tile's rows end just below their limit; one more is refused."""
    from pytorch_distributed_training_amd.ops.ref import MAX_WIDTH
    gen = torch.Generator().manual_seed(11)
    for M, N, K in ((70, 130, MAX_WIDTH - 3), (130, MAX_WIDTH, 8)):
        a, w = oracle.rows((M, 16), gen, device=device), oracle.rows((N if K == 8 else 16, 16), gen, device=device)
        a, w = (a.repeat(1, K // 16 + 1)[:, :K], w.repeat(9, K // 16 + 1)[:N, :K]) if K > 16 else (a[:, :K], w[:, :K])
        y, z = hip.linear_act_fwd(a, w, act=act, save=True)
        dy = y.clone()
        da, dw, db = hip.linear_act_bwd(a, w, dy, z, act)
        rows = slice(N - 130, N)                               # the last columns of y, or all of them
        if K > 16:
            turns, rest = divmod(K, 16)                        # the operands repeat every 16 columns
            want = turns * (a[:, :16].double() @ w[:, :16].double().t()) + a[:, :rest].double() @ w[:, :rest].double().t()
            size = (turns + 1) * (a[:, :16].double().abs() @ w[:, :16].double().abs().t())
        else:
            want, size = a.double() @ w[rows].double().t(), a.double().abs() @ w[rows].double().abs().t()
        bound = (K / 32 + 32) * 2.0 ** -23 * size
        within(z[:, rows] if z is not None else y[:, rows], want, bound * 1.01 + oracle.HALF * want.abs())
        # gradients: of the last columns alone, from dz as the formula has it
        g = dy.double()[:, rows] * (oracle.slope(z.double()[:, rows], act) if act != "none" else 1.0)
        off = g.abs() * oracle.HALF * 1.01 + dy.double()[:, rows].abs() * 3e-6
        at = a[:, -16:].double()
        want = g.t() @ at
        bound = off.t() @ at.abs() + (M / 32 + 32) * 2.0 ** -23 * (g.abs().t() @ at.abs())
        within(dw[rows, -16:] if K > 16 else dw[rows], want, bound * 1.01 + oracle.HALF * (want.abs() + bound))
        if K > 16:
            wt = w[:, -16:].double()
            want = g @ wt
            bound = off @ wt.abs() + (N / 32 + 32) * 2.0 ** -23 * (g.abs() @ wt.abs())
            within(da[:, -16:], want, bound * 1.01 + oracle.HALF * (want.abs() + bound))
        del a, w, y, z, dy, da, dw, db
    wide = torch.zeros(1, MAX_WIDTH + 1, dtype=torch.bfloat16, device=device)
    with pytest.raises(ValueError):
        hip.linear_act_fwd(wide, wide)
    with pytest.raises(ValueError):
        hip.linear_act_bwd(wide, wide, wide[:, :1])
    assert hip._real.pdt_linear_fwd(*[None] * 7, 0, 4, MAX_WIDTH + 1, MAX_WIDTH + 1, MAX_WIDTH + 1, 0, 64, 0, None) == -1
