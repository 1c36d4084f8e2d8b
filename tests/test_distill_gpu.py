"""GPU tier: the distillation kernels against the 64-bit oracle (small rows) and the reference operators (wide ones)."""
import math

import pytest
import torch

import _distill_oracle as oracle
from pytorch_distributed_training_amd.engine.graphs import ListProgram
from pytorch_distributed_training_amd.ops import ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def hip():
    from pytorch_distributed_training_amd.ops import hip as hip_ops
    return hip_ops


def check(hip, args, temperature, alpha, grad_scale=1.0, most=1.0):
    """``most``: the listed probabilities sum to that much (an lse of another temperature)."""
    student, labels, values, indices, lse = args
    rows = student.shape[0]
    loss, grad = hip.distill_ce(student, labels, values, indices, temperature, alpha, lse, grad_scale)
    if student.shape[1] * rows <= 20000:
        want, want_grad = oracle.distill(student, labels, values, indices, temperature, alpha, lse, grad_scale)
    else:
        want, want_grad = ref.distill_ce(student.float(), labels, values, indices, temperature, alpha, lse, grad_scale)
        want, want_grad = want.double().cpu(), want_grad.double().cpu()
    assert loss.dtype == torch.float32 and grad.dtype == student.dtype
    # the reference operator is fp32 itself: its own error on top of the kernel's
    assert abs(float(loss) - float(want)) <= 2 * most * oracle.loss_tolerance(want, temperature, alpha)
    off = (grad.double().cpu() - want_grad).abs()
    allowed = most * oracle.grad_tolerance(want_grad, student.dtype, rows, temperature, alpha, grad_scale)
    assert (off <= allowed).all(), (off - allowed).max()
    padded = grad.as_strided((rows, grad.stride(0)), (grad.stride(0), 1))
    assert grad.stride(0) % 64 == 0 and not padded[:, student.shape[1]:].any()


SIZES = [(1, 1, 1), (3, 2, 2), (5, 7, 7), (4, 63, 5), (2, 64, 64), (3, 65, 9), (9, 1000, 10), (3, 1001, 33), (2, 2048, 100),
         (2, 2049, 65), (3, 8193, 20), (2, 32769, 64), (2, 65537, 100), (1, 131072, 64), (1, 262144, 512)]


@pytest.mark.parametrize("rows,classes,k", SIZES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
def test_distill(hip, device, rows, classes, k, dtype, tail):
    for temperature, alpha, masked, wide in ((1.0, 0.5, False, 0), (2.5, 0.7, True, 3), (4.0, 1.0, False, 8)):
        args = oracle.inputs(rows, classes, k, dtype, temperature, classes + k, masked, tail, device, wide)
        check(hip, args, temperature, alpha, 64.0)


@pytest.mark.parametrize("classes", [9000, 40000, 50001, 65536, 100000, 131072, 140000])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("temperature", [1.0, 2.0, 3.0, 4.0])
def test_distill_both_terms_on_wide_rows(hip, device, classes, dtype, temperature):
    """Every way to the hard term's exponentials, rows that are held in registers, in LDS too, and read twice."""
    for wide, tail in ((0, True), (4, False)):
        args = oracle.inputs(2, classes, 20, dtype, temperature, classes, True, tail, device, wide)
        check(hip, args, temperature, 0.4, 16.0)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("classes", [30, 5000])
def test_distill_slots(hip, device, tail, classes):
    """Duplicates, 64-bit indices, classes out of range, strided values, slots in another type, no labels, 32-bit labels."""
    student, labels, values, indices, lse = oracle.inputs(6, classes, 12, torch.bfloat16, 2.0, 11, False, tail, device)
    indices[:, 7] = indices[:, 0]
    indices[:, 11] = indices[:, 0]
    indices[2] = indices[2, 0]                                   # one class in every slot
    indices[3, 5], indices[4, 6] = classes, -7
    if not tail:
        values = values * 1.5
    check(hip, (student, labels, values, indices, lse), 2.0, 0.6)
    check(hip, (student, labels.int(), values.float(), indices.long(), lse), 2.0, 0.6)
    check(hip, (student, None, values.t().contiguous().t(), indices.long().t().contiguous().t(), lse), 2.0, 1.0)
    far = indices.long()
    far[0, 1] = 1 << 40                                          # wraps to a class in 32 bits
    far[0, 2] = (1 << 32) + 1
    check(hip, (student, labels, values, far, lse), 2.0, 0.6)
    first, last = student[:1].expand(6, -1), labels.clone()
    last[0], last[1] = (1 << 32) + 2, -1
    filled = (indices >= 0) & (indices < classes)
    most = (values.double() - lse[:, None]).exp().mul(filled).sum(dim=1).max().clamp_min(1.0).item() if tail else 1.0
    check(hip, (first, last, values, indices, lse), 1.0, 0.3, most=most)


def test_rows_that_count_for_nothing(hip, device):
    for dtype in DTYPES:
        student, labels, values, indices, lse = oracle.inputs(5, 900, 8, dtype, 2.0, 4, device=device)
        student[0] = -math.inf
        indices[1], labels[1] = -1, -100
        values[2] = -math.inf
        student[3, :] = torch.finfo(dtype).min                    # a mask of the type's lowest value: equal, not empty
        student[4, 1:] = torch.finfo(dtype).min
        labels[3], labels[4] = 5, 0
        indices[4, 0], indices[4, 1:] = 0, -1
        lse[4] = values[4, 0].float() / 2                         # all of the teacher's mass on the one class
        check(hip, (student, labels, values, indices, lse), 2.0, 0.4)
        _, grad = hip.distill_ce(student, labels, values, indices, 2.0, 0.4, lse)
        assert not grad[0].any() and not grad[1].any()
    loss, grad = hip.distill_ce(student[:0], labels[:0], values[:0], indices[:0], 2.0, 0.4, lse[:0])
    assert float(loss) == 0.0 and grad.shape == (0, 900)


def test_confident_student_keeps_its_rest(hip, device):
    """The student's mass outside the list is e^-200: taken as 1 - (listed mass) it would be zero."""
    student = torch.randn(2, 3000, device=device)
    student[:, 7] = 200.0
    values = torch.tensor([[3.0], [2.0]], device=device)
    indices = torch.full((2, 1), 7, dtype=torch.int32, device=device)
    lse = torch.full((2,), 4.0, device=device)
    labels = torch.tensor([7, 9], device=device)
    check(hip, (student, labels, values, indices, lse), 1.0, 0.5)


@pytest.mark.parametrize("classes", [50, 5000, 70000])
def test_nan_reaches_the_loss(hip, device, classes):
    student, labels, values, indices, lse = oracle.inputs(3, classes, 4, torch.bfloat16, 2.0, 2, device=device)
    for bad in (math.nan, math.inf):
        z = student.clone()
        z[1, classes - 1] = bad
        assert math.isnan(float(hip.distill_ce(z, labels, values, indices, 2.0, 0.5, lse)[0]))
        grad = hip.distill_ce(z, labels, values, indices, 2.0, 0.5, lse)[1]
        assert grad[1].isnan().any() and not grad[0].isnan().any() and not grad[2].isnan().any()
    v = values.clone()
    v[2, 1] = math.nan
    for given in (None, lse):
        assert math.isnan(float(hip.distill_ce(student, labels, v, indices, 2.0, 0.5, given)[0]))
    z = student.clone()
    z[0] = math.nan
    assert math.isnan(float(hip.distill_ce(z, labels, values, indices, 2.0, 0.5, lse)[0]))


def test_rows_are_left_as_they_were_and_results_repeat(hip, device):
    student, labels, values, indices, lse = oracle.inputs(300, 5000, 20, torch.bfloat16, 2.0, 6, True, True, device)
    kept = [t.clone() for t in (student, labels, values, indices, lse)]
    first = hip.distill_ce(student, labels, values, indices, 2.0, 0.5, lse)
    for _ in range(3):
        again = hip.distill_ce(student, labels, values, indices, 2.0, 0.5, lse)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    for a, b in zip(kept, (student, labels, values, indices, lse)):
        assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


def test_more_than_four_gigabytes_of_logits(hip, device):
    """Row offsets pass 32 bits: the last rows against the same rows alone."""
    rows, classes, k = 9000, 262144, 4
    logits = torch.empty(rows, classes, dtype=torch.bfloat16, device=device)
    block = torch.randn(100, classes, device=device).to(torch.bfloat16)
    logits.view(90, 100, classes).copy_(block)
    values, indices, lse = hip.top_logits(logits, k, 2.0)
    want = hip.top_logits(logits[-1100:].clone(), k, 2.0)         # (as many rows as take the same kernel)
    for a, b in zip((values, indices, lse), want):
        assert torch.equal(a[-1100:], b)
    labels = torch.arange(rows, device=device)
    _, grad = hip.distill_ce(logits, labels, values, indices, 2.0, 0.5, lse, float(rows))
    _, want = hip.distill_ce(logits[-3:].clone(), labels[-3:], values[-3:], indices[-3:], 2.0, 0.5, lse[-3:], 3.0)
    assert torch.equal(grad[-3:], want)


# ------------------------------------------------------------------------------------------------ top logits
def check_top(hip, logits, k, temperature):
    values, indices, lse = hip.top_logits(logits, k, temperature)
    if logits.numel() <= 20000:
        want_v, want_i, want_l = oracle.top_logits(logits.cpu(), k, temperature)
    else:
        want_v, want_i, want_l = (t.cpu() for t in ref.top_logits(logits, k, temperature))
    assert values.dtype == logits.dtype and indices.dtype == torch.int32 and lse.dtype == torch.float32
    assert torch.equal(indices.cpu().long(), want_i.long())
    assert torch.equal(values.double().cpu().nan_to_num(99.0), want_v.double().nan_to_num(99.0))
    # fp32: a sum of exponentials to 1e-6, its logarithm and maximum to half a step of values up to 100 / T
    assert torch.allclose(lse.double().cpu(), want_l.double(), rtol=1e-6, atol=5e-6, equal_nan=True)


TOP_SIZES = [(1, 1, 1), (3, 5, 5), (4, 63, 10), (2, 64, 64), (3, 512, 32), (2, 1000, 10), (2, 1000, 512), (2, 1001, 33),
             (3, 2048, 32), (2, 2049, 100), (2, 8192, 128), (2, 8193, 20), (2, 32769, 512), (1, 65537, 100), (1, 131073, 256),
             (1, 262144, 512)]


@pytest.mark.parametrize("rows,classes,k", TOP_SIZES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_top_logits(hip, device, rows, classes, k, dtype):
    gen = torch.Generator().manual_seed(classes + k)
    logits = (torch.randn(rows, classes, generator=gen) * 3).to(dtype).to(device)
    check_top(hip, logits, k, 2.0)
    wide = torch.full((rows, classes + 5), math.nan, dtype=dtype, device=device)
    wide[:, :classes] = logits
    wide[0, classes // 3:classes] = -math.inf
    check_top(hip, wide[:, :classes], k, 1.0)
    ties = torch.randint(-2, 3, (rows, classes), generator=gen).to(dtype).to(device)
    check_top(hip, ties, k, 1.0)


@pytest.mark.parametrize("classes", [700, 5000, 33000, 70000])
def test_top_logits_of_rows_that_defeat_the_bound(hip, device, classes):
    """All equal, sorted either way, -inf throughout, NaNs, +-0, infinities: the exact cut, and ties to the lower class."""
    up = torch.arange(classes, device=device, dtype=torch.float32)
    rows = torch.stack([torch.ones_like(up), up, -up, torch.full_like(up, -math.inf), up % 3, torch.zeros_like(up),
                        torch.where(up % 2 == 0, 0.0, -0.0), up.sin()])
    rows[5, classes - 7:] = math.nan
    rows[5, 3] = math.inf
    rows[7, :classes - 4] = -math.inf
    for dtype in (torch.float32, torch.bfloat16):
        for k in (1, 31, 100, 500):
            check_top(hip, rows.to(dtype), k, 1.0)


@pytest.mark.parametrize("k", [1, 64, 128, 300])
def test_top_logits_of_many_wide_rows(hip, device, k):
    """Enough rows for several workgroups per CU; rows that defeat the bound among them."""
    gen = torch.Generator(device=device).manual_seed(k)
    logits = torch.randn(1100, 20011, device=device, generator=gen).to(torch.bfloat16)
    up = torch.arange(20011, device=device)
    logits[3], logits[4], logits[5] = 1.0, up.to(torch.bfloat16), (-up).to(torch.bfloat16)
    logits[6] = -math.inf
    logits[7, 20000] = math.nan
    logits[8, 11] = math.inf
    logits[9, 40:] = -math.inf
    check_top(hip, logits, k, 1.0)


def test_refusals(hip, device):
    student, labels, values, indices, lse = oracle.inputs(4, 9, 3, torch.float32, 1.0, 3, device=device)
    with pytest.raises(TypeError):
        hip.distill_ce(student.double(), labels, values, indices, 1.0, 0.5, lse)
    with pytest.raises(ValueError):
        hip.distill_ce(student, labels.cpu(), values, indices, 1.0, 0.5, lse)
    with pytest.raises(ValueError):
        hip.distill_ce(student, labels, values, indices, 0.0, 0.5, lse)
    with pytest.raises(ValueError):
        hip.distill_ce(student, labels, values, indices[:, :2], 1.0, 0.5, lse)
    with pytest.raises(ValueError):
        hip.top_logits(student.cpu(), 2)
    with pytest.raises(ValueError):
        hip.top_logits(student, 10)
    assert hip.top_logits(student[:0], 2)[0].shape == (0, 2)


def test_status_of_the_entry_points(hip):
    """The C entries refuse what the kernels are not built for before anything is launched."""
    fn = hip._real.pdt_distill_ce
    good = [None] * 8 + [0, 8, 2, 8, 2, 1, 2, 1, 64, 0, 0, 8, 4, 1.0, 0.5, 1.0, None]
    for at, bad in ((8, -1), (9, 0), (9, 262145), (10, 0), (10, 513), (16, 7), (17, 3), (18, -1), (19, 2), (20, 1), (21, 0.0),
                    (21, math.nan)):
        args = list(good)
        args[at] = bad
        assert fn(*args) == -1, (at, bad)
    fn = hip._real.pdt_top_logits
    good = [None] * 4 + [0, 8, 2, 8, 0, 1.0, None]
    assert fn(*good) == 0
    for at, bad in ((4, -1), (5, 0), (6, 0), (6, 9), (6, 513), (8, 3), (9, 0.0)):
        args = list(good)
        args[at] = bad
        assert fn(*args) == -1, (at, bad)


# ------------------------------------------------------------------------------------------------ streams, graphs, lists
def test_on_another_stream(hip, device):
    args = oracle.inputs(64, 3000, 10, torch.bfloat16, 2.0, 1, False, True, device)
    want = hip.distill_ce(*args[:4], 2.0, 0.5, args[4])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = hip.distill_ce(*args[:4], 2.0, 0.5, args[4])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_captured_and_recorded(hip, device):
    """Teacher and student in one graph and in one command list, replayed on new logits with eager work in between."""
    student, labels, _, _, _ = oracle.inputs(50, 3000, 10, torch.bfloat16, 2.0, 1, device=device)
    teacher = torch.randn(50, 3000, device=device).to(torch.bfloat16)

    def step():
        values, indices, lse = hip.top_logits(teacher, 10, 2.0)
        return hip.distill_ce(student, labels, values, indices, 2.0, 0.5, lse)

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    program = ListProgram(device, hip)
    with torch.cuda.use_mem_pool(program.pool):
        program.begin()
        recorded = step()
        program.finish()
    assert program.num_calls == 2
    for seed in range(4):
        gen = torch.Generator(device=device).manual_seed(seed)
        student.copy_(torch.randn(50, 3000, device=device, generator=gen))
        teacher.copy_(torch.randn(50, 3000, device=device, generator=gen))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured[0], want[0]) and torch.equal(captured[1], want[1])
        recorded[1].zero_()
        program.replay()
        assert torch.equal(recorded[0], want[0]) and torch.equal(recorded[1], want[1])
