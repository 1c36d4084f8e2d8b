"""CPU tier: the reference distillation operators against the 64-bit oracle, and every refusal."""
import math

import pytest
import torch

import _distill_oracle as oracle
from pytorch_distributed_training_amd.ops import ref


@pytest.mark.parametrize("rows,classes,k", [(1, 1, 1), (3, 2, 2), (5, 7, 7), (4, 65, 5), (6, 100, 33)])
@pytest.mark.parametrize("temperature,alpha", [(1.0, 0.5), (3.0, 0.9), (2.0, 1.0), (0.5, 0.0)])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("masked", [False, True])
def test_loss_and_gradient(rows, classes, k, temperature, alpha, tail, masked):
    args = oracle.inputs(rows, classes, k, torch.float32, temperature, rows * 31 + k, masked, tail)
    student, labels, values, indices, lse = args
    loss, grad = ref.distill_ce(student, labels, values, indices, temperature, alpha, lse, 2.0)
    want, want_grad = oracle.distill(student, labels, values, indices, temperature, alpha, lse, 2.0)
    assert abs(float(loss) - float(want)) <= oracle.loss_tolerance(want, temperature, alpha)
    assert ((grad.double() - want_grad).abs() <= oracle.grad_tolerance(want_grad, torch.float32, rows, temperature, alpha, 2.0)).all()


@pytest.mark.parametrize("tail", [False, True])
def test_gradient_against_differences(tail):
    student, labels, values, indices, lse = oracle.inputs(3, 11, 4, torch.float32, 2.0, 5, False, tail)
    _, grad = oracle.distill(student, labels, values, indices, 2.0, 0.7, lse)
    h = 1e-5
    for b in range(3):
        for c in range(11):
            moved = []
            for sign in (1, -1):
                z = student.double().clone()
                z[b, c] += sign * h
                moved.append(float(oracle.distill(z, labels, values, indices, 2.0, 0.7, lse)[0]))
            assert abs((moved[0] - moved[1]) / (2 * h) - float(grad[b, c])) < 1e-8     # central: h^2 / 6 f''' + 1e-16 / h
    got = ref.distill_ce(student, labels, values, indices, 2.0, 0.7, lse)[1]
    assert ((got.double() - grad).abs() <= oracle.grad_tolerance(grad, torch.float32, 3, 2.0, 0.7)).all()


def test_duplicate_slots_are_added_up():
    student, labels, values, indices, _ = oracle.inputs(4, 20, 6, torch.float32, 2.0, 9, tail=False)
    indices[:, 3] = indices[:, 0]
    indices[:, 5] = indices[:, 0]
    loss, grad = ref.distill_ce(student, labels, values, indices, 2.0, 0.8)
    want, want_grad = oracle.distill(student, labels, values, indices, 2.0, 0.8, None)
    assert abs(float(loss) - float(want)) <= oracle.loss_tolerance(want, 2.0, 0.8)
    assert ((grad.double() - want_grad).abs() <= oracle.grad_tolerance(want_grad, torch.float32, 4, 2.0, 0.8)).all()


def test_an_lse_of_another_temperature_still_has_the_gradient_of_its_loss():
    """The listed probabilities then sum to more than 1: the softmax is weighted with their sum."""
    student, labels, values, indices, lse = oracle.inputs(4, 30, 6, torch.float32, 2.0, 9)
    loss, grad = ref.distill_ce(student, labels, values, indices, 1.0, 0.8, lse)
    want, want_grad = oracle.distill(student, labels, values, indices, 1.0, 0.8, lse)
    most = torch.exp(values.double() - lse.double()[:, None]).sum(dim=1).max().item()        # the tolerances are for a mass of 1
    assert most > 2
    assert abs(float(loss) - float(want)) <= most * oracle.loss_tolerance(want, 1.0, 0.8)
    assert ((grad.double() - want_grad).abs() <= most * oracle.grad_tolerance(want_grad, torch.float32, 4, 1.0, 0.8)).all()


def test_student_equal_to_teacher_has_no_soft_loss():
    logits = torch.randn(5, 30, generator=torch.Generator().manual_seed(0)) * 3
    values, indices, lse = ref.top_logits(logits, 6, 2.0)
    loss, grad = ref.distill_ce(logits, None, values, indices, 2.0, 1.0, lse)
    assert abs(float(loss)) < 1e-5 and grad.abs().max() < 1e-6


def test_soft_targets_over_every_class_are_the_full_divergence():
    gen = torch.Generator().manual_seed(1)
    teacher, student = torch.randn(4, 12, generator=gen), torch.randn(4, 12, generator=gen)
    values, indices, lse = ref.top_logits(teacher, 12, 3.0)
    full = torch.nn.functional.kl_div(torch.log_softmax(student.double() / 3, 1), torch.softmax(teacher.double() / 3, 1),
                                      reduction="batchmean") * 9
    for given in (None, lse):
        loss, _ = ref.distill_ce(student, None, values, indices, 3.0, 1.0, given)
        assert abs(float(loss) - float(full)) <= oracle.loss_tolerance(full, 3.0, 1.0)


def test_rows_that_count_for_nothing():
    student, labels, values, indices, lse = oracle.inputs(4, 9, 3, torch.float32, 1.0, 3)
    student[0] = -math.inf
    indices[1] = -1
    labels[1] = -100
    indices[2] = 9                                                # no class either
    loss, grad = ref.distill_ce(student, labels, values, indices, 1.0, 0.5, lse)
    want, want_grad = oracle.distill(student, labels, values, indices, 1.0, 0.5, lse)
    assert abs(float(loss) - float(want)) <= oracle.loss_tolerance(want, 1.0, 0.5)
    assert grad[0].abs().max() == 0 and grad[1].abs().max() == 0 and grad[2].abs().max() > 0
    loss, grad = ref.distill_ce(student[:0], labels[:0], values[:0], indices[:0], 1.0, 0.5, lse[:0])
    assert float(loss) == 0 and grad.shape == (0, 9)


@pytest.mark.parametrize("rows,classes,k", [(1, 1, 1), (4, 30, 7), (3, 5, 5)])
def test_top_logits(rows, classes, k):
    gen = torch.Generator().manual_seed(classes)
    logits = torch.randint(-3, 4, (rows, classes), generator=gen).float()      # many ties
    logits[0, classes // 2:] = -math.inf
    if rows > 2:
        logits[1] = -math.inf
        logits[2, classes - 1] = math.nan
        logits[2, 0] = math.inf
    values, indices, lse = ref.top_logits(logits, k, 2.0)
    want_v, want_i, want_l = oracle.top_logits(logits, k, 2.0)
    assert torch.equal(indices.long(), want_i) and indices.dtype == torch.int32
    assert torch.equal(values.double().nan_to_num(99.0), want_v.nan_to_num(99.0))
    assert torch.allclose(lse.double(), want_l, rtol=1e-6, atol=1e-6, equal_nan=True)


def test_refusals():
    student, labels, values, indices, lse = oracle.inputs(4, 9, 3, torch.float32, 1.0, 3)

    def refuse(error, **other):
        args = dict(logits=student, labels=labels, values=values, indices=indices, temperature=1.0, alpha=0.5, lse=lse)
        args.update(other)
        with pytest.raises(error):
            ref.distill_ce(**args)

    refuse(TypeError, logits=student.double())
    refuse(ValueError, logits=student.t())
    refuse(ValueError, logits=student[0])
    refuse(ValueError, logits=student.t().contiguous().t())
    refuse(ValueError, logits=student[:, :0])
    refuse(ValueError, logits=torch.zeros(1, ref.MAX_CLASSES + 1).expand(4, -1))
    refuse(TypeError, labels=labels.float())
    refuse(ValueError, labels=labels[:3])
    refuse(ValueError, labels=torch.zeros(8, dtype=torch.int64)[::2])
    refuse(TypeError, values=values.double())
    refuse(TypeError, indices=indices.to(torch.int16))
    refuse(ValueError, values=values[:, :2])
    refuse(ValueError, values=values[:3], indices=indices[:3])
    refuse(ValueError, values=values[:, :0], indices=indices[:, :0])
    refuse(ValueError, values=torch.zeros(4, ref.MAX_TOP + 1), indices=torch.zeros(4, ref.MAX_TOP + 1, dtype=torch.int32))
    refuse(TypeError, lse=lse.double())
    refuse(ValueError, lse=lse[:2])
    refuse(ValueError, temperature=0.0)
    refuse(ValueError, temperature=math.nan)
    refuse(ValueError, alpha=1.5)
    refuse(ValueError, alpha=math.nan)
    for k in (0, 10, -1):
        with pytest.raises(ValueError):
            ref.top_logits(student, k)
    with pytest.raises(ValueError):
        ref.top_logits(torch.zeros(2, 2000), ref.MAX_TOP + 1)
    with pytest.raises(TypeError):
        ref.top_logits(student.long(), 2)
    with pytest.raises(ValueError):
        ref.top_logits(student, 2, math.inf)
