"""Edge cases of distill_ce, for the reference operators and the kernels alike (``ops``)."""
import math

import torch

import _distill_oracle as oracle


def check_padding_rows(ops, device, classes, dtype, temperature, tail):
    """Rows without a label and without a slot: NaN and infinities in them reach neither loss nor gradient."""
    student, labels, values, indices, lse = oracle.inputs(6, classes, 3, dtype, temperature, classes, False, tail, device)
    want_loss, want = ops.distill_ce(student[:2], labels[:2], values[:2], indices[:2], temperature, 0.6,
                                     lse[:2] if tail else None)
    labels[2:], indices[2:] = -100, -1
    student[2], student[3, classes // 2], student[4, 0], student[5] = math.nan, math.nan, math.inf, math.inf
    for alpha, given in ((0.6, labels), (1.0, labels.clone())):
        if alpha == 1.0:
            given[2:] = 1                                      # a label that alpha = 1 leaves out
        loss, grad = ops.distill_ce(student, given, values, indices, temperature, alpha, lse)
        assert not grad[2:].any() and not grad[2:].isnan().any() and not grad[:2].isnan().any() and math.isfinite(float(loss))
        if alpha == 0.6:                                       # (the mean is over all six rows)
            assert abs(float(loss) * 3 - float(want_loss)) <= 1e-6 * abs(float(want_loss))
            # one expression with the weights of 6 and of 2 rows: a sum of four products of a weight and a factor of at most 1,
            # which may cancel; five roundings of 2^-24 in each, in both calls, and half a step of the stored type in each
            weights = 0.5 * (0.4 + 0.6 * temperature)
            bound = 2 * 4 * 5 * 2.0 ** -24 * weights + torch.finfo(dtype).eps * 1.01 * want.float().abs()
            assert ((grad[:2].float() * 3 - want.float()).abs() <= bound).all()


def check_weight_zero(ops, device, classes, tail):
    """alpha = 0: no soft term, whatever the slots hold; alpha = 1: no hard term, whatever the label's logit is."""
    student, labels, values, indices, lse = oracle.inputs(4, classes, 3, torch.float32, 2.0, 7, False, tail, device)
    bare = oracle.distill(student, labels, values, indices, 2.0, 0.0, lse)
    tolerance = oracle.loss_tolerance(bare[0], 2.0, 0.0), oracle.grad_tolerance(bare[1], torch.float32, 4, 2.0, 0.0)
    poor = values.clone()
    poor[1], poor[2, 0] = math.nan, math.inf
    gone = student.clone()
    at = indices.long()[:, 2]
    hit = at != labels
    assert hit.any()
    gone[hit, at[hit]] = -math.inf                             # the student rules out a class that the teacher lists
    for z, v in ((student, poor), (gone, values)):
        loss, grad = ops.distill_ce(z, labels, v, indices, 2.0, 0.0, lse)
        want, want_grad = bare if z is student else oracle.distill(z, labels, values, torch.full_like(indices, -1), 2.0, 0.0, lse)
        assert abs(float(loss) - float(want)) <= tolerance[0], (float(loss), float(want))
        assert ((grad.double().cpu() - want_grad).abs() <= tolerance[1].clamp_min(2e-6)).all()
    loss, grad = ops.distill_ce(student, None, values, indices, 2.0, 0.0, lse)
    assert float(loss) == 0.0 and not grad.any()
    gone = student.clone()
    labels = torch.full_like(labels, classes - 1)
    gone[:, classes - 1] = -math.inf
    indices = torch.where(indices == classes - 1, torch.zeros_like(indices), indices)
    loss, grad = ops.distill_ce(gone, labels, values, indices, 2.0, 1.0, lse)
    want, want_grad = ops.distill_ce(gone, None, values, indices, 2.0, 1.0, lse)
    assert math.isfinite(float(loss)) and torch.equal(loss, want) and torch.equal(grad, want_grad)
