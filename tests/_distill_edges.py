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


def check_small_rest(ops, device, classes, temperature):
    """512 slots that hold all but 1e-5 of the teacher's mass, and a student as sure of them: the gradient of the classes that
    are not listed is q_i (q_r - P_r) / q_r, with both rests some 1e-5.  Taken as 1 minus an fp32 sum, P_r is off by a percent."""
    gen = torch.Generator().manual_seed(classes)
    k, T = 512, temperature
    values = (torch.randn(2, k, generator=gen) * 0.1 - math.log(k)) * T
    indices = torch.stack([torch.randperm(classes, generator=gen)[:k] for _ in range(2)]).to(torch.int32)
    total = torch.logsumexp(values.double() / T, 1)
    lse = (total + 1e-5).float()
    rest = 1.0 - torch.exp(values.double() / T - lse.double()[:, None]).sum(1)
    assert ((rest > 5e-6) & (rest < 2e-5)).all()
    student = torch.randn(2, classes, generator=gen) * T
    lift = 12.0 + math.log((classes - k) / k)
    student.scatter_(1, indices.long(), values + (lift + math.log(k)) * T)
    loss, grad = ops.distill_ce(student.to(device), None, values.to(device), indices.to(device), T, 1.0, lse.to(device))
    log_q = torch.log_softmax(student.double() / T, 1)
    unlisted = torch.ones(2, classes, dtype=torch.bool).scatter_(1, indices.long(), False)
    q = log_q.exp()
    q_rest = torch.where(unlisted, q, torch.zeros_like(q)).sum(1, keepdim=True)
    assert ((q_rest > 3e-6) & (q_rest < 3e-5)).all()
    share = q / q_rest * (T / 2)
    want = share * (q_rest - rest[:, None])
    # fp32: exponents of up to 30 with roundings of 2^-23 in the sums and in q_i, 1e-5 of each rest; the rest itself to 2^-23
    bound = share * 2e-5 * (q_rest + rest[:, None])
    off = (grad.double().cpu() - want).abs()[unlisted]
    assert (off <= bound[unlisted]).all(), (off / bound[unlisted]).max().item()


def check_lse(ops, device, classes, temperature):
    """Large logits: logits / T rounded once, in the result (an fp32 1 / T shifts every row by up to 2^-24 of it again)."""
    gen = torch.Generator().manual_seed(classes)
    logits = torch.randn(40, classes, generator=gen) * 3 + torch.arange(40)[:, None] * 8.0
    want = torch.logsumexp(logits.double() / temperature, 1)
    _, _, lse = ops.top_logits(logits.to(device), 3, temperature)
    # half a step of fp32; the sum of exponentials, whose weights are off by some 2e-7 of their exponents, and its logarithm: 3e-6
    assert ((lse.double().cpu() - want).abs() <= 2.0 ** -24 * 1.01 * want.abs() + 3e-6).all()
