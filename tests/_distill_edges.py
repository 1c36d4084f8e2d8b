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
