"""CPU tier: the reference distill_ce in rows that count for nothing, with a term of weight zero and with a small rest."""
import pytest
import torch

import _distill_edges as edges
from pytorch_distributed_training_amd.ops import ref


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_what_padding_rows_hold_reaches_nothing(tail, dtype):
    edges.check_padding_rows(ref, "cpu", 30, dtype, 2.0, tail)


@pytest.mark.parametrize("tail", [False, True])
def test_a_term_of_weight_zero_is_left_out(tail):
    edges.check_weight_zero(ref, "cpu", 30, tail)


@pytest.mark.parametrize("temperature", [1.0, 2.7, 3.0])
def test_a_small_rest_keeps_its_digits(temperature):
    edges.check_small_rest(ref, "cpu", 1500, temperature)


@pytest.mark.parametrize("temperature", [0.7, 2.7])
def test_lse_of_large_logits(temperature):
    edges.check_lse(ref, "cpu", 1500, temperature)
