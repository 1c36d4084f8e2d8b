"""GPU tier: distill_ce in rows that count for nothing, with a term of weight zero and with a small rest."""
import pytest
import torch

import _distill_edges as edges

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    from pytorch_distributed_training_amd.ops import hip as hip_ops
    return hip_ops


WIDTHS = [5, 500, 1000, 5000, 20000, 50001, 65536, 131072, 140001]       # every way in which a row is held


@pytest.mark.parametrize("classes", WIDTHS)
@pytest.mark.parametrize("temperature", [1.0, 2.0, 3.0, 4.0])
@pytest.mark.parametrize("tail", [False, True])
def test_what_padding_rows_hold_reaches_nothing(hip, device, classes, temperature, tail):
    for dtype in (torch.bfloat16, torch.float32):
        edges.check_padding_rows(hip, device, classes, dtype, temperature, tail)


@pytest.mark.parametrize("classes", [9, 1000, 20000])
@pytest.mark.parametrize("tail", [False, True])
def test_a_term_of_weight_zero_is_left_out(hip, device, classes, tail):
    edges.check_weight_zero(hip, device, classes, tail)


@pytest.mark.parametrize("classes", [1500, 9000, 70000])
@pytest.mark.parametrize("temperature", [1.0, 2.0, 2.7, 3.0])
def test_a_small_rest_keeps_its_digits(hip, device, classes, temperature):
    edges.check_small_rest(hip, device, classes, temperature)


@pytest.mark.parametrize("classes", [300, 1500, 9000, 70000])
@pytest.mark.parametrize("temperature", [0.7, 1.0, 1.3, 2.7, 3.0, 7.0])
def test_lse_of_large_logits(hip, device, classes, temperature):
    edges.check_lse(hip, device, classes, temperature)
