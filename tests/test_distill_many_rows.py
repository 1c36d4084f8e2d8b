"""Row counts that reach the limit of 32-bit row numbers."""
import pytest
import torch

from pytorch_distributed_training_amd.ops import ref


def test_more_rows_than_32_bits_count_are_refused():
    """As a 32-bit number 2^32 + 5 rows are five: nothing would be written to the others."""
    for rows in (ref.MAX_ROWS + 1, 2 ** 31, 2 ** 32 + 5):
        logits = torch.zeros(1, 4).expand(rows, 4)
        with pytest.raises(ValueError):
            ref.check_top_logits(logits, 2, 1.0)
        with pytest.raises(ValueError):
            ref.check_distill_ce(logits, None, logits[:, :2], torch.zeros(1, 2, dtype=torch.int32).expand(rows, 2), 1.0, 0.5, None)
        with pytest.raises(ValueError):
            ref.check_linear_act_fwd(logits, torch.zeros(3, 4), None, "none", None)
    ref.check_top_logits(torch.zeros(1, 4).expand(ref.MAX_ROWS, 4), 2, 1.0)
