"""Row counts that reach the limits of a launch and of 32-bit row numbers."""
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


@pytest.mark.gpu
def test_more_threads_than_32_bits_count(device):
    """2^26 rows at 64 threads each, and 2^22 at 1024, are more threads than one launch takes.  Row r is the window of a long
    vector that begins at its element r."""
    from pytorch_distributed_training_amd.ops import hip
    rows, classes, k = 2 ** 26 + 70, 10, 3
    base = torch.randn(rows + classes, device=device).to(torch.bfloat16)
    logits = base.as_strided((rows, classes), (1, 1))
    values, indices, lse = hip.top_logits(logits, k, 2.0)
    labels = torch.arange(rows, device=device, dtype=torch.int32) % (classes + 1)
    loss, grad = hip.distill_ce(logits, labels, values, indices, 2.0, 0.5, lse, float(rows))
    for at in (0, 2 ** 21 - 100, 2 ** 25 - 100, rows - 200):
        part = slice(at, at + 200)
        v, i, l = hip.top_logits(logits[part], k, 2.0)
        assert torch.equal(v, values[part]) and torch.equal(i, indices[part]) and torch.equal(l, lse[part])
        _, g = hip.distill_ce(logits[part], labels[part], v, i, 2.0, 0.5, l, 200.0)
        assert torch.equal(g, grad[part])
    total = 0.0
    for part in torch.arange(0, rows, 2 ** 23).tolist():
        cut = slice(part, min(part + 2 ** 23, rows))
        total += float(hip.distill_ce(logits[cut], labels[cut], values[cut], indices[cut], 2.0, 0.5, lse[cut])[0]) * (cut.stop - cut.start)
    assert abs(float(loss) - total / rows) <= 4 * 2.0 ** -24 * float(loss)     # a rounding of each mean, of 64-bit sums
    del grad, values, indices, lse, labels
    rows, classes, k = 2 ** 22 + 5, 600, 129
    logits = base.as_strided((rows, classes), (1, 1))
    values, indices, lse = hip.top_logits(logits, k, 1.0)
    for at in (0, 2 ** 21 - 100, rows - 200):
        part = slice(at, at + 200)
        v, i, l = hip.top_logits(logits[part], k, 1.0)
        assert torch.equal(v, values[part]) and torch.equal(i, indices[part]) and torch.equal(l, lse[part])
