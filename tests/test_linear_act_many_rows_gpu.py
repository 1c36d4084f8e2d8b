"""GPU tier: the linear operators on row counts at the limits of a launch and of 32-bit arithmetic."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    from pytorch_distributed_training_amd.ops import hip as hip_ops
    return hip_ops


def test_copies_of_more_threads_than_32_bits_count(hip, device):
    """An operand whose rows start anywhere is copied, 16 bytes a thread: 2^26 rows of 65 vectors.  Row r is the window of a long
    vector that begins at its element r; whole numbers, so that every sum is exact."""
    M, N, K = 2 ** 26 + 64, 3, 513
    base = torch.randint(-1, 2, (M + K,), device=device).to(torch.bfloat16)
    a = base.as_strided((M, K), (1, 1))
    w = torch.randint(-1, 2, (N, K), device=device).to(torch.bfloat16)
    y, _ = hip.linear_act_fwd(a, w)
    for at in (0, 2 ** 24 - 100, 2 ** 25 - 100, M - 70000):
        want = (a[at:at + 70000].double() @ w.double().t()).to(torch.bfloat16)
        assert torch.equal(y[at:at + 70000], want)


def test_the_last_rows_of_as_many_as_32_bits_number(hip, device):
    """4096 workgroups share the rows of dbias, and the last one's end lies past 2^31."""
    from pytorch_distributed_training_amd.ops.ref import MAX_ROWS
    dy = torch.zeros(MAX_ROWS, 8, dtype=torch.bfloat16, device=device)
    dy[-1000:] = 1.0
    a = torch.ones(1, 8, dtype=torch.bfloat16, device=device).expand(MAX_ROWS, 8)
    w = torch.ones(8, 8, dtype=torch.bfloat16, device=device)
    _, dw, db = hip.linear_act_bwd(a, w, dy, need_da=False)
    assert (db == 1000.0).all() and (dw == 1000.0).all()
