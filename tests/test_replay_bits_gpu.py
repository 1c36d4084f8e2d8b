"""GPU tier: with ordered sums a replayed step gives the eager step's bits: whatever differs without them is the order of sums."""
import pytest
import torch

from test_graphs_gpu import _make, _sync_state

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("model", ["ResNet18", "ResNet50"])
@pytest.mark.parametrize("replay", ["list", "graph"])
def test_replay_equals_eager_bit_for_bit_with_ordered_sums(model, replay):
    from pytorch_distributed_training_amd.ops import hip
    hip.set_deterministic(True)
    try:
        lead, opt = _make(False, False, model)
        subject, _ = _make(True, False, model, replay)
        gen = torch.Generator().manual_seed(5)
        for step in range(8):
            x = torch.randint(0, 255, (16, 64, 64, 3), generator=gen, dtype=torch.uint8).cuda()
            y = torch.randint(0, 100, (16,), generator=gen).cuda()
            _sync_state(subject, lead)
            want, got = lead.forward_backward(x, y), subject.forward_backward(x, y)
            assert torch.equal(got, want) and torch.equal(subject.params.g, lead.params.g), step
            assert torch.equal(subject.running_mean, lead.running_mean) and torch.equal(subject.running_var, lead.running_var), step
            opt.step(grad_scale=lead.reducer.grad_scale)
            lead.refresh_derived_weights()
        torch.cuda.synchronize()
        assert next(iter(subject._plans.values())) is not None, "the step was not recorded"
    finally:
        hip.set_deterministic(False)
