"""A backbone trained from a larger model's answers: the engine's forward, the distillation operators, the engine's backward."""
import pytest
import torch

import _distill_oracle as oracle
from pytorch_distributed_training_amd.engine import NativeResNet
from pytorch_distributed_training_amd.models import get_model, get_spec
from pytorch_distributed_training_amd.ops import ref

TEMPERATURE, ALPHA, K = 2.0, 0.7, 4


def distilled_step(student, teacher, ops, img, label):
    """What a training program does for one batch; gradients are in ``student.params`` afterwards."""
    values, classes, lse = ops.top_logits(teacher.forward(img, train=False), K, TEMPERATURE)
    logits = student.forward(img, train=True)
    loss, dlogits = ops.distill_ce(logits, label, values, classes, TEMPERATURE, ALPHA, lse)
    student.backward(dlogits)
    return loss, logits, dlogits, (values, classes, lse)


def test_gradients_of_the_whole_network_against_autograd():
    torch.manual_seed(0)
    net, big = get_model("ResNet18", 10), get_model("ResNet34", 10)
    student = NativeResNet(get_spec("ResNet18", 10), torch.device("cpu"), ref, torch.float32)
    teacher = NativeResNet(get_spec("ResNet34", 10), torch.device("cpu"), ref, torch.float32)
    student.load_state_dict(net.state_dict())
    teacher.load_state_dict(big.state_dict())
    img, label = torch.randn(4, 3, 64, 64), torch.randint(0, 10, (4,))
    loss, _, _, (values, classes, lse) = distilled_step(student, teacher, ref, img, label)
    net.train()
    z = net(img).double()
    want = sum(oracle.row_loss(z[b], int(label[b]), list(zip(classes[b].tolist(), values[b].tolist())), TEMPERATURE, ALPHA,
                               float(lse[b])) for b in range(4)) / 4
    want.backward()
    assert float(loss) == pytest.approx(float(want.detach()), rel=1e-4)
    g = student.params.export("g")
    for key, p in net.named_parameters():
        # Frobenius-relative: a ReLU whose pre-activation is some 1e-6 may flip between the two implementations
        err = (g[key] - p.grad).norm().item() / (p.grad.norm().item() + 1e-12)
        assert err < 3e-2, (key, err)


@pytest.mark.gpu
@pytest.mark.parametrize("classes", [1000, 100])
def test_step_on_the_kernels(device, classes):
    from pytorch_distributed_training_amd.ops import hip
    torch.manual_seed(0)
    student = NativeResNet(get_spec("ResNet18", classes), device, hip, torch.bfloat16)
    teacher = NativeResNet(get_spec("ResNet34", classes), device, hip, torch.bfloat16)
    student.load_state_dict(get_model("ResNet18", classes).state_dict())
    teacher.load_state_dict(get_model("ResNet34", classes).state_dict())
    B = 12
    img, label = torch.randn(B, 3, 64, 64, device=device), torch.randint(0, classes, (B,), device=device)
    kept = {}
    backward = student.backward

    def remember(dlogits):
        kept["pooled"] = student._saved["pooled"].clone()
        backward(dlogits)

    student.backward = remember
    loss, logits, dlogits, (values, at, lse) = distilled_step(student, teacher, hip, img, label)
    want, want_grad = oracle.distill(logits, label, values, at, TEMPERATURE, ALPHA, lse)
    assert abs(float(loss) - float(want)) <= oracle.loss_tolerance(want, TEMPERATURE, ALPHA)
    assert ((dlogits.double().cpu() - want_grad).abs() <= oracle.grad_tolerance(want_grad, torch.bfloat16, B, TEMPERATURE, ALPHA)).all()
    # the classifier's gradients, sums of B products and of B numbers in fp32, from that very dlogits; linear_act_bwd's too
    d, x = dlogits.double(), kept["pooled"].double()
    bound_w, bound_b = B * 2.0 ** -23 * (d.abs().t() @ x.abs()), B * 2.0 ** -23 * d.abs().sum(0)
    assert ((student.params.grad("fc.weight").double() - d.t() @ x).abs() <= bound_w).all()
    assert ((student.params.grad("fc.bias").double() - d.sum(0)).abs() <= bound_b).all()
    dw, db = torch.zeros(classes, x.shape[1], device=device), torch.zeros(classes, device=device)
    hip.linear_act_bwd(kept["pooled"], student.params.compute("fc.weight"), dlogits, dw=dw, dbias=db)
    assert ((dw.double() - d.t() @ x).abs() <= bound_w).all() and ((db.double() - d.sum(0)).abs() <= bound_b).all()
    assert student.params.g.isfinite().all() and student.params.grad("conv1.weight").any()
