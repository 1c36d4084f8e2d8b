"""64-bit oracle of the distillation operators, written from their definition row by row."""
import math

import torch


def top_logits(logits, k, temperature):
    values, indices, lse = [], [], []
    for row in logits.double().tolist():
        order = sorted((c for c in range(len(row)) if row[c] != -math.inf),
                       key=lambda c: (0 if math.isnan(row[c]) else 1, 0.0 if math.isnan(row[c]) else -row[c], c))[:k]
        values.append([row[c] for c in order] + [-math.inf] * (k - len(order)))
        indices.append(order + [-1] * (k - len(order)))
        lse.append(torch.logsumexp(torch.tensor(row, dtype=torch.float64) / temperature, 0).item())
    return torch.tensor(values, dtype=torch.float64), torch.tensor(indices), torch.tensor(lse, dtype=torch.float64)


def row_loss(z, label, slots, temperature, alpha, lse):
    """Loss of one row (``z`` [N] fp64); ``slots``: [(class, value)]; differentiable in ``z``."""
    N = z.shape[0]
    zero = (z * 0.0).nan_to_num(0.0, 0.0, 0.0).sum()
    if torch.isneginf(z).all():
        return zero
    out = zero
    log_q = torch.log_softmax(z / temperature, 0)
    slots = [(c, v) for c, v in slots if 0 <= c < N and v != -math.inf]
    if slots:
        total = lse if lse is not None else torch.logsumexp(torch.tensor([v / temperature for _, v in slots], dtype=torch.float64), 0)
        mass = {}
        for c, v in slots:
            mass[c] = mass.get(c, 0.0) + math.exp(v / temperature - total)
        soft = sum(P * (math.log(P) - log_q[c]) for c, P in mass.items() if P > 0)
        others = [c for c in range(N) if c not in mass and z[c] != -math.inf]
        rest = max(1.0 - sum(mass.values()), 0.0)
        if lse is not None and others and rest > 0:
            soft = soft + rest * (math.log(rest) - torch.logsumexp(log_q[others], 0))
        out = out + alpha * temperature ** 2 * soft
    if label is not None and 0 <= label < N:
        out = out - (1.0 - alpha) * torch.log_softmax(z, 0)[label]
    return out


def distill(logits, labels, values, indices, temperature, alpha, lse, grad_scale=1.0):
    """(mean loss, gradient) in 64 bits."""
    z = logits.detach().double().cpu().requires_grad_(True)
    B = z.shape[0]
    values, indices = values.double().cpu().tolist(), indices.cpu().tolist()
    labels = None if labels is None else labels.cpu().tolist()
    lse = None if lse is None else lse.double().cpu().tolist()
    loss = sum(row_loss(z[b], None if labels is None else labels[b], list(zip(indices[b], values[b])), temperature, alpha,
                        None if lse is None else lse[b]) for b in range(B)) / B
    (grad,) = torch.autograd.grad(loss * grad_scale, z)
    return loss.detach(), grad.nan_to_num(0.0, 0.0, 0.0) if torch.isneginf(z).any() else grad


def inputs(rows, classes, k, dtype, temperature, seed, masked=False, tail=True, device="cpu", wide=0):
    """Logits of a student and a teacher that agree somewhat; ``wide``: rows of a tensor ``wide`` columns wider."""
    gen = torch.Generator().manual_seed(seed)
    teacher = torch.randn(rows, classes, generator=gen) * 2
    teacher.scatter_add_(1, torch.randint(0, classes, (rows, 3), generator=gen), torch.rand(rows, 3, generator=gen) * 8)
    student = teacher * 0.6 + torch.randn(rows, classes, generator=gen)
    labels = torch.randint(0, classes, (rows,), generator=gen)
    if masked and classes > 4:
        student[:, -classes // 5:] = -math.inf
        teacher[:, -classes // 5:] = -math.inf
        labels = labels % (classes - (classes + 4) // 5)
    teacher = teacher.to(dtype).float()
    values, indices = torch.topk(teacher, k, dim=1)
    lse = torch.logsumexp(teacher / temperature, 1) if tail else None
    values, indices = values.to(dtype), indices.to(torch.int32)
    if masked:
        gone = torch.rand(rows, k, generator=gen) < 0.2
        gone |= torch.isinf(values)
        if rows > 2:
            gone[1] = True
            labels[2] = -100
        values = values.masked_fill(gone, math.nan).masked_fill(gone & (torch.rand(rows, k, generator=gen) < 0.5), -math.inf)
        indices = indices.masked_fill(gone, -1)
    student = student.to(dtype)
    if wide:
        big = torch.full((rows, classes + wide), math.nan, dtype=dtype)
        big[:, :classes] = student
        student = big.to(device)[:, :classes]
    move = lambda t: None if t is None else t.to(device)  # noqa: E731
    return move(student), move(labels), move(values), move(indices), move(lse)


def grad_tolerance(grad, dtype, rows, temperature, alpha, grad_scale=1.0):
    """Half a step of the stored type, and fp32 arithmetic: a gradient is a sum of four products of probabilities (each at
    most 1, through an exponential whose argument is rounded: 2e-6 relative where it is not negligible) with the weights."""
    scale = grad_scale / rows * ((1.0 - alpha) + alpha * temperature)
    half_step = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 2.0 ** -24
    smallest = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}[dtype]
    return grad.abs() * half_step * 1.01 + 8e-6 * scale + smallest


def loss_tolerance(loss, temperature, alpha):
    """fp32 arithmetic: logarithms of up to ~30 to 2^-23, 64-way sums; the soft term is scaled by alpha T^2."""
    return 2e-5 * (1.0 + alpha * temperature ** 2) + 2e-6 * abs(float(loss))
