"""Cases of the classifier-head and distillation operators: what is measured, their plain forms and their values in 64 bits.

``own`` false: elementary torch operations in 32 bits, rounded once at the end.  ``own`` true: the calls a training
program makes of the framework's operators (``get_ops(device)``).
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
_LARGEST_ROWS = 4096 * 131072                # logits of the largest distillation case
_LARGEST_SORT = 2048 * 131072                # ... and of the largest top_logits case
_LARGEST_PRODUCT = 8192 * 16384 * 4096       # multiply-adds of the largest product


def listed():
    return [
        # a distillation step on eight images per GPU: latency alone
        dict(name="distill 8x1000 k5 tail", op="distill", rows=8, classes=1000, k=5, dtype="bf16", temperature=2.0, alpha=0.5,
             tail=True, masked=False),
        # the repository's default per-GPU batch, 1000 classes, ten teacher logits per image
        dict(name="distill 1536x1000 k10", op="distill", rows=1536, classes=1000, k=10, dtype="bf16", temperature=4.0, alpha=0.9,
             tail=False, masked=False),
        # fp32 logits of an odd width: padding classes masked, some images without a teacher or without a label
        dict(name="distill 509x49999 k33 fp32", op="distill", rows=509, classes=49999, k=33, dtype="fp32", temperature=1.0,
             alpha=0.7, tail=True, masked=True),
        # a token batch over a large vocabulary, the teacher's rest kept as one class
        dict(name="distill 4096x131072 k64", op="distill", rows=4096, classes=131072, k=64, dtype="bf16", temperature=2.0,
             alpha=0.5, tail=True, masked=False),
        # the teacher's half of the second case
        dict(name="top 1536x1000 k10", op="top", rows=1536, classes=1000, k=10, dtype="bf16", temperature=4.0, masked=False),
        # three rows over a wide odd vocabulary: few rows, many candidates
        dict(name="top 3x50001 k100 fp16", op="top", rows=3, classes=50001, k=100, dtype="fp16", temperature=1.0, masked=True),
        # the teacher's half of a large token batch
        dict(name="top 2048x131072 k64", op="top", rows=2048, classes=131072, k=64, dtype="bf16", temperature=2.0, masked=False),
        # one image through the ResNet-50 classifier
        dict(name="linear 1x2048x1000", op="linear", rows=1, inner=2048, outer=1000, act="none", residual=False, save=False),
        # every size odd: a projection with its pre-activation kept for the backward pass
        dict(name="linear 333x1021x777 relu", op="linear", rows=333, inner=1021, outer=777, act="relu", residual=True, save=True),
        # the second product of a wide two-layer head, added onto its input
        dict(name="linear 8192x16384x4096 res", op="linear", rows=8192, inner=16384, outer=4096, act="none", residual=True,
             save=False),
        # gradients of the ResNet-50 classifier at the default batch
        dict(name="grads 1536x2048x1000", op="grads", rows=1536, inner=2048, outer=1000, act="none"),
        # gradients of the first product of a wide two-layer head
        dict(name="grads 4096x4096x16384 gelu", op="grads", rows=4096, inner=4096, outer=16384, act="gelu"),
    ]


def _spread(rng, low, high):
    """A whole number between ``low`` and ``high``, even over its logarithm; about half of them odd."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["distill", "top", "linear", "grads"])
    if op in ("distill", "top"):
        classes = _spread(rng, 10, 131072)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        most = (_LARGEST_ROWS if op == "distill" else _LARGEST_SORT) * 2 // _SIZE[dtype]
        rows = _spread(rng, 1, max(1, min(8192, most // classes)))
        k = _spread(rng, 1, min(256, classes))
        case = dict(op=op, rows=rows, classes=classes, k=k, dtype=dtype, temperature=rng.choice([1.0, 2.0, 4.0]),
                    masked=rng.random() < 0.3)
        if op == "distill":
            case.update(alpha=rng.choice([0.3, 0.5, 0.9, 1.0]), tail=rng.random() < 0.5)
        return case
    inner, outer = _spread(rng, 33, 16384), _spread(rng, 10, 16384)
    if rng.random() < 0.6:                   # widths that models have; the others are odd
        inner, outer = (inner + 63) // 64 * 64, (outer + 63) // 64 * 64
    most = _LARGEST_PRODUCT // (1 if op == "linear" else 2)
    rows = _spread(rng, 1, max(1, min(8192, most // (inner * outer))))
    case = dict(op=op, rows=rows, inner=inner, outer=outer, act=rng.choice(["none", "relu", "gelu", "silu"]))
    if op == "linear":
        case.update(residual=rng.random() < 0.5, save=rng.random() < 0.5)
    return case


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)


def _teacher_logits(case, gen):
    """Logits as a trained network gives them: noise, a few classes per row that stand out; masked: the last classes are padding."""
    B, N = case["rows"], case["classes"]
    t = torch.randn(B, N, device="cuda", generator=gen).mul_(2.0)
    for _ in range(3):
        at = torch.randint(0, N, (B, 1), device="cuda", generator=gen)
        t.scatter_add_(1, at, torch.rand(B, 1, device="cuda", generator=gen).mul_(8.0))
    if case["masked"]:
        t[:, N - max(1, N // 100):] = -math.inf
    return t


def prepare(case, seed):
    gen = _generator(seed)
    state = {"case": dict(case)}
    if case["op"] in ("distill", "top"):
        dtype = _TYPES[case["dtype"]]
        B, N, k, T = case["rows"], case["classes"], case["k"], case["temperature"]
        teacher = _teacher_logits(case, gen)
        if case["op"] == "top":
            state["logits"] = teacher.to(dtype)
        else:
            given = teacher.to(dtype)
            values, indices = torch.topk(given, k, dim=1)
            state["lse"] = torch.logsumexp(given.float() / T, dim=1) if case["tail"] else None
            last = N - max(1, N // 100) if case["masked"] else N
            state["labels"] = torch.where(torch.rand(B, device="cuda", generator=gen) < 0.8, indices[:, 0],
                                          torch.randint(0, last, (B,), device="cuda", generator=gen))
            indices = indices.to(torch.int32)
            if case["masked"]:               # padding of short teacher lists, images without a teacher, without a label
                short = torch.rand(B, 1, device="cuda", generator=gen) * 1.25
                gone = torch.arange(k, device="cuda")[None] >= (short * k).ceil()
                gone |= torch.isinf(values)
                values, indices = values.masked_fill(gone, -math.inf), indices.masked_fill(gone, -1)
                state["labels"][torch.rand(B, device="cuda", generator=gen) < 0.1] = -100
            state["values"], state["indices"] = values, indices
            teacher.mul_(0.6).add_(torch.randn(B, N, device="cuda", generator=gen))
            state["logits"] = teacher.to(dtype)
    else:
        M, K, N = case["rows"], case["inner"], case["outer"]

        def tensor(*shape, scale=1.0):
            return torch.randn(*shape, device="cuda", generator=gen).mul_(scale).to(torch.bfloat16)

        state["a"], state["w"] = tensor(M, K), tensor(N, K, scale=K ** -0.5)
        if case["op"] == "linear":
            state["bias"] = torch.randn(N, device="cuda", generator=gen).mul_(0.1)
            state["residual"] = tensor(M, N) if case["residual"] else None
        else:
            state["dy"] = tensor(M, N, scale=1.0 / M)
            state["z"] = tensor(M, N) if case["act"] != "none" else None
    return state


_operators = None


def _ops():
    """The framework's operators for the GPU, looked up once as a program does."""
    global _operators
    if _operators is None:
        from pytorch_distributed_training_amd.ops import get_ops
        _operators = get_ops(torch.device("cuda", torch.cuda.current_device()))
    return _operators


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case, op = state["case"], state["case"]["op"]
    if own:
        ops = _ops()
        if op == "distill":
            return ops.distill_ce(state["logits"], state["labels"], state["values"], state["indices"],
                                  temperature=case["temperature"], alpha=case["alpha"], lse=state["lse"])
        if op == "top":
            return ops.top_logits(state["logits"], case["k"], temperature=case["temperature"])
        if op == "linear":
            y, z = ops.linear_act_fwd(state["a"], state["w"], state["bias"], act=case["act"], residual=state["residual"],
                                      save=case["save"])
            return (y, z) if z is not None else (y,)
        return ops.linear_act_bwd(state["a"], state["w"], state["dy"], z=state["z"], act=case["act"])
    return {"distill": _plain_distill, "top": _plain_top, "linear": _plain_linear, "grads": _plain_grads}[op](state)


def _plain_distill(state):
    case, z, T, alpha = state["case"], state["logits"].float(), state["case"]["temperature"], state["case"]["alpha"]
    B, N = z.shape
    labels, lse = state["labels"], state["lse"]
    values, indices = state["values"].float(), state["indices"].long()
    valid = (indices >= 0) & (indices < N) & (values != -math.inf)
    listed_row = valid.any(dim=1, keepdim=True)
    t = torch.where(valid, values / T, torch.full_like(values, -math.inf))
    if lse is None:
        top = torch.where(listed_row, t.amax(dim=1, keepdim=True), torch.zeros_like(t[:, :1]))
        p = torch.exp(t - top)
        p = torch.where(listed_row, p / p.sum(dim=1, keepdim=True), torch.zeros_like(p))
    else:
        p = torch.exp(t - lse[:, None])
    p = torch.where(valid, p, torch.zeros_like(p))
    at = torch.where(valid, indices, torch.full_like(indices, N))     # column N: a bin for the slots that hold nothing
    P = torch.zeros(B, N + 1, device=z.device).scatter_add_(1, at, p)[:, :N]
    m = z.amax(dim=1, keepdim=True)
    some = m > -math.inf
    m = torch.where(some, m, torch.zeros_like(m))
    e = torch.exp((z - m) / T)
    S = torch.where(some, e.sum(dim=1, keepdim=True), torch.ones_like(m))
    q = e / S
    log_q = (z - m) / T - torch.log(S)
    soft = torch.where(P > 0, P * (torch.log(P) - log_q), torch.zeros_like(P)).sum(dim=1, keepdim=True)
    if lse is None:
        grad = q - P
    else:
        member = torch.zeros(B, N + 1, device=z.device, dtype=torch.bool).scatter_(1, at, True)[:, :N]
        q_rest = torch.where(member, torch.zeros_like(q), q).sum(dim=1, keepdim=True)
        P_rest = (1.0 - p.double().sum(dim=1, keepdim=True)).clamp_min(0.0).float()
        rest = (P_rest > 0) & (q_rest > 0)
        soft = soft + torch.where(rest, P_rest * (torch.log(P_rest) - torch.log(q_rest)), torch.zeros_like(q_rest))
        ratio = torch.where(q_rest > 0, (q_rest - P_rest) / q_rest, torch.zeros_like(q_rest))
        grad = torch.where(member, q - P, q * ratio)
    takes = (listed_row & some).float()
    loss = soft * takes * (alpha * T * T)
    grad = grad * (takes * (alpha * T))
    with_label = (labels >= 0) & (labels < N) & some[:, 0]
    lab = torch.where(with_label, labels, torch.zeros_like(labels))[:, None]
    e1 = torch.exp(z - m)
    S1 = torch.where(some, e1.sum(dim=1, keepdim=True), torch.ones_like(m))
    weight = (1.0 - alpha) * with_label[:, None].float()
    hard = torch.log(S1) + m - z.gather(1, lab)
    loss = loss + torch.where(weight > 0, weight * hard, torch.zeros_like(hard))
    q1 = (e1 / S1).scatter_add_(1, lab, torch.full_like(weight, -1.0))
    grad = grad + q1 * weight
    return loss.double().mean().float(), (grad / B).to(state["logits"].dtype)


def _plain_top(state):
    k, T = state["case"]["k"], state["case"]["temperature"]
    z = state["logits"].float()
    values, indices = torch.sort(z, dim=1, descending=True, stable=True)
    values, indices = values[:, :k], indices[:, :k].to(torch.int32)
    indices = torch.where(values == -math.inf, torch.full_like(indices, -1), indices)
    m = z.amax(dim=1, keepdim=True)
    some = m > -math.inf
    base = torch.where(some, m, torch.zeros_like(m))
    lse = base / T + torch.log(torch.exp((z - base) / T).sum(dim=1, keepdim=True))
    return values.to(state["logits"].dtype), indices, lse[:, 0]


def _plain_act(z, act):
    if act == "relu":
        return z.clamp_min(0.0)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _plain_slope(z, act):
    if act == "relu":
        return (z > 0).float()
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    return torch.ones_like(z)


def _plain_linear(state):
    case = state["case"]
    z = state["a"].float() @ state["w"].float().t() + state["bias"]
    y = _plain_act(z, case["act"])
    if state["residual"] is not None:
        y = y + state["residual"].float()
    if case["save"] and case["act"] != "none":
        return y.to(torch.bfloat16), z.to(torch.bfloat16)
    return (y.to(torch.bfloat16),)


def _plain_grads(state):
    dz = state["dy"].float()
    if state["z"] is not None:
        dz = dz * _plain_slope(state["z"].float(), state["case"]["act"])
    da = dz @ state["w"].float()
    dw = dz.t() @ state["a"].float()
    return da.to(torch.bfloat16), dw.to(torch.bfloat16), dz.double().sum(dim=0).float()


# ------------------------------------------------------------------------------------------------ least work
def work(case):
    if case["op"] in ("distill", "top"):
        B, N, k, s = case["rows"], case["classes"], case["k"], _SIZE[case["dtype"]]
        slots = B * k * (s + 4)
        if case["op"] == "top":
            return {"bytes": B * N * s + slots + 4 * B, "flops": 4 * B * N}
        return {"bytes": 2 * B * N * s + slots + 8 * B + (4 * B if case["tail"] else 0) + 4, "flops": 12 * B * N}
    M, K, N = case["rows"], case["inner"], case["outer"]
    if case["op"] == "linear":
        outs = 1 + int(case["residual"]) + int(case["save"] and case["act"] != "none")
        return {"bytes": 2 * (M * K + N * K + outs * M * N) + 4 * N, "flops": 2 * M * N * K}
    return {"bytes": 2 * (2 * M * K + 2 * N * K + (1 + int(case["act"] != "none")) * M * N) + 4 * N, "flops": 4 * M * N * K}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return {"distill": _exact_distill, "top": _exact_top, "linear": _exact_linear, "grads": _exact_grads}[case["op"]](state)


def _exact_distill(state):
    """On the listed classes alone (those of a row are distinct here): the gradient is a softmax corrected at a few places."""
    case, T, alpha = state["case"], state["case"]["temperature"], state["case"]["alpha"]
    z, labels, lse = state["logits"].double(), state["labels"], state["lse"]
    B, N = z.shape
    t, cols = state["values"].double() / T, state["indices"].long()
    r, s = torch.nonzero((cols >= 0) & (cols < N) & (t != -math.inf), as_tuple=True)
    t, c = t[r, s], cols[r, s]
    scale = torch.zeros(B, dtype=torch.float64, device=z.device).index_fill_(0, r, 1.0)
    if lse is None:
        total = torch.zeros_like(scale).index_add_(0, r, torch.exp(t)).log()
    else:
        total = lse.double()
    log_P = t - total[r]
    P = torch.exp(log_P)
    log_q = torch.log_softmax(z / T, dim=1)
    soft = torch.zeros_like(scale).index_add_(0, r, P * (log_P - log_q[r, c]))
    grad = torch.exp(log_q)
    if lse is not None:
        P_rest = (1.0 - torch.zeros_like(scale).index_add_(0, r, P)).clamp_min(0.0)
        log_q[r, c] = -math.inf
        log_rest = torch.logsumexp(log_q, dim=1)
        some = (log_rest > -math.inf) & (scale > 0)
        soft += torch.where(some & (P_rest > 0), torch.special.xlogy(P_rest, P_rest) - P_rest * log_rest.clamp_min(-1e300), 0.0)
        keep = torch.where(some, 1.0 - P_rest / torch.exp(log_rest).clamp_min(1e-300), 0.0)
        at_listed = grad[r, c]
        grad *= keep[:, None]
        grad[r, c] = at_listed - P
    else:
        grad[r, c] -= P
    del log_q
    grad *= (alpha * T / B) * scale[:, None]
    known = torch.nonzero((labels >= 0) & (labels < N))[:, 0]
    log_p = torch.log_softmax(z, dim=1)
    hard = -log_p[known, labels[known]].sum()
    weight = torch.zeros(B, dtype=torch.float64, device=z.device)
    weight[known] = (1.0 - alpha) / B
    grad += log_p.exp_().mul_(weight[:, None])
    grad[known, labels[known]] -= (1.0 - alpha) / B
    return ((1.0 - alpha) * hard + alpha * T * T * soft.sum()) / B, grad


def _exact_top(state):
    z, k, T = state["logits"].double(), state["case"]["k"], state["case"]["temperature"]
    values, _ = torch.topk(z, k, dim=1)
    return values, None, torch.logsumexp(z / T, dim=1)


def _exact_linear(state):
    case = state["case"]
    z = torch.addmm(state["bias"].double(), state["a"].double(), state["w"].double().t())
    kept = z.clone() if case["save"] and case["act"] != "none" else None
    if case["act"] == "relu":
        z = torch.where(z > 0, z, torch.zeros_like(z))
    elif case["act"] == "gelu":
        z = z * 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
    elif case["act"] == "silu":
        z = z * torch.sigmoid(z)
    if state["residual"] is not None:
        z = z + state["residual"].double()
    return (z, kept) if kept is not None else (z,)


def _exact_grads(state):
    dz, act = state["dy"].double(), state["case"]["act"]
    if act != "none":
        z = state["z"].double()
        if act == "relu":
            dz = torch.where(z > 0, dz, torch.zeros_like(dz))
        elif act == "gelu":
            dz = dz * (0.5 * torch.special.erfc(-z / math.sqrt(2.0)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi))
        else:
            s = torch.sigmoid(z)
            dz = dz * (s + z * s * (1 - s))
    return torch.mm(dz, state["w"].double()), torch.mm(dz.t(), state["a"].double()), dz.sum(dim=0)
