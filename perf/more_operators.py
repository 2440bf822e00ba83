"""Performance cases of the training step's operators that are made of matrix
products: the cross entropy of a projection onto a large vocabulary, and Muon's
orthogonalisation, each in its plain form and as the framework's kernels.

* ``loss``: the mean or sum of the tokens' cross entropies and the gradients of the
  hidden states, the projection and its bias.
* ``score``: each token's cross entropy, no gradients.
* ``polar``: the Newton-Schulz iteration on a batch of matrices.

A case is a dict of plain values.  ``own`` picks the side that ``run`` takes.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
_IGNORED = -100
_A, _B, _C = 2.0, -1.5, 0.5      # X <- a X + (b A + c A^2) X with A = X X^T
_EPS = 1e-7


def listed() -> list:
    return [
        # The trainer's step: 8 sequences of 1024 against its padded vocabulary,
        # soft-capped, FP32 bias, summed.
        {"name": "loss_8192x50304x768", "kind": "loss", "tokens": 8192, "vocab": 50304,
         "dim": 768, "softcap": 15.0, "bias": True, "ignored": 0.0, "reduction": "sum",
         "dtype": "bf16"},
        # Fine-tuning: an odd vocabulary, a ragged number of tokens, prompts that do not
        # count, FP16.
        {"name": "loss_1013x50257x1024", "kind": "loss", "tokens": 1013, "vocab": 50257,
         "dim": 1024, "softcap": 0.0, "bias": False, "ignored": 0.3, "reduction": "mean",
         "dtype": "fp16"},
        # A large model's step.
        {"name": "loss_16384x100352x2048", "kind": "loss", "tokens": 16384, "vocab": 100352,
         "dim": 2048, "softcap": 0.0, "bias": False, "ignored": 0.1, "reduction": "mean",
         "dtype": "bf16"},
        # A test's or a toy model's step: latency counts.
        {"name": "loss_37x307x72", "kind": "loss", "tokens": 37, "vocab": 307, "dim": 72,
         "softcap": 15.0, "bias": True, "ignored": 0.1, "reduction": "mean", "dtype": "bf16"},
        # Serving: the log-probability of one token of the small model.
        {"name": "score_1x50304x768", "kind": "score", "tokens": 1, "vocab": 50304, "dim": 768,
         "softcap": 15.0, "bias": True, "ignored": 0.0, "dtype": "bf16"},
        # Evaluation of a long text by a wide model.
        {"name": "score_4095x32000x4096", "kind": "score", "tokens": 4095, "vocab": 32000,
         "dim": 4096, "softcap": 0.0, "bias": False, "ignored": 0.0, "dtype": "bf16"},
        # The trainer's step: its 48 square block matrices, 12 iterations.
        {"name": "polar_48x768x768", "kind": "polar", "count": 48, "rows": 768, "cols": 768,
         "steps": 12, "dtype": "bf16"},
        # A wider model's projections, four times as tall as wide.
        {"name": "polar_16x4096x1024", "kind": "polar", "count": 16, "rows": 4096, "cols": 1024,
         "steps": 5, "dtype": "bf16"},
        # The largest: one matrix of a large model, FP32 gradients.
        {"name": "polar_1x4096x11008", "kind": "polar", "count": 1, "rows": 4096, "cols": 11008,
         "steps": 5, "dtype": "fp32"},
        # One matrix of the trainer's width: little parallel work.
        {"name": "polar_1x768x768", "kind": "polar", "count": 1, "rows": 768, "cols": 768,
         "steps": 5, "dtype": "bf16"},
        # Odd sizes, FP16, tall.
        {"name": "polar_5x1021x333", "kind": "polar", "count": 5, "rows": 1021, "cols": 333,
         "steps": 10, "dtype": "fp16"},
        # Small matrices of a test or a toy model.
        {"name": "polar_8x96x160", "kind": "polar", "count": 8, "rows": 96, "cols": 160,
         "steps": 5, "dtype": "bf16"},
    ]


def _log_uniform(rng, low: float, high: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    while True:
        kind = rng.choice(["loss", "loss", "score", "polar", "polar"])
        if kind == "polar":
            case = {"kind": kind, "count": _log_uniform(rng, 1, 48),
                    "rows": _log_uniform(rng, 16, 8192), "cols": _log_uniform(rng, 16, 8192),
                    "steps": rng.choice([3, 5, 5, 6, 8, 10, 12]),
                    "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
            if rng.random() < 0.5:
                case.update(rows=-(-case["rows"] // 64) * 64, cols=-(-case["cols"] // 64) * 64)
            if (work(case)["flops"] <= 2e12
                    and case["count"] * case["rows"] * case["cols"] <= 1 << 26):
                return case
            continue
        case = {"kind": kind, "tokens": _log_uniform(rng, 1, 16384),
                "vocab": _log_uniform(rng, 64, 131072), "dim": _log_uniform(rng, 16, 4096),
                "softcap": rng.choice([0.0, 0.0, 15.0, 30.0]), "bias": rng.random() < 0.5,
                "ignored": rng.choice([0.0, 0.1, 0.5]),
                "dtype": rng.choice(["bf16", "bf16", "fp16"])}
        if case["tokens"] < 32:       # of a few, all might be ignored
            case["ignored"] = 0.0
        if rng.random() < 0.75:
            case["dim"] = -(-case["dim"] // 8) * 8
        if kind == "loss":
            case["reduction"] = rng.choice(["mean", "sum"])
        if (case["tokens"] * case["vocab"] * case["dim"] <= 1.5e12
                and case["tokens"] * case["vocab"] <= 1.2e9):
            return case


def work(case: dict) -> dict:
    size = _SIZES[case["dtype"]]
    if case["kind"] == "polar":
        r, c = sorted((case["rows"], case["cols"]))
        # A step: X X^T and A A are symmetric, half of each is enough; P X is whole.
        flops = case["count"] * case["steps"] * (r * r * c + r * r * r + 2 * r * r * c)
        return {"bytes": case["count"] * r * c * (size + 2), "flops": flops}
    n, v, d = case["tokens"], case["vocab"], case["dim"]
    inputs = (n * d + v * d) * size + 8 * n + (4 * v if case["bias"] else 0)
    if case["kind"] == "score":
        return {"bytes": inputs + 4 * n, "flops": 2 * n * v * d}
    # Outputs: the gradients, of the inputs' sizes.
    return {"bytes": 2 * inputs - 8 * n + 4, "flops": 6 * n * v * d}


# ---- inputs


def _generator(seed: int, stream: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed * 64 + stream)


def _normal(shape, seed: int, stream: int) -> torch.Tensor:
    return torch.randn(shape, generator=_generator(seed, stream), device="cuda")


def _gradients(case: dict, seed: int) -> torch.Tensor:
    """Matrices whose singular values fall off as those of gradients do: a few
    strong directions over a broad rest."""
    count, rows, cols = case["count"], case["rows"], case["cols"]
    rank = min(rows, cols)
    fall = (1 + torch.arange(rank, device="cuda") / 16.0) ** -0.75
    left = _normal((count, rows, rank), seed, 0) * fall
    return 1e-3 / math.sqrt(rank) * torch.bmm(left, _normal((count, rank, cols), seed, 1))


def prepare(case: dict, seed: int) -> dict:
    dtype = _DTYPES[case["dtype"]]
    state = {"case": case}
    if case["kind"] == "polar":
        state["g"] = _gradients(case, seed).to(dtype)
        return state
    n, v, d = case["tokens"], case["vocab"], case["dim"]
    # Logits of a spread of about 2; half of the tokens are well predicted.
    weight = _normal((v, d), seed, 1) * (2.0 / math.sqrt(d))
    targets = torch.randint(0, v, (n,), generator=_generator(seed, 2), device="cuda")
    x = _normal((n, d), seed, 0)
    x[::2] += 3.0 * weight[targets[::2]]
    if case["ignored"]:
        drop = torch.rand(n, generator=_generator(seed, 3), device="cuda") < case["ignored"]
        targets[drop] = _IGNORED
    state.update(x=x.to(dtype), weight=weight.to(dtype), targets=targets,
                 bias=0.5 * _normal((v,), seed, 4) if case["bias"] else None)
    return state


# ---- the framework's operators


def _run_own(state: dict) -> dict:
    case = state["case"]
    if case["kind"] == "polar":
        from losslessly_compressed_tensors_amd.components.orthogonal import orthogonalize
        return {"out": orthogonalize(state["g"], case["steps"])}
    from losslessly_compressed_tensors_amd.components.losses import linear_cross_entropy

    how = {"softcap": case["softcap"] or None, "ignore_index": _IGNORED}
    if case["kind"] == "score":
        with torch.no_grad():
            return {"losses": linear_cross_entropy(state["x"], state["weight"], state["targets"],
                                                   state["bias"], reduction="none", **how)}
    x, weight = state["x"].detach().requires_grad_(), state["weight"].detach().requires_grad_()
    leaves, bias = [x, weight], state["bias"]
    if bias is not None:
        bias = bias.detach().requires_grad_()
        leaves.append(bias)
    loss = linear_cross_entropy(x, weight, state["targets"], bias, reduction=case["reduction"],
                                **how)
    grads = torch.autograd.grad(loss, leaves)
    return dict(zip(("loss", "grad_x", "grad_weight", "grad_bias"), (loss.detach(), *grads)))


# ---- the plain forms


def _plain_polar(state: dict) -> dict:
    case = state["case"]
    g = state["g"].float()
    tall = case["rows"] > case["cols"]
    x = g.transpose(1, 2).contiguous() if tall else g
    x = x / (x.square().sum((1, 2), keepdim=True, dtype=torch.float64).sqrt() + _EPS).float()
    for _ in range(case["steps"]):
        gram = torch.bmm(x, x.transpose(1, 2).contiguous())
        x = _A * x + torch.bmm(_B * gram + _C * torch.bmm(gram, gram), x)
    if tall:
        x = x.transpose(1, 2).contiguous()
    return {"out": x.to(torch.bfloat16)}


def _plain_loss(state: dict) -> dict:
    case, targets, bias = state["case"], state["targets"], state["bias"]
    x, weight = state["x"].float(), state["weight"].float()
    logits = x @ weight.T
    if bias is not None:
        logits = logits + bias
    slope = None
    if case["softcap"]:
        slope = (1 + (logits / case["softcap"]).square()).rsqrt()
        logits = logits * slope
    # The loss is log(1 + the others' weights over the target's), in 64 bits: of a well
    # predicted token it is far smaller than the logits that it is the difference of.
    counted = targets != _IGNORED
    at = targets.clamp(min=0).unsqueeze(1)
    hit = logits.gather(1, at)
    most = logits.amax(1, keepdim=True)
    others = (logits - most).exp().scatter(1, at, 0.0).sum(1, keepdim=True).double()
    loss = (others * (most - hit).double().exp()).log1p()
    losses = torch.where(counted, loss.squeeze(1), 0.0)
    if case["kind"] == "score":
        return {"losses": losses.float()}
    factor = counted.float()
    if case["reduction"] == "mean":
        factor = factor / counted.sum().clamp(min=1)
    grad = (logits - (hit.double() + loss).float()).exp()
    grad = grad.scatter(1, at, torch.expm1(-loss).float()) * factor.unsqueeze(1)
    if slope is not None:
        grad = grad * slope * slope * slope
    out = {"loss": (losses * factor.double()).sum().float(),
           "grad_x": (grad @ weight).to(state["x"].dtype),
           "grad_weight": (grad.T @ x).to(state["weight"].dtype)}
    if bias is not None:
        out["grad_bias"] = grad.sum(0, dtype=torch.float64).to(bias.dtype)
    return out


def run(state: dict) -> dict:
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _plain_polar(state) if state["case"]["kind"] == "polar" else _plain_loss(state)


# ---- the definitions in 64 bits


def _exact_polar(state: dict) -> dict:
    """The product of the steps' polynomials of M = X X^T, which all commute, times X."""
    g = state["g"].double()
    tall = state["case"]["rows"] > state["case"]["cols"]
    if tall:
        g = g.mT.contiguous()
    out = []
    for matrix in g.unbind(0):
        start = matrix / (torch.linalg.vector_norm(matrix) + _EPS)
        square = start @ start.mT
        one = torch.eye(square.shape[0], dtype=torch.float64, device=square.device)
        total = one
        for _ in range(state["case"]["steps"]):
            factor = _A * one + _B * square + _C * (square @ square)
            total = factor @ total
            square = factor @ square @ factor
        out.append(total @ start)
    out = torch.stack(out)
    return {"out": out.mT.contiguous() if tall else out}


def _exact_loss(state: dict) -> dict:
    """Row by row in pieces: the softmax's definition and the chain rule."""
    case, targets = state["case"], state["targets"]
    n, cap = case["tokens"], case["softcap"]
    weight = state["weight"].double()
    counted = (targets != _IGNORED).double()
    share = counted / counted.sum().clamp(min=1) if case.get("reduction") == "mean" else counted
    losses, grad_x = [], []
    grad_weight = torch.zeros_like(weight)
    grad_bias = weight.new_zeros(case["vocab"])
    piece = max(1, 2 ** 28 // case["vocab"])
    for first in range(0, n, piece):
        rows = slice(first, min(n, first + piece))
        x = state["x"][rows].double()
        z = torch.nn.functional.linear(x, weight,
                                       None if state["bias"] is None else state["bias"].double())
        slope = 1.0
        if cap:
            root = torch.sqrt(z * z + cap * cap)
            z, slope = cap * z / root, (cap / root) ** 3
        hit = targets[rows].clamp(min=0)
        at = torch.arange(len(hit), device=hit.device)
        log_p = torch.log_softmax(z, 1)
        losses.append(-log_p[at, hit] * counted[rows])
        if case["kind"] == "score":
            continue
        p = log_p.exp_()
        p[at, hit] -= 1.0
        p *= share[rows, None]
        p *= slope
        grad_x.append(p @ weight)
        grad_weight += p.mT @ x
        grad_bias += p.sum(0)
    losses = torch.cat(losses)
    if case["kind"] == "score":
        return {"losses": losses}
    out = {"loss": (losses * share).sum(), "grad_x": torch.cat(grad_x),
           "grad_weight": grad_weight}
    if state["bias"] is not None:
        out["grad_bias"] = grad_bias
    return out


def exact(case: dict, seed: int):
    # More than 20 seconds at the 30 TFLOP/s of large products in 64 bits.
    products = work(case)["flops"] * (2.0 if case["kind"] == "polar" else 1.0)
    if products > 2e14:
        return None
    state = prepare(case, seed)
    with torch.no_grad():
        return _exact_polar(state) if case["kind"] == "polar" else _exact_loss(state)
