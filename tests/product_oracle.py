"""The product operators' definitions in 64 bits on the CPU, and how far a kernel may
be from them.

Bounds count roundings: u = eps / 2 of a type is the most that one rounding to it
moves a value, relative to it; FP32 sums of n products are off by n 2^-24 of the sum of
the products' magnitudes at most.
"""
from __future__ import annotations

import torch

U32 = 2.0 ** -24


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def smallest(dtype) -> float:
    """Half of the spacing of the subnormal numbers."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


class CrossEntropy:
    """Losses and gradients of one call, from the definition, and their bounds."""

    def __init__(self, x, weight, targets, bias=None, softcap=None, ignore_index=-100,
                 reduction="mean", grad=None):
        self.dtype = weight.dtype
        dim = x.shape[-1]
        x = x.reshape(-1, dim).double()
        weight, targets = weight.double(), targets.reshape(-1)
        counted = targets != ignore_index
        x = torch.where(counted[:, None], x, 0.0)
        vocab = weight.shape[0]
        z = x @ weight.T
        # FP32 sums of dim products, the bias's addition.
        spread = x.abs() @ weight.abs().T
        if bias is not None:
            z = z + bias.double()
            spread = spread + bias.double().abs()
        z_off = (dim + 2) * U32 * spread
        slope = torch.ones_like(z)
        if softcap:
            root = (1 + (z / softcap).square()).rsqrt()
            z, slope = z * root, root ** 3
        z_off = z_off + 4 * U32 * z.abs()
        z_off = torch.where(z_off.isfinite(), z_off, 0.0)
        at = targets.clamp(0, vocab - 1)
        log_p = torch.log_softmax(z, 1)
        hit = torch.arange(len(at))
        bad = counted & ((targets < 0) | (targets >= vocab))
        losses = torch.where(counted, -log_p[hit, at], 0.0)
        self.losses = torch.where(bad, torch.nan, losses)
        # A loss moves by at most twice what a logit does; its own few roundings.
        most = z_off.amax(1)
        self.losses_off = 2 * most + 16 * U32 * (self.losses.abs() + losses.abs() + 1e-3)
        count = max(1, int(counted.sum()))
        share = counted.double()
        if reduction == "mean":
            share = share / count
        self.total = (self.losses * share).sum()
        self.total_off = (self.losses_off * share).sum() + 2 * U32 * self.total.abs()
        g = torch.ones((), dtype=torch.float64) if grad is None else grad.double().reshape(-1)
        share = share * g
        p = log_p.exp()
        dz = p.clone()
        dz[hit, at] = torch.where(counted, torch.expm1(-losses), 0.0)
        dz = dz * share[:, None] * slope
        dz = torch.where((share == 0)[:, None], 0.0, dz)
        dz = torch.where(bad[:, None], torch.nan, dz)
        # exp turns a difference into a relative one; the slope's cube triples its root's.
        relative = (2 * most + 32 * U32)[:, None] + (8 * z_off if softcap else 0.0)
        dz_off = dz.abs() * relative
        # The target's: exp(-loss) - 1 moves by the loss's difference.
        dz_off[hit, at] += (share.abs() * self.losses_off * p[hit, at]).nan_to_num(0.0)
        self.dz = dz
        self.grad_bias = dz.sum(0)
        self.grad_bias_off = dz_off.sum(0) + (len(at) + 4) * U32 * dz.abs().sum(0) + 1e-37
        u = half_step(self.dtype)
        # Rounded for the products; what FP16 holds 2^14 larger ends at 2^-25 of it, of the
        # largest factor.
        rounded = dz_off + u * dz.abs()
        if self.dtype == torch.float16:
            rounded = rounded + 2.0 ** -38 * share.abs().max()
        self.grad_x = dz @ weight
        off = rounded @ weight.abs() + (vocab + 4) * U32 * (dz.abs() @ weight.abs())
        self.grad_x_off = off * (1 + u) + u * self.grad_x.abs() + smallest(self.dtype)
        self.grad_weight = dz.T @ x
        off = rounded.T @ x.abs() + (len(at) + 4) * U32 * (dz.abs().T @ x.abs())
        self.grad_weight_off = off * (1 + u) + u * self.grad_weight.abs() + smallest(self.dtype)


def assert_within(got, exact, off, name=""):
    got = got.detach().cpu().double().reshape(exact.shape)
    assert torch.equal(got.isnan(), exact.isnan()), f"{name}: NaN in other places"
    infinite = exact.isinf()
    assert torch.equal(got[infinite], exact[infinite]), f"{name}: infinities"
    sure = exact.isfinite()
    far = (got - exact).abs()
    excess = torch.where(far == 0, 0.0, far / off)[sure]
    if excess.numel():
        worst = float(excess.max())
        assert worst <= 1, f"{name}: {worst:.3g} times its bound"


def polar(g, steps, scale=1.0, eps=1e-7):
    """The Newton-Schulz iteration of a matrix or a batch of them, in 64 bits."""
    g = g.double()
    tall = g.shape[-2] > g.shape[-1]
    x = g.mT if tall else g
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        a = x @ x.mT
        x = 2.0 * x + (-1.5 * a + 0.5 * (a @ a)) @ x
    return scale * (x.mT if tall else x)


def polar_off(steps) -> float:
    """How far a result may be, relative to the exact one's Frobenius norm.

    The result is rounded to BF16: 2^-8 of a value at most, evenly spread below that.  A
    step rounds X, A and P to FP16 (u = 2^-11 at most) for its products: with |X|, |A|,
    |P| <= 1 and |dP/dA| <= 1.5 they move it by u of X's norm through P X, by 1.5 u
    through each X of A, 1.5 u through A and 1.5 u through P; evenly spread and
    independent, sqrt(1 + 4 * 1.5^2) u / sqrt(3) together, and later steps do not let it
    grow faster than X.  A half more, since small matrices have few roundings."""
    step = (10.0 / 3) ** 0.5 * 2.0 ** -11
    return 1.5 * ((2.0 ** -8) ** 2 / 3 + steps * step ** 2) ** 0.5


def polar_floor(steps, values) -> float:
    """The same in absolute terms, of a matrix so small (against eps) that X's numbers are
    FP16's smallest: X times 2^10 is held to half of their spacing, 2^-25, and a step at most
    doubles what the steps before have left: 2^-35 (1 + 2 + .. + 2^steps) a value."""
    return values ** 0.5 * 2.0 ** (steps + 1 - 35)


def polar_rest_floor(steps, values) -> float:
    """:func:`polar_floor` with what the second number of X holds: that is 2^11 larger than the
    first, so half of the spacing of its smallest is 2^-46 of X."""
    return polar_floor(steps, values) * 2.0 ** -11


def polar_off_in_empty_directions(steps, rows) -> float:
    """What a matrix of rank 1 may be off beside :func:`polar_off`, relative to the norm: in
    directions that it does not have, what a step rounds is doubled by each step after it.

    A step's sums of `rows` products (FP32, 16 at a time) are off by 2^-23 of what they have
    come to, half of 1.2 |X| on average, each time; adding 2 X and X's two numbers round by
    2^-24 and 2^-23 of 2 |X| and |X|: ((rows / 16 + 1) 0.6 + 2) 2^-23 of |X| = 1 at most.
    Steps are independent: sqrt(4^steps + 4^(steps - 1) + ..) = 1.16 2^steps of that."""
    return 1.16 * 2.0 ** steps * ((rows / 16 + 1) * 0.6 + 2) * 2.0 ** -23
