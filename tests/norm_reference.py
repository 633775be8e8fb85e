"""The group norm with an activation and the 8-bit blocks, computed by their definition in float64, with the
error that fp32 arithmetic and one rounding to the data's type may leave.

Error model.  Half a step of the output's type, plus CONST * 2^-24 times the magnitudes that enter a sum: fp32
sums are taken over at most a few hundred terms a thread and then pairwise, so their relative error stays
within some tens of 2^-24 of the sum of magnitudes, and an element-wise formula rounds about ten times; the
16-bit types' activations add 1.5e-7 (2.5 * 2^-24) times their argument.  CONST = 64 covers both.

The mean enters with mean |x| of its group and not with |mean|: a sum of n values in fp32 rounds partial sums of
up to sum |x|, so its error is of the order 2^-24 * mean |x| after the division by n, in any order of summation, while
|mean| may be as small as the values happen to cancel.  (Six pixels of three channels with values around 1 and a
mean of 0.02: four roundings of partial sums near 1 are 4 * 2^-24 = 2.4e-7, above 64 * 2^-24 * 0.045 = 1.7e-7.)
"""

import ctypes

import torch

from spio_b200 import _clib

CONST = 64 * 2.0 ** -24

B200 = (148, 232448)  # multiprocessors, bytes of shared memory that a CTA may have

# Sizes for which the planner takes a certain launch on a B200: (n, c, h, w), groups, type, activation, and the forms of the
# forward pass, the forward pass that writes codes, the backward pass and the backward pass from codes: one launch or
# two, `n` where the image's last slab of channels is narrower than the others.
PLANNED = [
    ((2, 24, 66, 55), 12, torch.float16, "relu", "1n 1n 1n 1n"),
    ((4, 24, 42, 42), 3, torch.bfloat16, "relu", "1n 1n 1n 1n"),
    ((3, 72, 28, 30), 9, torch.float32, "none", "1n 1n 1n 1n"),
    ((1, 216, 42, 22), 108, torch.float32, "none", "1n 1n 1n 1n"),
    ((1, 72, 81, 112), 6, torch.float16, "none", "1 1 2n 2n"),
    ((1, 72, 118, 123), 36, torch.bfloat16, "relu", "1n 1n 2n 2n"),
    ((1, 696, 35, 32), 6, torch.float32, "gelu", "2n 2n 2n 2n"),
    ((1, 600, 39, 38), 3, torch.float32, "gelu", "2n 2n 2n 2n"),
    ((1, 600, 48, 60), 24, torch.bfloat16, "gelu", "2n 2n 2n 2n"),
    ((1, 72, 127, 166), 24, torch.bfloat16, "none", "2n 2n 2 2"),
    ((1, 624, 59, 65), 3, torch.float16, "silu", "2n 2n 2 2"),
    ((1, 744, 16, 15), 1, torch.float32, "gelu", "1 2 2 2"),
    ((3, 568, 28, 21), 4, torch.bfloat16, "silu", "1 2 2 2"),
    ((1, 40, 141, 178), 20, torch.float16, "silu", "1 2 2 2"),
    ((1, 712, 16, 11), 4, torch.float32, "silu", "1 1 2 1"),
    ((3, 24, 117, 119), 24, torch.bfloat16, "silu", "1n 1n 2 1n"),
    ((4, 280, 63, 32), 10, torch.float32, "none", "1 1 1 2"),
]


def plan_of(shape, groups, dtype, act, backward=False, coded=False):
    """What the library launches for these sizes on a B200."""
    n, c, h, w = shape
    types, acts = [torch.float16, torch.bfloat16, torch.float32], ["none", "relu", "silu", "gelu"]
    desc = _clib.GroupNorm2dDesc(n, h * w, c, groups, types.index(dtype), acts.index(act), 1e-5)
    info = _clib.GroupNorm2dPlanInfo()
    _clib.check(_clib.load().spio_groupnorm_2d_plan_for(ctypes.byref(desc), backward, coded, *B200, ctypes.byref(info)),
                "plan")
    return info.as_dict()


def half_step(t: torch.Tensor, dtype) -> torch.Tensor:
    """Largest rounding error of the float64 values ``t`` when stored as ``dtype``."""
    info = torch.finfo(dtype)
    return torch.clamp(t.abs() * (info.eps / 2), min=info.smallest_normal * info.eps / 2)


def blocks_of(x: torch.Tensor):
    """(codes int64 (n, c, h, w), scale float64 (n, c / 8, h, w)) of finite ``x``, by the definition."""
    top = torch.finfo(x.dtype).max
    v = x.detach().double().cpu().unflatten(1, (-1, 8))
    largest = v.abs().amax(2, keepdim=True)
    mantissa, exponent = torch.frexp(largest)              # largest = mantissa * 2^exponent, in [0.5, 1)
    k = exponent - 7 + (mantissa * 128 >= 127.5)           # the largest code is 127 at most
    k = torch.where(largest > 0, k, -126).clamp(min=-126).double()
    scale = torch.exp2(k)
    limit = torch.floor(top / scale)
    codes = torch.clamp(torch.round(v / scale), -limit, limit)
    return codes.flatten(1, 2).long(), scale.squeeze(2)


def restored(x: torch.Tensor) -> torch.Tensor:
    """float64 values of the 8-bit form of ``x``."""
    codes, scale = blocks_of(x)
    return codes.double() * scale.repeat_interleave(8, 1)


def _act(z, act):
    if act == "relu":
        return torch.relu(z)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return z * 0.5 * torch.erfc(-z * 0.5 ** 0.5)
    return z


def _slope(z, act):
    if act == "relu":
        return (z > 0).double()
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return 0.5 * torch.erfc(-z * 0.5 ** 0.5) + z * torch.exp(-z * z / 2) * (2 * torch.pi) ** -0.5
    return torch.ones_like(z)


class Reference:
    """float64 results and the error each output may have (``*_tol``)."""

    def __init__(self, x, groups, weight=None, bias=None, eps=1e-5, act="none", dy=None, checkpoint8=False):
        dtype = x.dtype
        n, c, h, w = x.shape
        wide = lambda t: t.reshape(n, groups, 1).expand(n, groups, c // groups).reshape(n, c, 1, 1)  # noqa: E731
        v = x.detach().double().cpu()
        wt = weight.detach().double().cpu() if weight is not None else torch.ones(c, dtype=torch.float64)
        bs = bias.detach().double().cpu() if bias is not None else torch.zeros(c, dtype=torch.float64)
        wt, bs = wt.reshape(1, c, 1, 1), bs.reshape(1, c, 1, 1)
        grouped = v.reshape(n, groups, -1)
        self.mean, var = grouped.mean(2), grouped.var(2, unbiased=False)
        self.rstd = (var + eps).rsqrt()
        mean, rstd = wide(self.mean), wide(self.rstd)
        z = (v - mean) * rstd * wt + bs
        # rounding of x - mean, of the products and of the statistics
        size = wide(grouped.abs().mean(2))                     # mean |x| of the group
        z_mag = (v.abs() + size) * rstd * wt.abs() + bs.abs()
        self.y = _act(z, act)
        self.y_tol = half_step(self.y, dtype) + CONST * z_mag
        if dy is None:
            return
        if checkpoint8:
            v = restored(x)
            z = (v - mean) * rstd * wt + bs
            z_mag = (v.abs() + size) * rstd * wt.abs() + bs.abs()
        g0 = dy.detach().double().cpu()
        hat, hat_mag = (v - mean) * rstd, (v.abs() + size) * rstd
        g = g0 * _slope(z, act)
        # the slopes' own slope is at most 1.2; ReLU's jumps, so a value next to zero may go either way
        g_tol = g0.abs() * CONST * (1 + 1.2 * z_mag * (act != "none") * (act != "relu"))
        if act == "relu":
            g_tol = g_tol + g0.abs() * (z.abs() <= CONST * z_mag)
        self.dbias = g.sum((0, 2, 3))
        self.dbias_tol = (g_tol + CONST * g.abs()).sum((0, 2, 3))
        self.dweight = (g * hat).sum((0, 2, 3))
        self.dweight_tol = (g_tol * hat_mag + CONST * g.abs() * hat_mag).sum((0, 2, 3))
        per_group = lambda t: wide(t.reshape(n, groups, -1).mean(2))  # noqa: E731
        s1, s2 = per_group(g * wt), per_group(g * wt * hat)
        e = g_tol + CONST * g.abs()
        s1_tol = per_group(e * wt.abs()) + CONST * per_group((g * wt).abs())
        s2_tol = per_group((e + CONST * g.abs()) * wt.abs() * hat_mag)
        self.dx = rstd * (g * wt - s1 - hat * s2)
        self.dx_tol = half_step(self.dx, dtype) + rstd * (
            e * wt.abs() + s1_tol + hat_mag * (s2_tol + CONST * s2.abs()) + CONST * (g * wt).abs())


def assert_within(got, want, tol, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= tol)      # a NaN is bad
    if bad.any():
        i = int(((got - want).abs() / tol).nan_to_num(nan=float("inf")).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values off, the worst at {i}: "
                             f"{got.flatten()[i]} for {want.flatten()[i]} +- {tol.flatten()[i]}")
