"""The ``spio::groupnorm_2d`` PyTorch operator: group norm over an NCHW tensor in channels_last memory format
with an affine map and an activation, forward and backward.

    z = (x - mean) * rstd * weight + bias,   y = activation(z)

Data is float16, bfloat16 or float32; statistics are fp32, weight and bias too or of the data's type.  With ``checkpoint8`` the forward pass
writes the 8-bit form of its input beside the output (see ``checkpoint8_function``) and the backward pass reads that
instead of the input.  The reference has no group norm.  The device work is done by libspio_b200 on torch's
current stream; CPU tensors raise.
"""

from __future__ import annotations

from typing import Optional

import torch

from .. import _clib

ACTIVATIONS = ("none", "relu", "silu", "gelu")

_fragment = torch.library.Library("spio", "FRAGMENT")
# The operator of groupnorm_2d() below, differentiable in x, weight and bias.
_fragment.define("groupnorm_2d(Tensor x, Tensor? weight, Tensor? bias, int num_groups, float eps, str activation, "
                 "bool checkpoint8) -> Tensor")
# (y, stats fp32 [n, groups, 2] = mean and reciprocal standard deviation, codes, exponents); the last two are empty
# without checkpoint8.
_fragment.define("groupnorm_2d_forward(Tensor x, Tensor? weight, Tensor? bias, int num_groups, float eps, "
                 "str activation, bool checkpoint8) -> (Tensor, Tensor, Tensor, Tensor)")
# (grad_input, grad_weight fp32, grad_bias fp32) from x or from its 8-bit form; a gradient that was not asked for
# comes back as an empty tensor.
_fragment.define("groupnorm_2d_backward(Tensor grad_output, Tensor? x, Tensor? codes, Tensor? exponents, Tensor stats, "
                 "Tensor? weight, Tensor? bias, int num_groups, str activation, bool needs_input_grad, "
                 "bool needs_weight_grad, bool needs_bias_grad) -> (Tensor, Tensor, Tensor)")
_clib.load_torch_ops_if_usable()

groupnorm_2d_op = torch.ops.spio.groupnorm_2d_forward
groupnorm_2d_backward_op = torch.ops.spio.groupnorm_2d_backward
_groupnorm_2d = torch.ops.spio.groupnorm_2d.default


@torch.library.register_fake("spio::groupnorm_2d")
def _groupnorm_2d_fake(x, weight, bias, num_groups, eps, activation, checkpoint8):
    return x.new_empty(x.shape).to(memory_format=torch.channels_last)


@torch.library.register_fake("spio::groupnorm_2d_forward")
def _groupnorm_2d_forward_fake(x, weight, bias, num_groups, eps, activation, checkpoint8):
    n, c, h, w = x.shape
    cl = torch.channels_last
    kept = ((x.new_empty(x.shape, dtype=torch.int8).to(memory_format=cl),
             x.new_empty((n, c // 8, h, w), dtype=torch.uint8).to(memory_format=cl)) if checkpoint8
            else (x.new_empty((0,), dtype=torch.int8), x.new_empty((0,), dtype=torch.uint8)))
    return (x.new_empty(x.shape).to(memory_format=cl), x.new_empty((n, num_groups, 2), dtype=torch.float32), *kept)


@torch.library.register_fake("spio::groupnorm_2d_backward")
def _groupnorm_2d_backward_fake(grad_output, x, codes, exponents, stats, weight, bias, num_groups, activation,
                                needs_input_grad, needs_weight_grad, needs_bias_grad):
    dy, c = grad_output, grad_output.shape[1]
    return (dy.new_empty(dy.shape).to(memory_format=torch.channels_last) if needs_input_grad else dy.new_empty((0,)),
            dy.new_empty(c if needs_weight_grad else 0, dtype=torch.float32),
            dy.new_empty(c if needs_bias_grad else 0, dtype=torch.float32))


def groupnorm_2d(x: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor] = None,
                 bias: Optional[torch.Tensor] = None, eps: float = 1e-5, activation: str = "none",
                 checkpoint8: bool = False) -> torch.Tensor:
    """``activation(group_norm(x))`` of an NCHW tensor (channels_last on a CUDA device; float16, bfloat16 or
    float32, a multiple of 8 channels).

    ``weight`` and ``bias`` are vectors of the channels, both fp32 or both of the data's type (of any type under
    autocast, where the data keeps its own); they are taken in fp32, and their gradients are rounded once.  ``activation`` is ``"none"``, ``"relu"``, ``"silu"`` or ``"gelu"`` (with the error function).  A group, rounded
    up to whole blocks of 8 channels, may span at most 2048 channels.  ``checkpoint8`` keeps the 8-bit form of
    ``x`` for the backward pass instead of ``x`` (1.125 bytes a value): the gradients are then taken at the
    restored values, with the statistics of ``x`` itself."""
    _clib.load_torch_ops()
    return _groupnorm_2d(x, weight, bias, num_groups, eps, activation, checkpoint8)
