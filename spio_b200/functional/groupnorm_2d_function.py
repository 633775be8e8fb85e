"""The ``spio::groupnorm_2d`` PyTorch operator: group norm over an NCHW tensor in channels_last memory format
with an affine map and an activation, forward and backward.

    z = (x - mean) * rstd * weight + bias,   y = activation(z)

Data is float16, bfloat16 or float32; statistics, weight and bias are fp32.  With ``checkpoint8`` the forward pass
writes the 8-bit form of its input beside the output (see ``checkpoint8_function``) and the backward pass reads that
instead of the input.  The reference has no group norm.  The device work is done by libspio_b200 on torch's
current stream; CPU tensors raise.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from .. import _clib
from ..util.eager import call_on, plain_eager, wants_grad
from .checkpoint8_function import TYPE_CODES, empty_codes, kernel_layout

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}
_CL = torch.channels_last


@lru_cache(maxsize=4096)
def _plan(device_index: int, shape, num_groups: int, dtype, activation: str, eps: float, backward: bool):
    """(reference to the descriptor, scratch bytes) of calls of this size."""
    n, c, h, w = shape
    assert dtype in TYPE_CODES, "expected float16, bfloat16 or float32"
    assert c > 0 and c % 8 == 0, "Number of channels must be a multiple of 8."
    assert num_groups > 0 and c % num_groups == 0, "Number of channels must be divisible by the number of groups."
    assert activation in ACTIVATIONS, f"activation must be one of {', '.join(ACTIVATIONS)}"
    assert eps >= 0, "eps must not be negative"
    desc = ctypes.byref(_clib.GroupNorm2dDesc(n, h * w, c, num_groups, TYPE_CODES[dtype], ACTIVATIONS[activation], eps))
    lib = _clib.load()
    scratch_bytes = lib.spio_groupnorm_2d_bwd_scratch_bytes if backward else lib.spio_groupnorm_2d_fwd_scratch_bytes
    with torch.cuda.device(device_index):
        return desc, max(scratch_bytes(desc), 16)


def _check(t: torch.Tensor, weight, bias) -> None:
    if not t.is_cuda:
        raise ValueError("spio groupnorm_2d runs on CUDA devices only (no CPU implementation)")
    assert t.dim() == 4, "expected an NCHW tensor"
    for v in (weight, bias):
        assert v is None or (v.dtype == torch.float32 and v.numel() == t.shape[1] and v.device == t.device), (
            "weight and bias are fp32 vectors of the channels on the data's device")


def _ptr(t: Optional[torch.Tensor]):
    return t.data_ptr() if t is not None and t.numel() else None


def _absent(like: torch.Tensor, dtype) -> torch.Tensor:
    return like.new_empty((0,), dtype=dtype)


def _vector(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return t if t is None or t.is_contiguous() else t.contiguous()


def _forward(x, weight, bias, num_groups, eps, activation, checkpoint8, want_stats=True):
    """(y, stats or None, codes or None, exponents or None) without torch's dispatcher."""
    _check(x, weight, bias)
    index = x.get_device()
    desc, nbytes = _plan(index, tuple(x.shape), num_groups, x.dtype, activation, eps, False)
    x, weight, bias = kernel_layout(x), _vector(weight), _vector(bias)
    y = torch.empty_like(x)
    stats = torch.empty((x.shape[0], num_groups, 2), device=x.device, dtype=torch.float32) if want_stats else None
    codes, exponents = empty_codes(x) if checkpoint8 else (None, None)
    scratch = torch.empty(nbytes, device=x.device, dtype=torch.uint8)
    _clib.check(call_on(index, _clib.load().spio_groupnorm_2d_fwd, y.data_ptr(), _ptr(stats), _ptr(codes),
                        _ptr(exponents), x.data_ptr(), _ptr(weight), _ptr(bias), desc, scratch.data_ptr(), nbytes),
                "groupnorm_2d")
    return y, stats, codes, exponents


def _backward_kernels(dy, x, codes, exponents, stats, weight, bias, num_groups, activation, needs_input_grad,
                      needs_weight_grad, needs_bias_grad):
    """(dx, dweight, dbias), None for those not asked for, without torch's dispatcher."""
    _check(dy, weight, bias)
    n, c, h, w = dy.shape
    index = dy.get_device()
    desc, nbytes = _plan(index, (n, c, h, w), num_groups, dy.dtype, activation, 0.0, True)
    if x is not None:
        assert x.dtype == dy.dtype and x.shape == dy.shape and x.device == dy.device
        x = kernel_layout(x)
    else:
        assert codes is not None and exponents is not None, "backward needs x or its 8-bit form"
        assert codes.dtype == torch.int8 and codes.shape == dy.shape and codes.device == dy.device
        assert exponents.dtype == torch.uint8 and exponents.device == dy.device
        assert tuple(exponents.shape) == (n, c // 8, h, w), "exponents must be (n, c / 8, h, w)"
        codes, exponents = kernel_layout(codes), kernel_layout(exponents)
    assert stats.dtype == torch.float32 and tuple(stats.shape) == (n, num_groups, 2) and stats.device == dy.device
    dy, stats, weight, bias = kernel_layout(dy), kernel_layout_1d(stats), _vector(weight), _vector(bias)
    dx = torch.empty_like(dy) if needs_input_grad else None
    dw = torch.empty(c, device=dy.device, dtype=torch.float32) if needs_weight_grad else None
    db = torch.empty(c, device=dy.device, dtype=torch.float32) if needs_bias_grad else None
    scratch = torch.empty(nbytes, device=dy.device, dtype=torch.uint8)
    coded = x is None
    _clib.check(call_on(index, _clib.load().spio_groupnorm_2d_bwd, _ptr(dx), _ptr(dw), _ptr(db), dy.data_ptr(),
                        _ptr(x), _ptr(codes) if coded else None, _ptr(exponents) if coded else None,
                        stats.data_ptr(), _ptr(weight), _ptr(bias), desc, scratch.data_ptr(), nbytes),
                "groupnorm_2d backward")
    return dx, dw, db


def kernel_layout_1d(t: torch.Tensor) -> torch.Tensor:
    """``t`` contiguous at a 16-byte boundary."""
    t = _vector(t)
    return t if t.data_ptr() % 16 == 0 else t.clone()


@torch.library.custom_op("spio::groupnorm_2d", mutates_args=())
def groupnorm_2d_op(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], num_groups: int,
                    eps: float, activation: str,
                    checkpoint8: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, stats fp32 [n, groups, 2] = mean and reciprocal standard deviation, codes, exponents); the last two
    are empty without ``checkpoint8``."""
    y, stats, codes, exponents = _forward(x, weight, bias, num_groups, eps, activation, checkpoint8)
    return (y, stats, codes, exponents) if checkpoint8 else (y, stats, _absent(x, torch.int8), _absent(x, torch.uint8))


@groupnorm_2d_op.register_fake
def _groupnorm_2d_fake(x, weight, bias, num_groups, eps, activation, checkpoint8):
    n, c, h, w = x.shape
    cl = torch.channels_last
    return (x.new_empty(x.shape).to(memory_format=cl), x.new_empty((n, num_groups, 2), dtype=torch.float32),
            x.new_empty(x.shape, dtype=torch.int8).to(memory_format=cl) if checkpoint8 else _absent(x, torch.int8),
            x.new_empty((n, c // 8, h, w), dtype=torch.uint8).to(memory_format=cl) if checkpoint8
            else _absent(x, torch.uint8))


@torch.library.custom_op("spio::groupnorm_2d_backward", mutates_args=())
def groupnorm_2d_backward_op(
    grad_output: torch.Tensor, x: Optional[torch.Tensor], codes: Optional[torch.Tensor],
    exponents: Optional[torch.Tensor], stats: torch.Tensor, weight: Optional[torch.Tensor],
    bias: Optional[torch.Tensor], num_groups: int, activation: str, needs_input_grad: bool, needs_weight_grad: bool,
    needs_bias_grad: bool,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(grad_input, grad_weight fp32, grad_bias fp32) from ``x`` or from its 8-bit form; a gradient that was not
    asked for comes back as an empty tensor."""
    grads = _backward_kernels(grad_output, x, codes, exponents, stats, weight, bias, num_groups, activation,
                              needs_input_grad, needs_weight_grad, needs_bias_grad)
    types = (grad_output.dtype, torch.float32, torch.float32)
    return tuple(g if g is not None else _absent(grad_output, t) for g, t in zip(grads, types))


@groupnorm_2d_backward_op.register_fake
def _groupnorm_2d_backward_fake(grad_output, x, codes, exponents, stats, weight, bias, num_groups, activation,
                                needs_input_grad, needs_weight_grad, needs_bias_grad):
    dy, c = grad_output, grad_output.shape[1]
    return (dy.new_empty(dy.shape).to(memory_format=torch.channels_last) if needs_input_grad
            else _absent(dy, dy.dtype),
            dy.new_empty(c if needs_weight_grad else 0, dtype=torch.float32),
            dy.new_empty(c if needs_bias_grad else 0, dtype=torch.float32))


def _setup_context(ctx, inputs, output):
    x, weight, bias, num_groups, _eps, activation, checkpoint8 = inputs
    _y, stats, codes, exponents = output
    ctx.mark_non_differentiable(stats, codes, exponents)
    ctx.checkpoint8 = checkpoint8
    ctx.save_for_backward(*((codes, exponents) if checkpoint8 else (x, None)), stats, weight, bias)
    ctx.num_groups, ctx.activation = num_groups, activation


def _backward(ctx, grad_y, _grad_stats, _grad_codes, _grad_exponents):
    first, second, stats, weight, bias = ctx.saved_tensors
    kept = (None, first, second) if ctx.checkpoint8 else (first, None, None)
    need = ctx.needs_input_grad
    want = (bool(need[0]), bool(need[1]) and weight is not None, bool(need[2]) and bias is not None)
    grads = groupnorm_2d_backward_op(grad_y, *kept, stats, weight, bias, ctx.num_groups, ctx.activation, *want)
    dx, dw, db = (g if w else None for g, w in zip(grads, want))
    return dx, dw, db, None, None, None, None


groupnorm_2d_op.register_autograd(_backward, setup_context=_setup_context)


def _autocast(ks, x, weight, bias, num_groups, eps, activation, checkpoint8):
    """Under CUDA autocast: the data keeps its type, weight and bias are taken in fp32."""
    autocast = torch._C.DispatchKeySet("AutocastCUDA")
    with torch._C._ExcludeDispatchKeyGuard(autocast):
        return torch.ops.spio.groupnorm_2d.default.redispatch(
            ks - autocast, x, weight.to(dtype=torch.float32) if weight is not None else None,
            bias.to(dtype=torch.float32) if bias is not None else None, num_groups, eps, activation, checkpoint8)


_fragment = torch.library.Library("spio", "FRAGMENT")
_fragment.impl("groupnorm_2d", _autocast, "AutocastCUDA", with_keyset=True)


class _GroupNorm2d(torch.autograd.Function):
    """The operator for plain eager calls."""

    @staticmethod
    def forward(ctx, x, weight, bias, num_groups, eps, activation, checkpoint8):
        y, stats, codes, exponents = _forward(x, weight, bias, num_groups, eps, activation, checkpoint8)
        if checkpoint8:
            ctx.save_for_backward(None, codes, exponents, stats, weight, bias)
        else:
            ctx.save_for_backward(x, None, None, stats, weight, bias)
        ctx.num_groups, ctx.activation = num_groups, activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        need = ctx.needs_input_grad
        return *_backward_kernels(grad_y, *ctx.saved_tensors, ctx.num_groups, ctx.activation, need[0], need[1],
                                  need[2]), None, None, None, None


def groupnorm_2d(x: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor] = None,
                 bias: Optional[torch.Tensor] = None, eps: float = 1e-5, activation: str = "none",
                 checkpoint8: bool = False) -> torch.Tensor:
    """``activation(group_norm(x))`` of an NCHW tensor (channels_last on a CUDA device; float16, bfloat16 or
    float32, a multiple of 8 channels).

    ``weight`` and ``bias`` are fp32 vectors of the channels; ``activation`` is ``"none"``, ``"relu"``, ``"silu"`` or
    ``"gelu"`` (with the error function).  ``checkpoint8`` keeps the 8-bit form of ``x`` for the backward pass
    instead of ``x`` (1.125 bytes a value): the gradients are then taken at the restored values, with the
    statistics of ``x`` itself."""
    grad = wants_grad(x, weight, bias)
    # weight and bias of another type: fp32 under autocast, refused otherwise, which the operator knows
    if (plain_eager(x, weight, bias) and (weight is None or weight.dtype == torch.float32)
            and (bias is None or bias.dtype == torch.float32)):
        if grad:
            return _GroupNorm2d.apply(x, weight, bias, num_groups, eps, activation, checkpoint8)
        return _forward(x, weight, bias, num_groups, eps, activation, False, want_stats=False)[0]
    # without a gradient to compute nothing is kept
    return groupnorm_2d_op(x, weight, bias, num_groups, eps, activation, checkpoint8 and grad)[0]
