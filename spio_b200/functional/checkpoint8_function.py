"""Activation checkpoints in 8 bits: ``spio::checkpoint8_pack`` / ``spio::checkpoint8_unpack``, and the
group-width-8 convolution that keeps its input in that form for the backward pass.

A block of 8 consecutive channels of a pixel -- one channel group of the gw8 convolution -- becomes 8 signed
codes and one exponent byte and stands for ``code * 2**(exponent - 127)``: 1.125 bytes a value.  The scale is
the smallest power of two (``2**-126`` at least) for which the block's largest magnitude rounds to at most 127,
so a restored value is off by at most half a step, 1/127 of the block's largest magnitude.  (Where rounding up
would leave the range of the type, codes stop at 63 and the error is up to 1/64 of that magnitude.)  A block with an infinity or a NaN
is restored as NaN, so that a gradient scaler still finds it.

The reference keeps the convolution's input as it is (spio/functional/conv2d_gw8_function.py:150-171); this
form has no counterpart there.  The device work is done by libspio_b200 on torch's current stream; CPU tensors
raise.
"""

from __future__ import annotations

from functools import partial
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from .. import _clib
from ..util.eager import call_on, plain_eager
from ..util.tensor_format import to_channels_last
from .conv2d_gw8_function import backward_kernels, conv2d_gw8, conv2d_gw8_backward_op, forward_kernels

TYPE_CODES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_CL = torch.channels_last


def kernel_layout(t: torch.Tensor) -> torch.Tensor:
    """``t`` in channels_last order at a 16-byte boundary (itself if it is already)."""
    if not t.is_contiguous(memory_format=_CL):
        t = t.contiguous(memory_format=_CL)
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=_CL)


def _check_image(x: torch.Tensor, what: str) -> None:
    if not x.is_cuda:
        raise ValueError(f"spio {what} runs on CUDA devices only (no CPU implementation)")
    assert x.dim() == 4, "expected an NCHW tensor"


def empty_codes(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Unset codes and exponents for ``x``."""
    n, c, h, w = x.shape
    return (torch.empty((n, c, h, w), device=x.device, dtype=torch.int8, memory_format=_CL),
            torch.empty((n, c // 8, h, w), device=x.device, dtype=torch.uint8, memory_format=_CL))


def _pack(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    _check_image(x, "checkpoint8_pack")
    assert x.dtype in TYPE_CODES, "expected float16, bfloat16 or float32"
    assert x.shape[1] % 8 == 0, "Number of channels must be a multiple of 8."
    x = kernel_layout(x)
    codes, exponents = empty_codes(x)
    _clib.check(call_on(x.get_device(), _clib.load().spio_checkpoint8_pack, codes.data_ptr(), exponents.data_ptr(),
                        x.data_ptr(), x.numel() // 8, TYPE_CODES[x.dtype]), "checkpoint8_pack")
    return codes, exponents


def _unpack(codes: torch.Tensor, exponents: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    _check_image(codes, "checkpoint8_unpack")
    assert dtype in TYPE_CODES, "expected float16, bfloat16 or float32"
    assert codes.dtype == torch.int8 and exponents.dtype == torch.uint8
    assert codes.device == exponents.device
    n, c, h, w = codes.shape
    assert c % 8 == 0 and tuple(exponents.shape) == (n, c // 8, h, w), "exponents must be (n, c / 8, h, w)"
    x = torch.empty((n, c, h, w), device=codes.device, dtype=dtype, memory_format=_CL)
    codes, exponents = kernel_layout(codes), to_channels_last(exponents)
    _clib.check(call_on(codes.get_device(), _clib.load().spio_checkpoint8_unpack, x.data_ptr(), codes.data_ptr(),
                        exponents.data_ptr(), codes.numel() // 8, TYPE_CODES[dtype]), "checkpoint8_unpack")
    return x


@torch.library.custom_op("spio::checkpoint8_pack", mutates_args=())
def checkpoint8_pack_op(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(codes, exponents) of an NCHW tensor."""
    return _pack(x)


@checkpoint8_pack_op.register_fake
def _checkpoint8_pack_fake(x):
    n, c, h, w = x.shape
    return (x.new_empty(x.shape, dtype=torch.int8).to(memory_format=torch.channels_last),
            x.new_empty((n, c // 8, h, w), dtype=torch.uint8).to(memory_format=torch.channels_last))


@torch.library.custom_op("spio::checkpoint8_unpack", mutates_args=())
def checkpoint8_unpack_op(codes: torch.Tensor, exponents: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """The tensor of ``dtype`` that the codes and exponents stand for."""
    return _unpack(codes, exponents, dtype)


@checkpoint8_unpack_op.register_fake
def _checkpoint8_unpack_fake(codes, exponents, dtype):
    return codes.new_empty(codes.shape, dtype=dtype).to(memory_format=torch.channels_last)


def checkpoint8_pack(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """The 8-bit form of an NCHW tensor (channels_last, a multiple of 8 channels; float16, bfloat16 or float32):
    ``(codes int8 (n, c, h, w), exponents uint8 (n, c / 8, h, w))``, both channels_last.  Not differentiable."""
    return _pack(x) if plain_eager(x) else checkpoint8_pack_op(x.detach())


def checkpoint8_unpack(codes: torch.Tensor, exponents: torch.Tensor,
                       dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """The values that ``codes`` and ``exponents`` stand for, as a channels_last tensor of ``dtype``.  They are
    exact in the type that was packed."""
    if plain_eager(codes, exponents):
        return _unpack(codes, exponents, dtype)
    return checkpoint8_unpack_op(codes, exponents, dtype)


# ---- the convolution with its input kept in 8 bits


def _conv_forward(inputs, weight, bias, *args) -> torch.Tensor:
    assert weight.device == inputs.device and (bias is None or bias.device == inputs.device)
    return forward_kernels(inputs, weight, bias, *args)


@torch.library.custom_op("spio::conv2d_gw8_checkpoint8", mutates_args=())
def conv2d_gw8_checkpoint8_op(
    inputs: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, stride: int = 1,
    padding_y: int = 0, padding_x: int = 0, dilation: int = 1, groups: int = 1,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, codes, exponents): the convolution and the 8-bit form of its input."""
    y = _conv_forward(inputs, weight, bias, stride, padding_y, padding_x, dilation, groups)
    return y, *_pack(inputs)


@conv2d_gw8_checkpoint8_op.register_fake
def _conv2d_gw8_checkpoint8_fake(inputs, weight, bias=None, stride: int = 1, padding_y: int = 0,
                                 padding_x: int = 0, dilation: int = 1, groups: int = 1):
    y = torch.ops.spio.conv2d_gw8(inputs, weight, bias, stride, padding_y, padding_x, dilation, groups)
    return (y, *_checkpoint8_pack_fake(inputs))


def _setup_context(ctx, inputs, output):
    _x, weight, bias, _stride, padding_y, padding_x, *_ = inputs
    _y, codes, exponents = output
    ctx.mark_non_differentiable(codes, exponents)
    ctx.save_for_backward(codes, exponents, weight, bias)
    ctx.padding = (padding_y, padding_x)


def _gradients(ctx, grad_output, unpack, backward):
    codes, exponents, weight, bias = ctx.saved_tensors
    need = ctx.needs_input_grad
    want = (need[0], need[1], need[2] and bias is not None)
    # only the weight gradient reads the input's values; the others take its shape and type from `x`
    x = unpack(codes, exponents, torch.float16) if want[1] else torch.empty_like(codes, dtype=torch.float16)
    grads = backward(x, weight, bias, grad_output, *ctx.padding, *want)
    return tuple(g if w else None for g, w in zip(grads, want)) + (None,) * 5


def _backward(ctx, grad_output, _grad_codes, _grad_exponents):
    return _gradients(ctx, grad_output, checkpoint8_unpack_op, conv2d_gw8_backward_op)


conv2d_gw8_checkpoint8_op.register_autograd(_backward, setup_context=_setup_context)


def _autocast(ks, inputs, weight, bias=None, *args, **kwargs):
    """Under CUDA autocast: run in fp16 (bias in fp32) and return the input's dtype."""
    in_dtype = inputs.dtype
    autocast = torch._C.DispatchKeySet("AutocastCUDA")
    with torch._C._ExcludeDispatchKeyGuard(autocast):
        y, codes, exponents = torch.ops.spio.conv2d_gw8_checkpoint8.default.redispatch(
            ks - autocast, inputs.to(dtype=torch.float16), weight.to(dtype=torch.float16),
            bias.to(dtype=torch.float32) if bias is not None else None, *args, **kwargs)
    return y.to(dtype=in_dtype), codes, exponents


_fragment = torch.library.Library("spio", "FRAGMENT")
_fragment.impl("conv2d_gw8_checkpoint8", _autocast, "AutocastCUDA", with_keyset=True)


class _Conv2dGw8Checkpoint8(torch.autograd.Function):
    """The operator for plain eager calls."""

    @staticmethod
    def forward(ctx, inputs, weight, bias, stride, padding_y, padding_x, dilation, groups):
        y = _conv_forward(inputs, weight, bias, stride, padding_y, padding_x, dilation, groups)
        ctx.save_for_backward(*_pack(inputs), weight, bias)
        ctx.padding = (padding_y, padding_x)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        # autograd wants the weight gradient in the weight's type: the kernels round their sums once
        return _gradients(ctx, grad_output, _unpack,
                          partial(backward_kernels, own_scratch=True, grad_weight_dtype=torch.float16))


def conv2d_gw8_checkpoint8(inputs: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                           stride: int = 1, padding_y: int = 0, padding_x: int = 0, dilation: int = 1,
                           groups: int = 1) -> torch.Tensor:
    """:func:`conv2d_gw8` that keeps the 8-bit form of ``inputs`` for the backward pass (1.125 bytes a value
    instead of 2).  Output, input gradient and bias gradient are those of :func:`conv2d_gw8`; the weight gradient
    is taken at the restored input."""
    if torch.is_grad_enabled() and weight.requires_grad:
        if (inputs.dtype == weight.dtype == torch.float16 and (bias is None or bias.dtype == torch.float32)
                and plain_eager(inputs, weight, bias)):
            return _Conv2dGw8Checkpoint8.apply(inputs, weight, bias, stride, padding_y, padding_x, dilation, groups)
        return conv2d_gw8_checkpoint8_op(inputs, weight, bias, stride, padding_y, padding_x, dilation, groups)[0]
    # nothing will read the input again
    return conv2d_gw8(inputs, weight, bias, stride, padding_y, padding_x, dilation, groups)
