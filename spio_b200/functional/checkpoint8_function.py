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

from typing import Optional, Tuple

import torch

from .. import _clib
from ..util.tensor_format import to_channels_last
from .conv2d_gw8_function import conv2d_gw8, conv2d_gw8_backward_op

TYPE_CODES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


def kernel_layout(t: torch.Tensor) -> torch.Tensor:
    """``t`` in channels_last order at a 16-byte boundary (itself if it is already)."""
    t = to_channels_last(t)
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.channels_last)


def _check_image(x: torch.Tensor, what: str) -> None:
    if x.device.type != "cuda":
        raise ValueError(f"spio {what} runs on CUDA devices only (no CPU implementation)")
    assert x.dim() == 4, "expected an NCHW tensor"


def empty_codes(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Unset codes and exponents for ``x``."""
    n, c, h, w = x.shape
    cl = torch.channels_last
    return (torch.empty((n, c, h, w), device=x.device, dtype=torch.int8, memory_format=cl),
            torch.empty((n, c // 8, h, w), device=x.device, dtype=torch.uint8, memory_format=cl))


def _pack_into(codes: torch.Tensor, exponents: torch.Tensor, x: torch.Tensor) -> None:
    """``x`` in kernel layout."""
    with torch.cuda.device(x.device):
        _clib.check(_clib.load().spio_checkpoint8_pack(
            codes.data_ptr(), exponents.data_ptr(), x.data_ptr(), x.numel() // 8, TYPE_CODES[x.dtype],
            torch.cuda.current_stream(x.device).cuda_stream), "checkpoint8_pack")


@torch.library.custom_op("spio::checkpoint8_pack", mutates_args=())
def checkpoint8_pack_op(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    _check_image(x, "checkpoint8_pack")
    assert x.dtype in TYPE_CODES, "expected float16, bfloat16 or float32"
    assert x.shape[1] % 8 == 0, "Number of channels must be a multiple of 8."
    codes, exponents = empty_codes(x)
    _pack_into(codes, exponents, kernel_layout(x))
    return codes, exponents


@checkpoint8_pack_op.register_fake
def _checkpoint8_pack_fake(x):
    n, c, h, w = x.shape
    return (x.new_empty(x.shape, dtype=torch.int8).to(memory_format=torch.channels_last),
            x.new_empty((n, c // 8, h, w), dtype=torch.uint8).to(memory_format=torch.channels_last))


@torch.library.custom_op("spio::checkpoint8_unpack", mutates_args=())
def checkpoint8_unpack_op(codes: torch.Tensor, exponents: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    _check_image(codes, "checkpoint8_unpack")
    assert dtype in TYPE_CODES, "expected float16, bfloat16 or float32"
    assert codes.dtype == torch.int8 and exponents.dtype == torch.uint8
    assert codes.device == exponents.device
    n, c, h, w = codes.shape
    assert c % 8 == 0 and tuple(exponents.shape) == (n, c // 8, h, w), "exponents must be (n, c / 8, h, w)"
    x = torch.empty((n, c, h, w), device=codes.device, dtype=dtype, memory_format=torch.channels_last)
    codes, exponents = kernel_layout(codes), to_channels_last(exponents)
    with torch.cuda.device(codes.device):
        _clib.check(_clib.load().spio_checkpoint8_unpack(
            x.data_ptr(), codes.data_ptr(), exponents.data_ptr(), codes.numel() // 8, TYPE_CODES[dtype],
            torch.cuda.current_stream(codes.device).cuda_stream), "checkpoint8_unpack")
    return x


@checkpoint8_unpack_op.register_fake
def _checkpoint8_unpack_fake(codes, exponents, dtype):
    return codes.new_empty(codes.shape, dtype=dtype).to(memory_format=torch.channels_last)


def checkpoint8_pack(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """The 8-bit form of an NCHW tensor (channels_last, a multiple of 8 channels; float16, bfloat16 or float32):
    ``(codes int8 (n, c, h, w), exponents uint8 (n, c / 8, h, w))``, both channels_last.  Not differentiable."""
    return checkpoint8_pack_op(x.detach())


def checkpoint8_unpack(codes: torch.Tensor, exponents: torch.Tensor,
                       dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """The values that ``codes`` and ``exponents`` stand for, as a channels_last tensor of ``dtype``.  They are
    exact in the type that was packed."""
    return checkpoint8_unpack_op(codes, exponents, dtype)


# ---- the convolution with its input kept in 8 bits


@torch.library.custom_op("spio::conv2d_gw8_checkpoint8", mutates_args=())
def conv2d_gw8_checkpoint8_op(
    inputs: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, stride: int = 1,
    padding_y: int = 0, padding_x: int = 0, dilation: int = 1, groups: int = 1,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, codes, exponents): the convolution and the 8-bit form of its input."""
    y = conv2d_gw8(inputs, weight, bias, stride, padding_y, padding_x, dilation, groups)
    codes, exponents = empty_codes(inputs)
    _pack_into(codes, exponents, kernel_layout(inputs))
    return y, codes, exponents


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


def _backward(ctx, grad_output, _grad_codes, _grad_exponents):
    codes, exponents, weight, bias = ctx.saved_tensors
    need = ctx.needs_input_grad
    want = (need[0], need[1], need[2] and bias is not None)
    # The weight gradient is the only one that reads the input; the others need its shape alone, which the
    # codes' (an eighth-bit tensor of the same shape) unset storage stands in for.
    x = (checkpoint8_unpack_op(codes, exponents, torch.float16) if want[1]
         else torch.empty_like(codes, dtype=torch.float16))
    grads = conv2d_gw8_backward_op(x, weight, bias, grad_output, *ctx.padding, *want)
    grad_input, grad_weight, grad_bias = (g if w else None for g, w in zip(grads, want))
    return grad_input, grad_weight, grad_bias, None, None, None, None, None


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


def conv2d_gw8_checkpoint8(inputs: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                           stride: int = 1, padding_y: int = 0, padding_x: int = 0, dilation: int = 1,
                           groups: int = 1) -> torch.Tensor:
    """:func:`conv2d_gw8` that keeps the 8-bit form of ``inputs`` for the backward pass (1.125 bytes a value
    instead of 2).  Output, input gradient and bias gradient are those of :func:`conv2d_gw8`; the weight gradient
    is taken at the restored input."""
    if torch.is_grad_enabled() and weight.requires_grad:
        return conv2d_gw8_checkpoint8_op(inputs, weight, bias, stride, padding_y, padding_x, dilation, groups)[0]
    # nothing will read the input again
    return conv2d_gw8(inputs, weight, bias, stride, padding_y, padding_x, dilation, groups)
