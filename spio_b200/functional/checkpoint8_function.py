"""Activation checkpoints in 8 bits: ``spio::checkpoint8_pack`` / ``spio::checkpoint8_unpack``, and the
group-width-8 convolution that keeps its input in that form for the backward pass.

A block of 8 consecutive channels of a pixel -- one channel group of the gw8 convolution -- becomes 8 signed
codes and one exponent byte and stands for ``code * 2**(exponent - 127)``: 1.125 bytes a value.  The scale is
the smallest power of two (``2**-126`` at least) for which the block's largest magnitude rounds to at most 127,
so a restored value is off by at most half a step, 1/127 of the block's largest magnitude.  (Where rounding up
would leave the range of the type, codes stop at 63 and the error is up to 1/64 of that magnitude.  Where the scale
is at its floor the error is up to ``2**-127``, which may be all of a value.)  A block with an infinity or a NaN is
restored as NaN, so that a gradient scaler still finds it.

The reference keeps the convolution's input as it is (spio/functional/conv2d_gw8_function.py:150-171); this
form has no counterpart there.  The device work is done by libspio_b200 on torch's current stream; CPU tensors
raise.
"""

from __future__ import annotations

from functools import lru_cache
from typing import Optional, Tuple

import torch
from torch.overrides import handle_torch_function, has_torch_function

from .. import _clib
from ..compiler import flags
from ..kernels import Conv2dGw8Params, conv2d_gw8_kernel_factory, conv2d_gw8_wgrad_kernel_factory
from ..kernels.kernel import Kernel
from ..kernels.kernel_cache import KernelCache
from ..kernels.kernel_params_logger import kernel_params_logging_is_enabled
from ..util.eager import plain_eager
from . import conv2d_gw8_function
from .conv2d_gw8_function import _is_unit, conv2d_gw8, conv2d_gw8_backward_op

_fragment = torch.library.Library("spio", "FRAGMENT")
_fragment.define("checkpoint8_pack(Tensor x) -> (Tensor, Tensor)")
_fragment.define("checkpoint8_unpack(Tensor codes, Tensor exponents, ScalarType dtype) -> Tensor")
# conv2d_gw8_checkpoint8 for plain eager calls, with the tile configurations of its three kernels
_fragment.define("conv2d_gw8_checkpoint8_planned(Tensor inputs, Tensor weight, Tensor? bias, int padding_y, "
                 "int padding_x, int[] tunes) -> Tensor")
_clib.load_torch_ops_if_usable()

checkpoint8_pack_op = torch.ops.spio.checkpoint8_pack
checkpoint8_unpack_op = torch.ops.spio.checkpoint8_unpack
_conv_planned = torch.ops.spio.conv2d_gw8_checkpoint8_planned.default
_pack, _unpack = checkpoint8_pack_op.default, checkpoint8_unpack_op.default


@torch.library.register_fake("spio::checkpoint8_pack")
def _checkpoint8_pack_fake(x):
    n, c, h, w = x.shape
    return (x.new_empty(x.shape, dtype=torch.int8).to(memory_format=torch.channels_last),
            x.new_empty((n, c // 8, h, w), dtype=torch.uint8).to(memory_format=torch.channels_last))


@torch.library.register_fake("spio::checkpoint8_unpack")
def _checkpoint8_unpack_fake(codes, exponents, dtype):
    return codes.new_empty(codes.shape, dtype=dtype).to(memory_format=torch.channels_last)


def checkpoint8_pack(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """The 8-bit form of an NCHW tensor (channels_last, a multiple of 8 channels; float16, bfloat16 or float32):
    ``(codes int8 (n, c, h, w), exponents uint8 (n, c / 8, h, w))``, both channels_last.  Not differentiable."""
    if has_torch_function((x,)):      # a torch.fx proxy, a tensor subclass
        return handle_torch_function(checkpoint8_pack, (x,), x)
    _clib.load_torch_ops()
    return _pack(x.detach() if x.requires_grad else x)


def checkpoint8_unpack(codes: torch.Tensor, exponents: torch.Tensor,
                       dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """The values that ``codes`` and ``exponents`` stand for, as a channels_last tensor of ``dtype``.  They are
    exact in the type that was packed."""
    _clib.load_torch_ops()
    return _unpack(codes, exponents, dtype)


# ---- the convolution with its input kept in 8 bits


@torch.library.custom_op("spio::conv2d_gw8_checkpoint8", mutates_args=())
def conv2d_gw8_checkpoint8_op(
    inputs: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, stride: int = 1,
    padding_y: int = 0, padding_x: int = 0, dilation: int = 1, groups: int = 1,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, codes, exponents): the convolution and the 8-bit form of its input."""
    assert weight.device == inputs.device and (bias is None or bias.device == inputs.device)
    y = conv2d_gw8(inputs, weight, bias, stride, padding_y, padding_x, dilation, groups)
    return y, *_pack(inputs)


@conv2d_gw8_checkpoint8_op.register_fake
def _conv2d_gw8_checkpoint8_fake(inputs, weight, bias=None, stride: int = 1, padding_y: int = 0,
                                 padding_x: int = 0, dilation: int = 1, groups: int = 1):
    y = torch.ops.spio.conv2d_gw8(inputs, weight, bias, stride, padding_y, padding_x, dilation, groups)
    return (y, *_checkpoint8_pack_fake(inputs))


def _setup_context(ctx, inputs, output):
    x, weight, bias, _stride, padding_y, padding_x, *_ = inputs
    _y, codes, exponents = output
    ctx.mark_non_differentiable(codes, exponents)
    kept = (codes, exponents) if ctx.needs_input_grad[1] else (None, None)   # for the weight gradient alone
    ctx.save_for_backward(*kept, weight, bias)
    ctx.padding, ctx.size = (padding_y, padding_x), x.shape


def _backward(ctx, grad_output, _grad_codes, _grad_exponents):
    codes, exponents, weight, bias = ctx.saved_tensors
    need = ctx.needs_input_grad
    want = (need[0], need[1], need[2] and bias is not None)
    # only the weight gradient reads the input's values; the others take its shape and type from `x`
    x = (_unpack(codes, exponents, torch.float16) if want[1]
         else torch.empty(ctx.size, dtype=torch.float16, device=weight.device, memory_format=torch.channels_last))
    grads = conv2d_gw8_backward_op(x, weight, bias, grad_output, *ctx.padding, *want)
    return tuple(g if w else None for g, w in zip(grads, want)) + (None,) * 5


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


_fragment.impl("conv2d_gw8_checkpoint8", _autocast, "AutocastCUDA", with_keyset=True)


@lru_cache(maxsize=4096)
def _tunes(generation: int, device, x_shape, w_shape, has_bias: bool, padding) -> Optional[list]:
    """The tile configurations of the forward, input-gradient and weight-gradient kernels that the factories choose for
    these sizes, or None if one of them is not built into the library."""
    del generation
    params = Conv2dGw8Params(*x_shape, padding=padding, r=w_shape[2], s=w_shape[3], has_bias=has_bias)
    params.validate()
    kernels = (conv2d_gw8_kernel_factory.get_kernel(params, device),
               conv2d_gw8_kernel_factory.get_kernel(params, device, igrad=True),
               conv2d_gw8_wgrad_kernel_factory.get_kernel(params, device))
    if any(type(k) is not Kernel for k in kernels):
        return None
    return [getattr(k._tune, name) if k._tune is not None else 0 for k in kernels for name, _ in _clib.Tune._fields_]


def _eager_tunes(inputs, weight, bias, stride, padding_y, padding_x, dilation, groups) -> Optional[list]:
    """:func:`_tunes` for a plain eager call that the C++ operator can serve, else None."""
    if (conv2d_gw8_function._CHECK_STATUS or kernel_params_logging_is_enabled() or flags.jit.get()
            or not inputs.is_cuda or inputs.dim() != 4 or inputs.dtype != torch.float16
            or weight.dtype != torch.float16 or (bias is not None and bias.dtype != torch.float32)
            or not plain_eager(inputs, weight, bias)):
        return None
    assert _is_unit(stride) and _is_unit(dilation)
    assert groups == inputs.shape[1] // 8
    assert weight.dim() == 4 and weight.shape[0] == inputs.shape[1] and weight.shape[1] == 8, (
        "Only group width of 8 is supported.")
    return _tunes(KernelCache.generation, inputs.device, inputs.shape, weight.shape, bias is not None,
                  (padding_y, padding_x))


def conv2d_gw8_checkpoint8(inputs: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                           stride: int = 1, padding_y: int = 0, padding_x: int = 0, dilation: int = 1,
                           groups: int = 1) -> torch.Tensor:
    """:func:`conv2d_gw8` that keeps the 8-bit form of ``inputs`` for the backward pass (1.125 bytes a value
    instead of 2; nothing where the weight requires no gradient).  Output, input gradient and bias gradient are those of :func:`conv2d_gw8`; the weight gradient
    is taken at the restored input."""
    if has_torch_function((inputs, weight, bias)):      # a torch.fx proxy, a tensor subclass
        return handle_torch_function(conv2d_gw8_checkpoint8, (inputs, weight, bias), inputs, weight, bias, stride=stride,
                                     padding_y=padding_y, padding_x=padding_x, dilation=dilation, groups=groups)
    _clib.load_torch_ops()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (inputs, weight, bias)):
        tunes = _eager_tunes(inputs, weight, bias, stride, padding_y, padding_x, dilation, groups)
        if tunes is not None:
            return _conv_planned(inputs, weight, bias, padding_y, padding_x, tunes)
        return conv2d_gw8_checkpoint8_op(inputs, weight, bias, stride, padding_y, padding_x, dilation, groups)[0]
    # nothing is kept
    return conv2d_gw8(inputs, weight, bias, stride, padding_y, padding_x, dilation, groups)
