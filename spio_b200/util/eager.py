"""When a call of a Python operator may take its C++ form instead.

A Python operator costs 20 to 50 us of host time in eager mode (about 200 us with its backward pass), more than
the kernels of a small tensor.  A plain eager call of the convolution with the 8-bit checkpoint therefore takes an
operator in C++ (csrc/torch_ops.cpp); whatever has to see the public operator -- fake tensors, tensor subclasses,
tracing and compilation, functorch transforms, forward-mode derivatives, dispatch modes such as profilers'
counters -- still finds that.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

_PLAIN = (torch.Tensor, torch.nn.Parameter)


def plain_eager(*tensors) -> bool:
    """Whether these arguments (tensors or None) are ordinary eager tensors that nothing watches."""
    for t in tensors:
        if t is not None and type(t) not in _PLAIN:
            return False
    return (not torch.compiler.is_compiling()
            and torch._C._len_torch_dispatch_stack() == 0
            and torch._C._len_torch_function_stack() == 0
            and torch._C._functorch.peek_interpreter_stack() is None
            and torch._C._get_tracing_state() is None
            and forward_ad._current_level < 0)
