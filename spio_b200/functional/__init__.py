"""Functional operators (the names the reference exports from spio.functional)."""

from .conv2d_gw8_function import (conv2d_gw8, conv2d_gw8_backward_op, get_grad_weight_dtype,
                                  set_grad_weight_dtype)
from .layernorm_2d_function import layernorm_2d, layernorm_2d_op, layernorm_2d_backward_op
from .checkpoint8_function import (checkpoint8_pack, checkpoint8_pack_op, checkpoint8_unpack, checkpoint8_unpack_op,
                                   conv2d_gw8_checkpoint8, conv2d_gw8_checkpoint8_op)
from .groupnorm_2d_function import groupnorm_2d, groupnorm_2d_backward_op, groupnorm_2d_op
