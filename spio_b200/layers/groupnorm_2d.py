"""``GroupNorm2d``: group norm with an activation over an NCHW tensor, backed by the ``spio::groupnorm_2d`` operator
(channels_last float16, bfloat16 or float32 data on a CUDA device; parameters in fp32 or of the data's type, of any type
under autocast)."""

from __future__ import annotations

import math
from typing import Optional

import torch
from torch import nn

from ..functional.groupnorm_2d_function import ACTIVATIONS, groupnorm_2d


def _fits(num_groups: int, num_channels: int) -> bool:
    """The kernels hold whole groups and whole blocks of 8 channels in one thread block."""
    return math.lcm(num_channels // num_groups, 8) <= 2048


class GroupNorm2d(nn.Module):
    """``activation(group_norm(x))``; ``checkpoint8`` keeps the input in 8 bits for the backward pass."""

    def __init__(self, num_groups: int, num_channels: int, eps: float = 1e-5, affine: bool = True,
                 activation: str = "none", checkpoint8: bool = False, device=None, dtype=torch.float32):
        super().__init__()
        if num_channels <= 0 or num_channels % 8 != 0 or num_groups <= 0 or num_channels % num_groups != 0:
            raise ValueError("GroupNorm2d needs a multiple of 8 channels that the number of groups divides")
        if not _fits(num_groups, num_channels):
            raise ValueError("GroupNorm2d: groups (rounded up to whole blocks of 8 channels) may span at most 2048 channels")
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}")
        self.num_groups = num_groups
        self.num_channels = num_channels
        self.eps = eps
        self.affine = affine
        self.activation = activation
        self.checkpoint8 = checkpoint8
        if affine:
            self.weight = nn.Parameter(torch.ones(num_channels, device=device, dtype=dtype))
            self.bias = nn.Parameter(torch.zeros(num_channels, device=device, dtype=dtype))
        else:
            self.register_parameter("weight", None)
            self.register_parameter("bias", None)

    @staticmethod
    def match(module: nn.Module) -> bool:
        """True for an ``nn.GroupNorm`` that this layer can replace when it is applied to an image tensor."""
        return (isinstance(module, nn.GroupNorm) and module.num_channels % 8 == 0
                and _fits(module.num_groups, module.num_channels))

    @staticmethod
    def activation_of(module: Optional[nn.Module]) -> Optional[str]:
        """The name of the activation that ``module`` computes, or None if the norm cannot take it in."""
        if isinstance(module, nn.ReLU):
            return "relu"
        if isinstance(module, nn.SiLU):
            return "silu"
        if isinstance(module, nn.GELU) and module.approximate == "none":
            return "gelu"
        return None

    @staticmethod
    def from_torch_module(module: nn.GroupNorm, activation: str = "none", checkpoint8: bool = False) -> "GroupNorm2d":
        """Same parameters (shared, not copied) as the given ``nn.GroupNorm``."""
        if not GroupNorm2d.match(module):
            raise ValueError(f"{module} does not match GroupNorm2d")
        gn = GroupNorm2d(module.num_groups, module.num_channels, eps=module.eps, affine=module.affine,
                         activation=activation, checkpoint8=checkpoint8)
        if module.affine:
            gn.weight = module.weight
            gn.bias = module.bias
        gn.train(module.training)
        return gn

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return groupnorm_2d(x, self.num_groups, self.weight, self.bias, self.eps, self.activation, self.checkpoint8)

    def extra_repr(self) -> str:
        return (f"{self.num_groups}, {self.num_channels}, eps={self.eps}, affine={self.affine}, "
                f"activation={self.activation}, checkpoint8={self.checkpoint8}")
