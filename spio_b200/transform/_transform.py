"""Swap supported ``nn.Conv2d`` modules of a model for this package's layers.

``transform`` and ``scan_modules`` behave like the reference's
(spio/transform/_transform.py:16-108): the model is traced with torch.fx, every
``call_module`` node whose module a layer class matches is served by a new layer that
shares the old parameters, and a ``GraphModule`` is returned.  Because the replacement
keeps the submodule's qualified name, the graph itself needs no rewriting: the module is
replaced under its parent and the graph recompiled.  On request group norms are replaced as well, with the
activations behind them (the reference has no group norm).
"""

from __future__ import annotations

from typing import List, Optional, Tuple

import torch
from torch import fx

from ..layers import Conv2dGw8, GroupNorm2d
from ..util.logger import log

spio_modules_classes = [Conv2dGw8]


def _matching_class(module):
    for cls in spio_modules_classes:
        if cls.match(module):
            return cls
    return None


def _set_submodule(root: torch.nn.Module, qualified_name: str, new: torch.nn.Module) -> None:
    parent_name, _, leaf = qualified_name.rpartition(".")
    parent = root.get_submodule(parent_name) if parent_name else root
    setattr(parent, leaf, new)


def _following_activation(traced: fx.GraphModule, node: fx.Node) -> Optional[str]:
    """The activation module that alone uses ``node``'s value, by the name that :class:`GroupNorm2d` gives it."""
    if len(node.users) != 1:
        return None
    user = next(iter(node.users))
    return GroupNorm2d.activation_of(traced.get_submodule(user.target)) if user.op == "call_module" else None


def _replace_group_norm(traced: fx.GraphModule, nodes: List[fx.Node], checkpoint8: bool) -> torch.nn.Module:
    """The layer that serves every call of one group norm.  It takes in the activation behind them if that is the
    same at each."""
    activations = {_following_activation(traced, node) for node in nodes}
    activation = activations.pop() if len(activations) == 1 else None
    if activation is not None:
        for node in nodes:
            user = next(iter(node.users))
            user.replace_all_uses_with(node)
            traced.graph.erase_node(user)
    return GroupNorm2d.from_torch_module(traced.get_submodule(nodes[0].target), activation or "none", checkpoint8)


def _transform(model: torch.nn.Module, group_norm: bool = False,
               checkpoint8: bool = False) -> Tuple[fx.GraphModule, int]:
    """The transformed model and how many modules were replaced."""
    traced = fx.symbolic_trace(model)
    calls = {}
    for node in traced.graph.nodes:
        if node.op == "call_module":
            calls.setdefault(node.target, []).append(node)
    replaced = 0
    for target, nodes in calls.items():
        module = traced.get_submodule(target)
        cls = _matching_class(module)
        if cls is not None:
            # (a class that a user has added to the list need not know the option)
            options = {"checkpoint8": True} if checkpoint8 and hasattr(cls, "checkpoint8") else {}
            new = cls.from_torch_module(module, **options)
        elif group_norm and GroupNorm2d.match(module):
            new = _replace_group_norm(traced, nodes, checkpoint8)
        else:
            continue
        _set_submodule(traced, target, new)
        replaced += 1
        log(f"replaced a {type(module).__module__}.{type(module).__qualname__} module with "
            f"{type(new).__module__}.{new}")
    traced.delete_all_unused_submodules()
    traced.recompile()
    return traced, replaced


def transform(model: torch.nn.Module, group_norm: bool = False, checkpoint8: bool = False) -> fx.GraphModule:
    """The model with every supported module replaced by its counterpart of this package.

    ``group_norm`` replaces the ``nn.GroupNorm`` modules too, each with the ReLU, SiLU or GELU module behind it:
    for models whose group norms all see image tensors on a CUDA device, as ``GroupNorm2d`` does.  ``checkpoint8`` lets the new
    layers keep their inputs in 8 bits for the backward pass."""
    return _transform(model, group_norm, checkpoint8)[0]


class _ScanInterpreter(fx.Interpreter):
    def __init__(self, graph_module: fx.GraphModule):
        super().__init__(graph_module)
        self.params_lst: List = []

    def call_module(self, target, args, kwargs):
        module = self.fetch_attr(target)
        cls = _matching_class(module)
        if cls is not None:
            self.params_lst.append(cls.Params.from_torch_module(module, *args))
        return super().call_module(target, args, kwargs)


def scan_modules(model: torch.nn.Module, *args) -> List:
    """Run the model once on ``args`` and return the Params of every module that
    :func:`transform` would replace, in execution order."""
    interp = _ScanInterpreter(fx.symbolic_trace(model))
    interp.run(*args)
    return interp.params_lst
