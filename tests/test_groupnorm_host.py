"""Group norm and 8-bit checkpoints without a GPU: refusals of the C ABI and of the operators, shapes under fake
tensors, module matching."""

import ctypes

import pytest
import torch
from torch import nn
from torch._subclasses import FakeTensorMode

from spio_b200 import _clib
from spio_b200.functional import (checkpoint8_pack, checkpoint8_unpack, conv2d_gw8_checkpoint8, groupnorm_2d,
                                  groupnorm_2d_op)
from spio_b200.layers import GroupNorm2d
from tests.norm_reference import B200, PLANNED, blocks_of, plan_of, restored


def desc(n=2, pixels=12, c=32, groups=4, type=0, activation=0, eps=1e-5):
    return ctypes.byref(_clib.GroupNorm2dDesc(n, pixels, c, groups, type, activation, eps))


@pytest.mark.parametrize("bad,message", [
    (dict(c=12), "multiple of 8"), (dict(c=0), "multiple of 8"), (dict(groups=5), "divisible"), (dict(groups=0), "divisible"),
    (dict(groups=-1), "divisible"), (dict(type=3), "data type"), (dict(activation=4), "activation"), (dict(n=-1), "negative"),
    (dict(pixels=-1), "negative"), (dict(pixels=2 ** 31), "pixels"), (dict(c=4096, groups=1), "2048 channels"),
    (dict(c=8 * 257 * 3, groups=8), "2048 channels"),
])
def test_library_refuses_descriptors(bad, message):
    lib = _clib.load()
    assert lib.spio_groupnorm_2d_fwd(16, None, None, None, 16, None, None, desc(**bad), 16, 1 << 20, None) != 0
    assert message in _clib.last_error()
    assert lib.spio_groupnorm_2d_bwd(16, None, None, 16, 16, None, None, 16, None, None, desc(**bad), 16, 1 << 20, None) != 0
    assert message in _clib.last_error()
    assert lib.spio_groupnorm_2d_fwd_scratch_bytes(desc(**bad)) == 0
    assert lib.spio_groupnorm_2d_bwd_scratch_bytes(desc(**bad)) == 0


def test_library_refuses_pointers():
    lib = _clib.load()
    fwd, bwd = lib.spio_groupnorm_2d_fwd, lib.spio_groupnorm_2d_bwd
    for args, message in [((None, None, None, None, 16), "NULL"), ((16, None, None, None, None), "NULL"),
                          ((24, None, None, None, 16), "16-byte"), ((16, None, None, None, 8), "16-byte"),
                          ((16, 4, None, None, 16), "8-byte"), ((16, None, 16, None, 16), "together"),
                          ((16, None, 12, 16, 16), "8-byte"), ((16, None, 16, 18, 16), "4-byte")]:
        assert fwd(*args, None, None, desc(), 16, 1 << 20, None) != 0 and message in _clib.last_error(), args
    for args, message in [((16, None, None, None, 16, None, None, 16), "NULL"), ((16, None, None, 16, None, None, None, 16), "NULL"),
                          ((16, None, None, 16, 16, None, None, None), "NULL"), ((8, None, None, 16, 16, None, None, 16), "16-byte"),
                          ((16, None, None, 16, None, 16, None, 16), "together")]:
        assert bwd(*args, None, None, desc(), 16, 1 << 20, None) != 0 and message in _clib.last_error(), args
    assert bwd(16, None, None, 16, 16, None, None, 16, None, None, desc(), 8, 1 << 20, None) != 0
    assert "16-byte" in _clib.last_error()
    # fp32 pieces of 32 bytes are written at once
    assert fwd(16, None, None, None, 16, None, None, desc(type=2), 16, 1 << 20, None) != 0 and "32-byte" in _clib.last_error()
    assert bwd(16, None, None, 16, 16, None, None, 16, None, None, desc(type=2), 16, 1 << 20, None) != 0
    assert "32-byte" in _clib.last_error()
    assert lib.spio_checkpoint8_unpack(16, 16, 16, 1, 2, None) != 0 and "32-byte" in _clib.last_error()
    # nothing to do is no error: an empty batch, no gradient asked for
    assert fwd(None, None, None, None, None, None, None, desc(n=0), None, 0, None) == 0
    assert bwd(None, None, None, None, None, None, None, None, None, None, desc(), None, 0, None) == 0
    pack, unpack = lib.spio_checkpoint8_pack, lib.spio_checkpoint8_unpack
    for args, message in [((16, 16, 16, -1, 0), "negative"), ((16, 16, 16, 1, 5), "type"), ((None, 16, 16, 1, 0), "NULL"),
                          ((16, 16, 8, 1, 0), "16-byte"), ((12, 16, 16, 1, 0), "8-byte"), ((16, 16, 16, 1 << 41, 0), "many")]:
        assert pack(*args, None) != 0 and message in _clib.last_error(), args
    assert pack(None, None, None, 0, 0, None) == 0 and unpack(None, None, None, 0, 2, None) == 0


def test_operators_refuse_cpu_tensors():
    x = torch.randn(2, 16, 3, 3)
    for call in (lambda: groupnorm_2d(x, 4), lambda: groupnorm_2d(x.requires_grad_(True), 4), lambda: checkpoint8_pack(x),
                 lambda: checkpoint8_unpack(torch.zeros(1, 8, 1, 1, dtype=torch.int8), torch.zeros(1, 1, 1, 1, dtype=torch.uint8))):
        with pytest.raises(ValueError, match="CUDA devices only"):
            call()


def test_shapes_under_fake_tensors():
    with FakeTensorMode():
        x = torch.empty(2, 32, 5, 7, device="cuda", dtype=torch.bfloat16)
        w = torch.ones(32, device="cuda")
        y = groupnorm_2d(x, 4, w, w, activation="silu")
        assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous(memory_format=torch.channels_last)
        _, stats, codes, exponents = groupnorm_2d_op(x, w, None, 4, 1e-5, "none", True)
        assert stats.shape == (2, 4, 2) and codes.shape == x.shape and exponents.shape == (2, 4, 5, 7)
        codes, exponents = checkpoint8_pack(x)
        assert codes.dtype == torch.int8 and exponents.dtype == torch.uint8
        assert checkpoint8_unpack(codes, exponents, torch.bfloat16).dtype == torch.bfloat16
        k = torch.empty(32, 8, 3, 3, device="cuda", dtype=torch.float16, requires_grad=True)
        y = conv2d_gw8_checkpoint8(x.half(), k, None, padding_y=1, padding_x=0, groups=4)
        assert y.shape == (2, 32, 5, 5) and y.requires_grad


def test_module_matching():
    assert GroupNorm2d.match(nn.GroupNorm(4, 32)) and not GroupNorm2d.match(nn.GroupNorm(4, 36))
    assert not GroupNorm2d.match(nn.BatchNorm2d(32)) and not GroupNorm2d.match(nn.GroupNorm(1, 4096))
    gn = GroupNorm2d.from_torch_module(nn.GroupNorm(4, 32, eps=1e-3, affine=False).eval(), "gelu", True)
    assert gn.weight is None and gn.eps == 1e-3 and gn.checkpoint8 and not gn.training
    assert [GroupNorm2d.activation_of(m) for m in (nn.ReLU(), nn.SiLU(), nn.GELU(), nn.GELU("tanh"), nn.Tanh())] == [
        "relu", "silu", "gelu", None, None]
    with pytest.raises(ValueError):
        GroupNorm2d.from_torch_module(nn.GroupNorm(4, 36))
    with pytest.raises(ValueError):
        GroupNorm2d(4, 32, activation="tanh")


def test_reference_blocks():
    """The tests' own definition of the 8-bit form, on numbers worked out by hand."""
    x = torch.tensor([127.0, 63.5, -1.5, 0.5, 0, 0, 0, 0], dtype=torch.float32).reshape(1, 8, 1, 1)
    codes, scale = blocks_of(x)
    assert scale.item() == 1 and codes.flatten().tolist() == [127, 64, -2, 0, 0, 0, 0, 0]
    codes, scale = blocks_of(x + torch.tensor([0.5, 0, 0, 0, 0, 0, 0, 0]).reshape(1, 8, 1, 1))   # 127.5 would round to 128
    assert scale.item() == 2 and codes.flatten().tolist() == [64, 32, -1, 0, 0, 0, 0, 0]
    top = torch.full((1, 8, 1, 1), 65504.0, dtype=torch.float16)
    codes, scale = blocks_of(top)
    assert scale.item() == 1024 and set(codes.flatten().tolist()) == {63} and bool(restored(top).half().isfinite().all())
    codes, scale = blocks_of(torch.zeros(1, 8, 1, 1))
    assert scale.item() == 2.0 ** -126 and not bool(codes.any())


@pytest.mark.parametrize("shape,groups,dtype,act,forms", PLANNED, ids=str)
def test_forms_of_launch(shape, groups, dtype, act, forms):
    """The sizes of the GPU test of this name reach what they are there for."""
    for form, (backward, coded) in zip(forms.split(), ((0, 0), (0, 1), (1, 0), (1, 1))):
        p = plan_of(shape, groups, dtype, act, backward, coded)
        narrower = p["slab_pieces"] * p["slabs"] != shape[1] // 8
        assert f"{2 - p['one_launch']}{'n' * narrower}" == form, (backward, coded, p)
        # what any plan keeps to
        assert p["parts"] % p["cluster"] == 0 and 1 <= p["cluster"] <= 16 and p["smem_bytes"] <= B200[1]
        assert p["slab_pieces"] <= p["threads"] and 0 <= p["slab_pieces"] * p["slabs"] - shape[1] // 8 < p["slab_pieces"]
        assert p["grid"] == shape[0] * p["slabs"] * p["parts"] and p["parts"] <= shape[2] * shape[3]
        assert (p["slab_pieces"] * 8) % (shape[1] // groups) == 0          # whole groups
        sums = 8 * shape[0] * p["parts"] * shape[1]                        # of the backward pass, for the channels
        assert p["scratch_bytes"] >= sums if backward else (p["scratch_bytes"] > 0) == (p["one_launch"] == 0)


def test_plan_refusals():
    lib, info = _clib.load(), _clib.GroupNorm2dPlanInfo()
    for d, sms, out, message in [(desc(groups=5), 148, info, "divisible"), (desc(n=0), 148, info, "empty"),
                                 (desc(pixels=0), 148, info, "empty"), (desc(), 0, info, "device"), (desc(), 148, None, "NULL")]:
        out = ctypes.byref(out) if out is not None else None
        assert lib.spio_groupnorm_2d_plan_for(d, 0, 0, sms, B200[1], out) != 0 and message in _clib.last_error()
    assert ctypes.sizeof(_clib.GroupNorm2dPlanInfo) == 8 * 4 + 8
    for d in (desc(), desc(n=1, pixels=1 << 20)):      # too little shared memory for any launch
        assert lib.spio_groupnorm_2d_plan_for(d, 0, 0, 148, 1024, ctypes.byref(info)) != 0 and "fits" in _clib.last_error()


def test_parameter_types_under_fake_tensors():
    """16-bit parameters beside data of their type are taken, other mixtures refused."""
    with FakeTensorMode():
        x = torch.empty(2, 32, 5, 7, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        w = torch.ones(32, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        y = groupnorm_2d(x, 4, w, w, activation="silu", checkpoint8=True)
        assert y.requires_grad and y.dtype == torch.bfloat16
        for weight, bias in ((w, w.float()), (w.half(), None), (None, w.double())):
            with pytest.raises(ValueError, match="weight and bias"):
                groupnorm_2d(x, 4, weight, bias)
