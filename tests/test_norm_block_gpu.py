"""Convolution, group norm with an activation and 8-bit checkpoints together, as a residual block uses them: each
step's output and gradients against float64 at the values it was given, the transformed module against the same
chain of operators, and a captured training step."""

import pytest
import torch
from torch import nn

from spio_b200.functional import conv2d_gw8, conv2d_gw8_checkpoint8, groupnorm_2d
from spio_b200.kernels import device_status
from spio_b200.transform import transform
from tests.norm_reference import CONST, Reference, assert_within, half_step, restored

CL = torch.channels_last
C, GROUPS = 64, (4, 16)


class Block(nn.Module):
    """conv -> norm -> SiLU -> conv -> norm -> GELU, added to the input"""

    def __init__(self):
        super().__init__()
        self.conv1 = nn.Conv2d(C, C, 3, padding=1, groups=C // 8)
        self.norm1 = nn.GroupNorm(GROUPS[0], C)
        self.act1 = nn.SiLU()
        self.conv2 = nn.Conv2d(C, C, 5, padding=2, groups=C // 8, bias=False)
        self.norm2 = nn.GroupNorm(GROUPS[1], C)
        self.act2 = nn.GELU()

    def forward(self, x):
        return x + self.act2(self.norm2(self.conv2(self.act1(self.norm1(self.conv1(x))))))


def make_block(seed):
    """A block whose convolution weights are fp16 values, so that autocast rounds nothing."""
    torch.manual_seed(seed)
    block = Block()
    with torch.no_grad():
        for conv in (block.conv1, block.conv2):
            conv.weight.copy_(conv.weight.half())
        for norm in (block.norm1, block.norm2):
            norm.weight.uniform_(0.5, 1.5)
            norm.bias.normal_(0, 0.5)
    return block.cuda().to(memory_format=CL)


def make_data(shape, seed):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(shape, generator=gen).half().cuda().contiguous(memory_format=CL) for _ in range(2)]


def conv_reference(x, w, b, dy, padding, checkpoint8):
    """((y, dx, dw, db), their tolerances): one rounding to fp16 -- none for the bias -- and fp32 sums, whose error is
    counted in the magnitudes that enter them."""

    def conv(x, w, b):
        return nn.functional.conv2d(x, w, b, padding=padding, groups=C // 8)

    def grads(x, w, dy):
        x, w = x.requires_grad_(True), w.requires_grad_(True)
        return torch.autograd.grad(conv(x, w, None), (x, w), dy)

    x, w, dy = (t.detach().double().cpu() for t in (x, w, dy))
    b = torch.zeros(C, dtype=torch.float64) if b is None else b.detach().double().cpu()
    kept = restored(x.half()) if checkpoint8 else x
    y, y_size = conv(x, w, b), conv(x.abs(), w.abs(), b.abs())
    (dx, _), (_, dw) = grads(x.clone(), w.clone(), dy), grads(kept.clone(), w.clone(), dy)
    dx_size, dw_size = grads(kept.abs(), w.abs(), dy.abs())
    want = (y, dx, dw, dy.sum((0, 2, 3)))
    size = (y_size, dx_size, dw_size, dy.abs().sum((0, 2, 3)))
    return want, tuple((half_step(v, torch.float16) if i < 3 else 0) + CONST * s for i, (v, s) in enumerate(zip(want, size)))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, C, 13, 11), (1, C, 1, 1), (3, C, 32, 7)], ids=str)
@pytest.mark.parametrize("checkpoint8", [False, True])
def test_block(shape, checkpoint8):
    block, (x, dy) = make_block(21), make_data(shape, 22)
    x.requires_grad_(True)
    half = lambda t: t.detach().half().contiguous(memory_format=CL).requires_grad_(True)  # noqa: E731
    w1, w2 = half(block.conv1.weight), half(block.conv2.weight)
    b1 = block.conv1.bias
    n1, n2 = block.norm1, block.norm2

    def conv(x, w, b, pad):
        if checkpoint8:
            return conv2d_gw8_checkpoint8(x, w, b, padding_y=pad, padding_x=pad, groups=C // 8)
        return conv2d_gw8(x, w, b, 1, pad, pad, 1, C // 8)

    t1 = conv(x, w1, b1, 1)
    t2 = groupnorm_2d(t1, GROUPS[0], n1.weight, n1.bias, activation="silu", checkpoint8=checkpoint8)
    t3 = conv(t2, w2, None, 2)
    t4 = groupnorm_2d(t3, GROUPS[1], n2.weight, n2.bias, activation="gelu", checkpoint8=checkpoint8)
    leaves = (x, w1, b1, n1.weight, n1.bias, w2, n2.weight, n2.bias)
    gx, gw1, gb1, gn1w, gn1b, gw2, gn2w, gn2b, g1, g2, g3 = torch.autograd.grad(t4, (*leaves, t1, t2, t3), dy)
    assert device_status() == 0

    for name, got, (want, tol) in (
            ("conv1", (t1, gx, gw1, gb1), conv_reference(x, w1, b1, g1, 1, checkpoint8)),
            ("conv2", (t3, g2, gw2), conv_reference(t2, w2, None, g3, 2, checkpoint8))):
        for what, g, v, e in zip(("y", "dx", "dw", "db"), got, want, tol):
            assert_within(g, v, e, f"{name} {what}")
    for name, t, groups, norm, act, out, g_out, got in (
            ("norm1", t1, GROUPS[0], n1, "silu", t2, g2, (g1, gn1w, gn1b)),
            ("norm2", t3, GROUPS[1], n2, "gelu", t4, dy, (g3, gn2w, gn2b))):
        ref = Reference(t, groups, norm.weight, norm.bias, act=act, dy=g_out, checkpoint8=checkpoint8)
        assert_within(out, ref.y, ref.y_tol, f"{name} y")
        for what, g in zip(("dx", "dweight", "dbias"), got):
            assert_within(g, getattr(ref, what), getattr(ref, what + "_tol"), f"{name} {what}")

    # the transformed module runs the same kernels
    fast = transform(block, group_norm=True, checkpoint8=checkpoint8)
    with torch.autocast("cuda", dtype=torch.float16):
        y = fast(x)
    assert torch.equal(y, x + t4)
    grads = torch.autograd.grad(y, (x, block.conv1.weight, b1, n1.weight, n1.bias, block.conv2.weight, n2.weight, n2.bias), dy)
    assert torch.equal(grads[0], gx + dy)
    for g, want in zip(grads[1:], (gw1, gb1, gn1w, gn1b, gw2, gn2w, gn2b)):
        assert torch.equal(g, want.to(g.dtype))


@pytest.mark.gpu
def test_captured_block():
    """A captured training step of the block on new data, and two captured steps that share nothing."""
    block, (x, dy) = make_block(23), make_data((2, C, 14, 14), 24)
    fast = transform(block, group_norm=True, checkpoint8=True)
    params = list(fast.parameters())

    def step():
        with torch.autocast("cuda", dtype=torch.float16, cache_enabled=False):
            y = fast(x)
        return (y.detach(), *torch.autograd.grad(y, params, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step())
    for seed in (25, 26):
        x2, dy2 = make_data((2, C, 14, 14), seed)
        x.copy_(x2), dy.copy_(dy2)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = step()
        for out in outs:
            assert all(torch.equal(p, q) for p, q in zip(out, want))
    assert device_status() == 0


@pytest.mark.gpu
def test_example_runs_with_8_bit_checkpoints():
    """The example network trains with its convolutions' inputs kept in 8 bits: the same loss, finite gradients."""
    from spio_b200.examples.convnext_gw8 import ConvNeXtGw8, train_step

    torch.manual_seed(27)
    model = ConvNeXtGw8(widths=(32, 64), depths=(1, 1), num_classes=10).cuda().to(memory_format=CL)
    images = torch.randn(2, 3, 64, 64, device="cuda").contiguous(memory_format=CL)
    labels = torch.randint(0, 10, (2,), device="cuda")
    want = train_step(transform(model), images, labels)
    model.zero_grad(set_to_none=True)
    fast = transform(model, checkpoint8=True)
    assert torch.equal(train_step(fast, images, labels), want)
    assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in fast.parameters())


def test_transform_of_group_norms():
    block = Block()
    kept = transform(block)
    assert isinstance(kept.norm1, nn.GroupNorm) and not kept.conv1.checkpoint8
    fast = transform(block, group_norm=True, checkpoint8=True)
    assert (fast.norm1.activation, fast.norm2.activation) == ("silu", "gelu")
    assert fast.norm1.checkpoint8 and fast.conv1.checkpoint8 and "checkpoint8=True" in repr(fast.conv1)
    assert not hasattr(fast, "act1") and fast.norm1.weight is block.norm1.weight
    assert sorted(fast.state_dict()) == sorted(block.state_dict())
    assert len([n for n in fast.graph.nodes if n.op == "call_module"]) == 4
    # a transformed model can be transformed again: its layers are looked through
    names = [getattr(n.target, "__name__", "") for n in transform(fast, group_norm=True).graph.nodes]
    assert names.count("conv2d_gw8_checkpoint8") == 2 and sum("groupnorm_2d" in n for n in names) == 2


def test_transform_keeps_activations_that_it_must_not_take_in():
    class Net(nn.Module):
        def __init__(self):
            super().__init__()
            self.norm, self.shared, self.odd = nn.GroupNorm(4, 32), nn.GroupNorm(4, 32), nn.GroupNorm(4, 36)
            self.wide = nn.GroupNorm(1, 4096)
            self.relu, self.silu, self.tanh = nn.ReLU(), nn.SiLU(), nn.Tanh()

        def forward(self, x, z, q):
            a = self.norm(x)
            both = self.relu(a) + a                                             # the value before the ReLU is used too
            return self.relu(self.shared(both)) + self.silu(self.shared(x)), self.tanh(self.odd(z)), self.wide(q)

    net = Net()
    fast = transform(net, group_norm=True)
    assert fast.norm.activation == "none" and fast.shared.activation == "none"
    assert isinstance(fast.odd, nn.GroupNorm) and isinstance(fast.wide, nn.GroupNorm)
    x, z, q = torch.randn(2, 32, 3, 3), torch.randn(2, 36, 3, 3), torch.randn(1, 4096, 1, 1)
    for name in ("norm", "shared"):                 # the graph itself, with torch's layer back in place
        setattr(fast, name, getattr(net, name))
    assert all(torch.equal(p, q) for p, q in zip(fast(x, z, q), net(x, z, q)))


@pytest.mark.parametrize("checkpoint8", [False, True])
def test_transform_with_a_layer_class_of_the_user(monkeypatch, checkpoint8):
    """A class in the list of layers needs no more than it always did: match and from_torch_module(module)."""
    from spio_b200.transform import _transform

    class Twice(nn.Module):
        @staticmethod
        def match(module):
            return isinstance(module, nn.Identity)

        @staticmethod
        def from_torch_module(module):
            return Twice()

        def forward(self, x):
            return 2 * x

    monkeypatch.setattr(_transform, "spio_modules_classes", _transform.spio_modules_classes + [Twice])
    fast = _transform.transform(nn.Sequential(nn.Identity(), nn.Conv2d(16, 16, 3, groups=2)), checkpoint8=checkpoint8)
    assert isinstance(getattr(fast, "0"), Twice) and getattr(fast, "1").checkpoint8 == checkpoint8
