"""The 8-bit form of activations and the convolution that keeps its input in it."""

import gc

import pytest
import torch

from oracle import oracle as O
from spio_b200.functional import (checkpoint8_pack, checkpoint8_unpack, conv2d_gw8, conv2d_gw8_checkpoint8,
                                  conv2d_gw8_checkpoint8_op)
from spio_b200.kernels import device_status
from tests.norm_reference import blocks_of, restored

pytestmark = pytest.mark.gpu
CL = torch.channels_last
TYPES = [torch.float16, torch.bfloat16, torch.float32]
SHAPES = [(1, 8, 1, 1), (2, 24, 17, 5), (3, 40, 7, 3), (1, 1024, 3, 5), (2, 64, 56, 56), (513, 8, 1, 1)]


def image(values, c=8):
    """The values as the pixels' channels of a (1, c, 1, n / c) image."""
    return values.reshape(1, 1, -1, c).permute(0, 3, 1, 2)


def check_exact(x):
    codes, exponents = checkpoint8_pack(x)
    want_codes, want_scale = blocks_of(x)
    assert codes.dtype == torch.int8 and exponents.dtype == torch.uint8
    assert codes.is_contiguous(memory_format=CL) and exponents.is_contiguous(memory_format=CL)
    assert torch.equal(codes.cpu().long(), want_codes)
    assert torch.equal(torch.exp2(exponents.cpu().double() - 127), want_scale)
    back = checkpoint8_unpack(codes, exponents, x.dtype)
    assert back.dtype == x.dtype and back.is_contiguous(memory_format=CL)
    assert torch.equal(back.double().cpu(), restored(x))
    # half a step of the block's scale, or up to a whole one at the top of the type's range
    err = (back.double().cpu() - x.double().cpu()).abs()
    assert bool((err <= 0.5 * want_scale.repeat_interleave(8, 1)).all()) or float(x.abs().max()) > 0.99 * torch.finfo(x.dtype).max


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_pack_and_unpack_are_exact(shape, dtype):
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(shape, generator=gen) * torch.exp(2 * torch.randn(shape, generator=gen))
    check_exact(x.to(dtype).cuda().contiguous(memory_format=CL))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_every_fp16_and_bf16_value_as_the_largest_and_ties(dtype):
    bits = torch.arange(0, 1 << 16, dtype=torch.int32).to(torch.int16)
    source = torch.bfloat16 if dtype is torch.bfloat16 else torch.float16
    top = bits.view(source)
    top = top[top.isfinite()].to(dtype)
    # the value beside fractions of it: halves of a step, which tie, among them
    fractions = torch.tensor([1.0, 0.5, 1 / 3, 63.5 / 127, 2.5 / 128, -1.5 / 64, 0.0, -0.7])
    block = (top.float()[:, None] * fractions).to(dtype)
    check_exact(image(block.reshape(-1)).cuda())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_range_ends(dtype):
    info = torch.finfo(dtype)
    tiny = info.smallest_normal * info.eps
    rows = [[info.max] * 8, [info.max, -info.max, info.max / 2, 1, 0, tiny, -tiny, info.max * (1 - 2 ** -7)],
            [tiny] * 8, [0.0] * 8, [-0.0] * 8, [info.smallest_normal, tiny, 0, 0, -tiny * 3, 0, 0, 0],
            [127.0, 126.5, 125.5, 63.5, -0.5, 0.5, 1.5, -127.0], [127.5, 1, 2, 3, 4, 5, 6, 7]]
    x = image(torch.tensor(rows, dtype=torch.float64).to(dtype).reshape(-1)).cuda()
    check_exact(x)
    back = checkpoint8_unpack(*checkpoint8_pack(x), dtype)
    assert bool(back.isfinite().all())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_nonfinite_blocks_come_back_as_nan(dtype, bad):
    x = torch.randn(2, 24, 3, 3, generator=torch.Generator().manual_seed(2)).to(dtype).cuda().contiguous(memory_format=CL)
    x[1, 13, 2, 0] = bad
    codes, exponents = checkpoint8_pack(x)
    back = checkpoint8_unpack(codes, exponents, dtype)
    assert bool(back[1, 8:16, 2, 0].isnan().all()) and int(exponents[1, 1, 2, 0]) == 255
    back[1, 8:16, 2, 0] = 0
    assert bool(back.isfinite().all())


def test_layouts_and_empty_tensors():
    x = torch.randn(2, 16, 5, 6, device="cuda").half()
    a, b = checkpoint8_pack(x), checkpoint8_pack(x.contiguous(memory_format=CL))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    back = checkpoint8_unpack(b[0], b[1])
    assert torch.equal(checkpoint8_unpack(b[0].contiguous(), b[1].contiguous()), back)     # NCHW order of both
    off = torch.empty(x.numel() + 1, device="cuda", dtype=x.dtype)[1:].view(2, 5, 6, 16).permute(0, 3, 1, 2).copy_(x)
    assert torch.equal(checkpoint8_pack(off)[0], b[0])
    odd = torch.empty(b[1].numel() + 1, device="cuda", dtype=torch.uint8)[1:].view(2, 5, 6, 2).permute(0, 3, 1, 2).copy_(b[1])
    assert torch.equal(checkpoint8_unpack(b[0], odd), back)                               # exponents at an odd address
    codes, exponents = checkpoint8_pack(x[:0])
    assert codes.shape == (0, 16, 5, 6) and exponents.shape == (0, 2, 5, 6)
    assert checkpoint8_unpack(codes, exponents).shape == (0, 16, 5, 6)
    for dtype in TYPES:     # any exponent byte stands for its power of two
        e = torch.arange(256, dtype=torch.uint8, device="cuda").reshape(1, 1, 1, 256)
        c = torch.arange(-128, 128, dtype=torch.int8, device="cuda").repeat(8).reshape(1, 8, 1, 256)
        want = (c.double() * torch.exp2(e.double() - 127)).where(e < 255, torch.nan)
        want = torch.where(e == 0, 0.0, want)
        assert torch.equal(checkpoint8_unpack(c, e, dtype).nan_to_num(nan=7.0, posinf=8.0, neginf=9.0),
                           want.to(torch.float32).to(dtype).nan_to_num(nan=7.0, posinf=8.0, neginf=9.0))


def test_refusals():
    x = torch.zeros(2, 16, 3, 3, device="cuda").half()
    codes, exponents = checkpoint8_pack(x)
    for call in (lambda: checkpoint8_pack(x.cpu()), lambda: checkpoint8_pack(x[:, :12]), lambda: checkpoint8_pack(x[0]),
                 lambda: checkpoint8_pack(x.double()), lambda: checkpoint8_unpack(codes, exponents[:, :1]),
                 lambda: checkpoint8_unpack(codes, exponents, torch.float64), lambda: checkpoint8_unpack(codes.short(), exponents),
                 lambda: checkpoint8_unpack(codes, exponents.cpu()),
                 lambda: conv2d_gw8_checkpoint8(x, torch.zeros(16, 8, 3, 3, device="cuda"), groups=2)):
        with pytest.raises(Exception):
            call()


CONVS = [O.Shape(2, 32, 11, 13, 3, 3, 1, 1), O.Shape(3, 96, 9, 31, 5, 5, 2, 2), O.Shape(1, 64, 30, 7, 1, 3, 0, 1),
         O.Shape(4, 8, 6, 6, 2, 2, 1, 1)]


@pytest.mark.parametrize("sh", CONVS, ids=str)
@pytest.mark.parametrize("has_bias", [False, True])
def test_convolution(sh, has_bias):
    x, w, b, dy = O.make_inputs(sh, seed=31, bias=has_bias)
    put = lambda t: None if t is None else (t.cuda().contiguous(memory_format=CL) if t.dim() == 4 else t.cuda()).requires_grad_(True)  # noqa: E731
    xd, wd, bd = put(x), put(w), put(b)
    leaves = [t for t in (xd, wd, bd) if t is not None]
    args = dict(padding_y=sh.pad_h, padding_x=sh.pad_w, groups=sh.groups)
    g = dy.cuda().contiguous(memory_format=CL)
    y = conv2d_gw8_checkpoint8(xd, wd, bd, **args)
    grads = torch.autograd.grad(y, leaves, g)
    plain = conv2d_gw8(xd, wd, bd, **args)
    want = list(torch.autograd.grad(plain, leaves, g))
    # the weight gradient is that of the convolution of the restored input, by the same kernels
    back = checkpoint8_unpack(*checkpoint8_pack(xd)).requires_grad_(True)
    (want[1],) = torch.autograd.grad(conv2d_gw8(back, wd, bd, **args), wd, g)
    assert device_status() == 0
    assert torch.equal(y, plain)
    assert all(torch.equal(p, q) for p, q in zip(grads, want))
    dw = O.torch_grads(restored(x).half(), w, dy, sh)[1]
    O.assert_close(grads[1], dw, sh, "wgrad", str(sh), atol_scale=1.0 + 1e-3 * float(dw.abs().max())
                   / O.reference_tolerance(sh, "wgrad")[0])


def test_convolution_under_autocast_and_with_frozen_parts():
    sh = CONVS[0]
    x, w, _, dy = O.make_inputs(sh, seed=32, bias=False)
    x32, w32 = x.float().cuda().requires_grad_(True), w.float().cuda().requires_grad_(True)
    with torch.autocast("cuda", dtype=torch.float16):
        y = conv2d_gw8_checkpoint8(x32, w32, None, padding_y=1, padding_x=1, groups=sh.groups)
        ref = conv2d_gw8(x32, w32, None, 1, 1, 1, 1, sh.groups)
    assert y.dtype == torch.float32 and torch.equal(y, ref)
    g = dy.float().cuda()
    dx, dw = torch.autograd.grad(y, (x32, w32), g)
    rx, _ = torch.autograd.grad(ref, (x32, w32), g)
    assert torch.equal(dx, rx) and dw.dtype == torch.float32
    frozen = conv2d_gw8_checkpoint8(x.cuda().requires_grad_(True), w.cuda(), None, padding_y=1, padding_x=1, groups=sh.groups)
    assert frozen.requires_grad
    only_weight = conv2d_gw8_checkpoint8(x.cuda(), w.cuda().requires_grad_(True), None, padding_y=1, padding_x=1, groups=sh.groups)
    only_weight.backward(dy.cuda())
    # asked for the input gradient alone, the input's values are not restored
    xd, wd = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    y, _, _ = conv2d_gw8_checkpoint8_op(xd, wd, None, 1, 1, 1, 1, sh.groups)
    (dx,) = torch.autograd.grad(y, xd, dy.cuda())
    (rx,) = torch.autograd.grad(conv2d_gw8(xd, wd, None, 1, 1, 1, 1, sh.groups), xd, dy.cuda())
    assert torch.equal(dx, rx)


def test_second_derivatives_are_refused():
    sh = CONVS[0]
    x, w, _, dy = O.make_inputs(sh, seed=33, bias=False)
    xd, wd = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    y = conv2d_gw8_checkpoint8(xd, wd, None, padding_y=1, padding_x=1, groups=sh.groups)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(y, (xd, wd), dy.cuda(), create_graph=True)


def test_compiled_calls():
    """They take the Python operator: the same values as the plain eager calls."""
    sh = CONVS[0]
    x, w, b, dy = (t.cuda() for t in O.make_inputs(sh, seed=34))
    f = lambda x, w: (conv2d_gw8_checkpoint8(x, w, b, padding_y=1, padding_x=1, groups=sh.groups) * dy).sum()  # noqa: E731
    leaves = [t.clone().requires_grad_(True) for t in (x, w)]
    want = torch.autograd.grad(f(*leaves), leaves)
    compiled = torch.compile(f, backend="aot_eager", fullgraph=True)
    got = torch.autograd.grad(compiled(*leaves), leaves)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_memory_kept_for_the_backward_pass():
    """1.125 bytes a value instead of 2, once the input itself has been dropped."""
    sh = O.Shape(8, 64, 56, 56, 3, 3, 1, 1)
    w = torch.randn(64, 8, 3, 3, device="cuda").half().requires_grad_(True)
    kept = []
    for conv in (conv2d_gw8, conv2d_gw8_checkpoint8):
        gc.collect()      # what earlier tests left in cycles is not to be freed in between
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        x = torch.randn(sh.n, sh.c, sh.h, sh.w, device="cuda").half().contiguous(memory_format=CL)
        y = conv(x, w, None, padding_y=1, padding_x=1, groups=8)
        size = y.numel()
        del x
        torch.cuda.synchronize()
        kept.append(torch.cuda.memory_allocated() - before - 2 * size)
        del y
    assert kept[0] >= 2 * size and kept[1] <= 1.125 * size + (1 << 20), kept


def test_a_frozen_weight_keeps_no_input():
    """Without a weight gradient nothing reads the input again, and neither it nor its codes are kept."""
    sh = O.Shape(8, 64, 56, 56, 3, 3, 1, 1)
    w, b = torch.randn(64, 8, 3, 3, device="cuda").half(), torch.randn(64, device="cuda")
    conv2d_gw8_checkpoint8(torch.zeros(8, 64, 56, 56, device="cuda").half(), w, b, padding_y=1, padding_x=1, groups=8)
    for trained_bias in (False, True):
        bias = b.clone().requires_grad_(trained_bias)
        gc.collect()
        torch.cuda.synchronize()
        leaf = torch.randn(sh.n, sh.c, sh.h, sh.w, device="cuda").half().contiguous(memory_format=CL).requires_grad_(True)
        dy = torch.randn_like(leaf)
        before = torch.cuda.memory_allocated()
        x = leaf * 2
        y = conv2d_gw8_checkpoint8(x, w, bias, padding_y=1, padding_x=1, groups=8)
        size = y.numel()
        del x
        torch.cuda.synchronize()
        assert torch.cuda.memory_allocated() - before - 2 * size <= 1 << 20
        torch.cuda.reset_peak_memory_stats()
        held = torch.cuda.memory_allocated()
        got = torch.autograd.grad(y, [leaf] + [bias] * trained_bias, dy)
        torch.cuda.synchronize()
        assert torch.cuda.max_memory_allocated() - held <= 2 * (2 * size) + (1 << 20)      # the two gradients of the input
        del y
        want = torch.autograd.grad(conv2d_gw8(leaf * 2, w, bias, 1, 1, 1, 1, 8), [leaf] + [bias] * trained_bias, dy)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        del got, want, leaf, dy


def test_a_frozen_weight_under_autocast():
    """The Python operator, which packs but keeps nothing."""
    sh = O.Shape(8, 64, 56, 56, 3, 3, 1, 1)
    w = torch.randn(64, 8, 3, 3, device="cuda")

    def step(conv, x):
        with torch.autocast("cuda", dtype=torch.float16):
            return conv(x, w, None, 1, 1, 1, 1, 8)

    kept = []
    for conv in (conv2d_gw8, conv2d_gw8_checkpoint8):
        x = torch.randn(sh.n, sh.c, sh.h, sh.w, device="cuda").contiguous(memory_format=CL).requires_grad_(True)
        step(conv, x)
        gc.collect()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = step(conv, x)
        torch.cuda.synchronize()
        kept.append(torch.cuda.memory_allocated() - before - 4 * y.numel())
        dy = torch.randn_like(y)
        assert torch.equal(torch.autograd.grad(y, x, dy)[0], torch.autograd.grad(step(conv2d_gw8, x), x, dy)[0])
        del y, dy
    assert kept[1] <= 1 << 20 < kept[0], kept
