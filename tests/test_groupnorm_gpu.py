"""Group norm with an activation (spio::groupnorm_2d): forward, backward, the 8-bit checkpoint, special values,
layouts, streams and CUDA graphs, against the definition in float64."""

import itertools
import threading

import pytest
import torch
from torch import nn

from spio_b200.functional import conv2d_gw8_checkpoint8, groupnorm_2d, groupnorm_2d_backward_op, groupnorm_2d_op
from spio_b200.layers import GroupNorm2d
from spio_b200.transform import transform
from tests.norm_reference import CONST, PLANNED, Reference, assert_within, half_step, plan_of

pytestmark = pytest.mark.gpu
CL = torch.channels_last
TYPES = [torch.float16, torch.bfloat16, torch.float32]
ACTS = ["none", "relu", "silu", "gelu"]

# (n, c, h, w, groups): channels a group from 1 to 2048, groups that straddle pieces of 8 channels (3, 5, 6, 12, 20),
# one pixel, odd sizes, wide images, more channels than one slab, many images, one image over many CTAs
SHAPES = [
    (1, 8, 1, 3, 1), (2, 8, 3, 5, 8), (3, 24, 7, 5, 8), (2, 40, 9, 11, 8), (2, 96, 14, 14, 32), (3, 96, 5, 7, 16),
    (1, 256, 16, 16, 32), (2, 160, 13, 9, 8), (70, 64, 3, 3, 8), (1, 64, 131, 67, 32), (2, 1024, 4, 4, 1),
    (1, 2048, 3, 3, 1), (2, 1536, 3, 2, 512), (5, 16, 1, 1, 1), (2, 768, 7, 7, 32), (1, 32, 200, 180, 4),
    (2, 520, 6, 6, 5), (300, 8, 2, 2, 2),
]


def make(shape, dtype, seed=0, affine=True, offset=0.5):
    n, c, h, w = shape
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((n, c, h, w), generator=gen) * torch.exp(0.4 * torch.randn(1, c, 1, 1, generator=gen))
    x = (x + offset * torch.randn(1, c, 1, 1, generator=gen)).to(dtype)
    dy = torch.randn((n, c, h, w), generator=gen).to(dtype)
    wt = 1 + 0.3 * torch.randn(c, generator=gen) if affine else None
    bs = 0.3 * torch.randn(c, generator=gen) if affine else None
    put = lambda t: None if t is None else (t.cuda().contiguous(memory_format=CL) if t.dim() == 4 else t.cuda())  # noqa: E731
    return put(x), put(dy), put(wt), put(bs)


def check_all(shape, groups, dtype, act, checkpoint8=False, affine=True, seed=0, eps=1e-5, offset=0.5):
    x, dy, w, b = make(shape, dtype, seed, affine, offset)
    ref = Reference(x, groups, w, b, eps, act, dy, checkpoint8)
    leaves = [t.requires_grad_(True) for t in (x, w, b) if t is not None]
    y = groupnorm_2d(x, groups, w, b, eps, act, checkpoint8)
    assert y.dtype == dtype and y.is_contiguous(memory_format=CL)
    assert_within(y, ref.y, ref.y_tol, "y")
    grads = torch.autograd.grad(y, leaves, dy)
    assert_within(grads[0], ref.dx, ref.dx_tol, "dx")
    assert grads[0].dtype == dtype
    if affine:
        assert_within(grads[1], ref.dweight, ref.dweight_tol, "dweight")
        assert_within(grads[2], ref.dbias, ref.dbias_tol, "dbias")


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_forward_and_backward(shape, dtype):
    act = ACTS[SHAPES.index(shape) % 4]
    check_all(shape[:4], shape[4], dtype, act, seed=1)


@pytest.mark.parametrize("shape", SHAPES[1::2], ids=str)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_checkpoint8(shape, dtype):
    act = ACTS[(SHAPES.index(shape) // 2 + 2) % 4]
    check_all(shape[:4], shape[4], dtype, act, checkpoint8=True, seed=2)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("checkpoint8", [False, True])
def test_activations(act, dtype, checkpoint8):
    check_all((3, 48, 10, 9), 6, dtype, act, checkpoint8, seed=3)
    check_all((2, 48, 10, 9), 16, dtype, act, checkpoint8, affine=False, seed=4)


def test_statistics_of_data_far_from_zero():
    """An offset of 1000 standard deviations: differences to a pivot keep the variance."""
    x, _, _, _ = make((2, 64, 40, 30), torch.float32, seed=5)
    x = (x + 1000).requires_grad_(False)
    _, stats, _, _ = groupnorm_2d_op(x, None, None, 8, 1e-5, "none", False)
    ref = Reference(x, 8)
    torch.testing.assert_close(stats[..., 0].double().cpu(), ref.mean, rtol=2.0 ** -22, atol=0)
    torch.testing.assert_close(stats[..., 1].double().cpu(), ref.rstd, rtol=2e-5, atol=0)
    # a constant image has the mean itself and no variance
    for value in (0.0, 3.0, 1000.0):
        x = torch.full((2, 24, 37, 21), value, device="cuda").contiguous(memory_format=CL)
        y, stats, _, _ = groupnorm_2d_op(x, None, None, 8, 1e-5, "none", False)
        assert torch.equal(y, torch.zeros_like(y)) and bool((stats[..., 0] == value).all())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("checkpoint8", [False, True])
def test_nonfinite_values_stay_in_their_group(dtype, bad, checkpoint8):
    x, dy, w, b = make((3, 32, 9, 8), dtype, seed=6)
    clean = groupnorm_2d(x, 4, w, b, activation="relu")
    x[1, 11, 4, 3] = bad                              # group 1 (channels 8 .. 15) of image 1
    x.requires_grad_(True)
    y = groupnorm_2d(x, 4, w, b, activation="relu", checkpoint8=checkpoint8)
    hit = torch.zeros_like(y, dtype=torch.bool)
    hit[1, 8:16] = True
    assert bool(y[hit].isnan().all()) and torch.equal(y[~hit], clean[~hit])
    (dx,) = torch.autograd.grad(y, x, dy)
    assert bool(dx[hit].isnan().all()) and bool(dx[~hit].isfinite().all())


def test_empty_tensors():
    w, b = torch.ones(16, device="cuda", requires_grad=True), torch.zeros(16, device="cuda", requires_grad=True)
    for shape, c8 in itertools.product([(0, 16, 4, 4), (3, 16, 0, 5)], [False, True]):
        x = torch.empty(shape, device="cuda", dtype=torch.float16, requires_grad=True)
        y = groupnorm_2d(x, 4, w, b, checkpoint8=c8)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
        assert y.shape == shape and dx.shape == shape
        assert torch.equal(dw, torch.zeros_like(dw)) and torch.equal(db, torch.zeros_like(db))


def test_layouts_offsets_and_expanded_gradients():
    x, dy, w, b = make((2, 32, 6, 7), torch.float16, seed=7)
    want = groupnorm_2d(x, 8, w, b, activation="silu")
    assert torch.equal(groupnorm_2d(x.contiguous(), 8, w, b, activation="silu"), want)       # NCHW order
    padded = torch.empty(x.numel() + 1, device="cuda", dtype=x.dtype)[1:]                    # off a 16-byte boundary
    off = padded.view(2, 6, 7, 32).permute(0, 3, 1, 2).copy_(x)
    assert off.data_ptr() % 16 and torch.equal(groupnorm_2d(off, 8, w, b, activation="silu"), want)
    wide = torch.randn(2, 64, 6, 7, device="cuda").half().contiguous(memory_format=CL)       # a slice of channels
    part = wide[:, 16:48]
    assert torch.equal(groupnorm_2d(part, 8, w, b), groupnorm_2d(part.clone(), 8, w, b))
    strided = torch.stack([w, w], 1)[:, 0]
    assert not strided.is_contiguous() and torch.equal(groupnorm_2d(x, 8, strided, b, activation="silu"), want)
    xs = x.clone().requires_grad_(True)
    (got,) = torch.autograd.grad(groupnorm_2d(xs, 8, w, b, activation="silu").sum(), xs)     # an expanded scalar
    (ref,) = torch.autograd.grad(groupnorm_2d(xs, 8, w, b, activation="silu"), xs, torch.ones_like(x))
    assert torch.equal(got, ref)


def test_only_requested_gradients_and_reproducibility():
    x, dy, w, b = make((4, 64, 28, 28), torch.bfloat16, seed=8)
    _, stats, _, _ = groupnorm_2d_op(x, w, b, 8, 1e-5, "gelu", False)
    full = groupnorm_2d_backward_op(dy, x, None, None, stats, w, b, 8, "gelu", True, True, True)
    again = groupnorm_2d_backward_op(dy, x, None, None, stats, w, b, 8, "gelu", True, True, True)
    assert all(torch.equal(p, q) for p, q in zip(full, again))
    for want in itertools.product([False, True], repeat=3):
        got = groupnorm_2d_backward_op(dy, x, None, None, stats, w, b, 8, "gelu", *want)
        for g, f, on in zip(got, full, want):
            assert torch.equal(g, f) if on else g.numel() == 0
    # a frozen norm: weight and bias without gradients
    xs = x.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(groupnorm_2d(xs, 8, w, b, activation="gelu"), xs, dy)
    assert torch.equal(dx, full[0])


def test_gradient_against_differences():
    """fp32: the directional derivative of the loss against a central difference in float64 steps of 1e-3 (whose
    own error is h^2 / 6 of the third derivative, and 2^-23 / h of the outputs' rounding: 1e-3 in all)."""
    x, dy, w, b = make((2, 16, 5, 6), torch.float32, seed=9)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    for act in ("none", "silu", "gelu"):
        grads = torch.autograd.grad(groupnorm_2d(x, 4, w, b, activation=act), leaves, dy)
        for i, leaf in enumerate(leaves):
            step = torch.randn(leaf.shape, generator=torch.Generator().manual_seed(i)).to(leaf.device)
            ends = []
            for sign in (1, -1):
                moved = [t.detach() + (sign * 1e-3 * step if j == i else 0) for j, t in enumerate(leaves)]
                ends.append((groupnorm_2d(moved[0], 4, moved[1], moved[2], activation=act).double() * dy.double()).sum())
            numeric = float(ends[0] - ends[1]) / 2e-3
            direct = float((grads[i].double() * step.double()).sum())
            scale = float((grads[i].double() * step.double()).norm()) + float(dy.double().norm())
            assert abs(numeric - direct) <= 1e-3 * scale, (act, i)


def test_absent_weight_or_bias():
    x, dy, w, b = make((2, 32, 6, 5), torch.float32, seed=15)
    for weight, bias in ((w, None), (None, b)):
        ref = Reference(x, 4, weight, bias, 1e-5, "silu", dy)
        given = (weight if weight is not None else bias).clone().requires_grad_(True)
        xs = x.clone().requires_grad_(True)
        y = groupnorm_2d(xs, 4, given if weight is not None else None, given if bias is not None else None, activation="silu")
        assert_within(y, ref.y, ref.y_tol, "y")
        dx, dv = torch.autograd.grad(y, (xs, given), dy, retain_graph=True)
        assert_within(dx, ref.dx, ref.dx_tol, "dx")
        assert_within(dv, ref.dweight if weight is not None else ref.dbias,
                      ref.dweight_tol if weight is not None else ref.dbias_tol, "vector")
        (dv2,) = torch.autograd.grad(y, (given,), dy)      # without the input gradient
        assert torch.equal(dv, dv2)


def test_second_derivatives_are_refused():
    x, dy, w, b = make((2, 16, 4, 4), torch.float32, seed=16)
    x.requires_grad_(True)
    y = groupnorm_2d(x, 4, w, b, activation="silu")
    (dx,) = torch.autograd.grad(y, x, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        dx.square().sum().backward()


@pytest.mark.parametrize("shape,groups,act,dtype", [((4, 24, 144, 122), 2, "relu", torch.float16),
                                                    ((2, 8, 223, 200), 1, "none", torch.float32)], ids=str)
def test_sizes_where_only_the_checkpoint_takes_two_launches(shape, groups, act, dtype):
    """(On a B200.)  The scratch memory has to serve the form that needs more of it."""
    for checkpoint8 in (False, True):
        check_all(shape, groups, dtype, act, checkpoint8, seed=18)


@pytest.mark.parametrize("shape,groups,act,dtype", [((1, 160, 140, 170), 32, "silu", torch.float16),
                                                    ((1, 256, 140, 170), 64, "gelu", torch.bfloat16),
                                                    ((1, 520, 100, 111), 13, "silu", torch.float16),
                                                    ((1, 448, 75, 131), 7, "none", torch.float32)], ids=str)
def test_one_large_image(shape, groups, act, dtype):
    """(On a B200.)  Two launches with several slabs of channels, the last of them narrower."""
    for checkpoint8 in (False, True):
        check_all(shape, groups, dtype, act, checkpoint8, seed=23)


@pytest.mark.parametrize("shape,groups", [((1500, 24, 2, 1), 3), ((4097, 8, 1, 3), 1), ((2049, 64, 3, 3), 8)], ids=str)
def test_many_small_images(shape, groups):
    """Gradients of weight and bias that are summed over the images by the CTAs of a cluster."""
    check_all(shape, groups, torch.float16, "relu", seed=21)
    check_all(shape, groups, torch.bfloat16, "gelu", True, seed=22)


def test_forward_mode_derivatives_are_refused():
    x, dy, w, b = make((2, 16, 4, 4), torch.float32, seed=19)
    stats = groupnorm_2d_op(x, w, b, 4, 1e-5, "none", False)[1]
    with torch.autograd.forward_ad.dual_level():
        dual = lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: groupnorm_2d(dual(x), 4, w, b), lambda: groupnorm_2d(x, 4, dual(w), b),
                     lambda: groupnorm_2d(x, 4, w, dual(b)),
                     lambda: groupnorm_2d_backward_op(dual(dy), x, None, None, stats, w, b, 4, "none", True, True, True)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_functional_transforms_are_refused():
    """(As they are by the other operators of the package.)"""
    x, _, w, b = make((2, 16, 4, 4), torch.float32, seed=20)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda x: groupnorm_2d(x, 4, w, b, activation="gelu").sum())(x)


def test_compiled_model_traces_through_the_operator():
    """torch.compile sees one opaque operator (eager backend: nothing else is compiled)."""
    x, _, w, b = make((2, 32, 6, 6), torch.float16, seed=17)
    layer = GroupNorm2d(4, 32, activation="gelu", checkpoint8=True).cuda()
    with torch.no_grad():
        layer.weight.copy_(w), layer.bias.copy_(b)
    compiled = torch.compile(layer, backend="aot_eager", fullgraph=True)
    xs, xc = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    y, yc = layer(xs), compiled(xc)
    assert torch.equal(y, yc)
    y.sum().backward(), yc.sum().backward()
    assert torch.equal(xs.grad, xc.grad)


def test_autocast_keeps_the_data_type():
    x, _, w, b = make((2, 32, 6, 6), torch.float32, seed=10)
    w16 = w.half().requires_grad_(True)
    with torch.autocast("cuda", dtype=torch.float16):
        y = groupnorm_2d(x, 4, w16, b, activation="silu")
        y16 = groupnorm_2d(x.half(), 4, w16, b, activation="silu")
    assert y.dtype == torch.float32 and y16.dtype == torch.float16
    assert torch.equal(y, groupnorm_2d(x, 4, w16.float(), b, activation="silu"))
    y.sum().backward()
    assert w16.grad.dtype == torch.float16


def test_module_takes_the_place_of_torch_layers():
    torch.manual_seed(0)
    ref = nn.Sequential(nn.GroupNorm(8, 64), nn.SiLU()).cuda()
    with torch.no_grad():
        ref[0].weight.uniform_(0.5, 1.5), ref[0].bias.uniform_(-0.2, 0.2)
    fused = GroupNorm2d.from_torch_module(ref[0], activation=GroupNorm2d.activation_of(ref[1]))
    assert fused.weight is ref[0].weight and sorted(fused.state_dict()) == ["bias", "weight"]
    x = torch.randn(3, 64, 12, 10, device="cuda").contiguous(memory_format=CL).requires_grad_(True)
    dy = torch.randn_like(x)
    got, want = fused(x), ref(x)
    torch.testing.assert_close(got, want, rtol=1e-5, atol=2e-5)
    params = [x, ref[0].weight, ref[0].bias]
    for g, r in zip(torch.autograd.grad(got, params, dy), torch.autograd.grad(want, params, dy)):
        torch.testing.assert_close(g, r, rtol=1e-4, atol=2e-4)


def test_streams_and_two_calls_at_once():
    x, dy, w, b = make((4, 64, 56, 56), torch.float16, seed=11)
    want = groupnorm_2d(x, 8, w, b, activation="silu")
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = []
    for s in streams:
        with torch.cuda.stream(s):
            results += [groupnorm_2d(x, 8, w, b, activation="silu") for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(r, want) for r in results)


@pytest.mark.parametrize("checkpoint8", [False, True])
def test_captured_training_step(checkpoint8):
    """Forward and backward captured with a live eager graph of other leaves, replayed on new data, twice in a row;
    two graphs share nothing."""
    shape, groups = (4, 96, 14, 14), 32
    x, dy, w, b = make(shape, torch.float16, seed=12)
    stays = [t.clone().requires_grad_(True) for t in (x, w, b)]
    eager = groupnorm_2d(stays[0], groups, stays[1], stays[2], activation="silu")     # kept alive across the capture
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def step():
        y = groupnorm_2d(leaves[0], groups, leaves[1], leaves[2], activation="silu", checkpoint8=checkpoint8)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

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
    for seed in (13, 14):
        x2, dy2, w2, b2 = make(shape, torch.float16, seed=seed)
        with torch.no_grad():
            for t, v in zip((*leaves, dy), (x2, w2, b2, dy2)):
                t.copy_(v)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = step()
        for out in outs:
            assert all(torch.equal(p, q) for p, q in zip(out, want))
    torch.autograd.grad(eager, stays, torch.ones_like(eager))


def test_refusals():
    x, _, w, b = make((2, 32, 4, 4), torch.float16)
    bad = [
        lambda: groupnorm_2d(x.cpu(), 4),
        lambda: groupnorm_2d(x.double(), 4),
        lambda: groupnorm_2d(x[0], 4),
        lambda: groupnorm_2d(x, 5),
        lambda: groupnorm_2d(x, 0),
        lambda: groupnorm_2d(x[:, :12], 4),
        lambda: groupnorm_2d(x, 4, w.half(), b),
        lambda: groupnorm_2d(x, 4, w[:16], b),
        lambda: groupnorm_2d(x, 4, w.cpu(), b),
        lambda: groupnorm_2d(x, 4, w.view(1, 32, 1, 1), b),
        lambda: groupnorm_2d(x, 4, activation="tanh"),
        lambda: groupnorm_2d(x, 4, eps=-1.0),
        lambda: groupnorm_2d(torch.zeros(1, 4096, 1, 1, device="cuda"), 1),
    ]
    for call in bad:
        with pytest.raises(Exception):
            call()
    torch.cuda.synchronize()
    with pytest.raises(ValueError):
        GroupNorm2d(3, 32)
    with pytest.raises(ValueError):
        GroupNorm2d(4, 36)
    with pytest.raises(ValueError):
        GroupNorm2d(1, 4096)


def test_offsets_beyond_32_bits():
    """An fp16 tensor of 4.4 GB: the last image's values are those of the image alone."""
    n, c, h, w = 70, 64, 700, 700
    x = torch.empty((n, c, h, w), device="cuda", dtype=torch.float16, memory_format=CL).zero_()
    gen = torch.Generator(device="cuda").manual_seed(0)
    x[-1] = torch.randn((c, h, w), device="cuda", generator=gen).half()
    assert x.numel() > 2 ** 31
    y, stats, codes, exponents = groupnorm_2d_op(x, None, None, 8, 1e-5, "none", True)
    one = groupnorm_2d_op(x[-1:].clone(memory_format=CL), None, None, 8, 1e-5, "none", True)
    # the two sizes may be split over CTAs differently: the statistics agree to their rounding
    torch.testing.assert_close(stats[-1:], one[1], rtol=CONST, atol=CONST)
    torch.testing.assert_close(y[-1:], one[0], rtol=2 ** -10, atol=1e-6)
    assert torch.equal(codes[-1:], one[2]) and torch.equal(exponents[-1:], one[3])
    assert not bool(y[0].any())
    dx, dw, db = groupnorm_2d_backward_op(y, None, codes, exponents, stats, None, None, 8, "none", True, True, True)
    assert bool(dx[-1].isfinite().all()) and not bool(dx[0].any())
    torch.testing.assert_close(db, y[-1].double().sum((1, 2)).float(), rtol=0, atol=CONST * float(y[-1].double().abs().sum((1, 2)).max()))


@pytest.mark.parametrize("shape,groups", [((64, 64, 23, 23), 8), ((9, 256, 37, 29), 64), ((7, 24, 61, 53), 3),
                                          ((2051, 8, 3, 1), 1)], ids=str)
def test_clusters_one_behind_the_other(shape, groups):
    """Launches back to back, so that clusters begin where others have just left: their CTAs read each other's sums
    (groups of the slab fewer and more than a warp can take, parts of unequal size, the sum over many images)."""
    x, dy, w, b = make(shape, torch.float16, seed=26)
    check_all(shape, groups, torch.float16, "silu", seed=26)
    results = []
    for _ in range(20):
        y, stats, _, _ = groupnorm_2d_op(x, w, b, groups, 1e-5, "silu", False)
        results.append((y, stats, *groupnorm_2d_backward_op(dy, x, None, None, stats, w, b, groups, "silu", True, True, True)))
    assert all(torch.equal(p, q) for r in results[1:] for p, q in zip(r, results[0]))


@pytest.mark.parametrize("shape,groups,dtype,act,forms", PLANNED, ids=str)
def test_every_form_of_launch(shape, groups, dtype, act, forms):
    """One launch and two, the last slab of channels narrower or not, the same form for all passes or not (that these
    sizes take those forms is tested without a GPU)."""
    for checkpoint8 in (False, True):
        check_all(shape, groups, dtype, act, checkpoint8, seed=27)


def test_two_threads_that_share_a_kernel():
    """Host threads that launch one kernel with different amounts of shared memory, each on a stream of its own."""
    sizes = [((4, 256, 20, 20), 256), ((4, 96, 40, 40), 3)]
    for backward in (False, True):
        plans = [plan_of(s, g, torch.float16, "relu", backward) for s, g in sizes]
        assert all(p["one_launch"] and p["smem_bytes"] > 48 * 1024 for p in plans)
        assert plans[0]["threads"] == plans[1]["threads"] and plans[0]["smem_bytes"] != plans[1]["smem_bytes"], plans
    data = [make(s, torch.float16, seed=31) for s, _ in sizes]
    once = lambda x, dy, w, b, g: (lambda y, st: (y, *groupnorm_2d_backward_op(dy, x, None, None, st, w, b, g, "relu", True,  # noqa: E731
                                                                               True, True)))(*groupnorm_2d_op(x, w, b, g, 1e-5, "relu", False)[:2])
    want = [once(*d, g) for d, (_, g) in zip(data, sizes)]
    torch.cuda.synchronize()
    failures, start = [], threading.Barrier(4)

    def work(i):
        try:
            stream = torch.cuda.Stream()
            start.wait(timeout=60)
            with torch.cuda.stream(stream):
                for _ in range(400):
                    got = once(*data[i % 2], sizes[i % 2][1])
            stream.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(got, want[i % 2]))
        except Exception as e:      # noqa: BLE001
            failures.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads], [t.join() for t in threads]
    assert not failures, failures[0]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape,groups", [((3, 32, 9, 8), 4), ((2, 48, 10, 9), 16), ((1, 696, 35, 32), 6)], ids=str)
@pytest.mark.parametrize("checkpoint8", [False, True])
def test_nonfinite_gradients_where_relu_is_off(dtype, shape, groups, checkpoint8):
    """ReLU selects: an infinite or NaN gradient at a place that it has set to zero is left out, as by torch's layers."""
    x, dy, w, b = make(shape, dtype, seed=28)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = groupnorm_2d(x, groups, w, b, activation="relu", checkpoint8=checkpoint8)
    z = nn.functional.group_norm(x.detach().double(), groups, w.detach().double(), b.detach().double())
    flat = lambda t: t.permute(0, 2, 3, 1).reshape(-1)  # noqa: E731  (a view: channels_last)
    off = flat(z).argsort()[:3]                             # far below zero, from the input's 8-bit form too
    assert not bool(flat(y)[off].any()) and float(flat(z)[off].max()) < -1
    flat(dy)[off] = 0
    want = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    flat(dy)[off] = torch.tensor([float("inf"), float("-inf"), float("nan")], device="cuda", dtype=dtype)
    got = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    assert all(bool(p.isfinite().all()) and torch.equal(p, q) for p, q in zip(got, want))
    on = int(flat(z).argmax())                              # where ReLU is on it still shows
    flat(dy)[on] = float("inf")
    assert not bool(torch.autograd.grad(y, leaves, dy)[0].isfinite().all())


@pytest.mark.parametrize("affine", ["none", "frozen", "trained"])
@pytest.mark.parametrize("checkpoint8", [False, True])
@pytest.mark.parametrize("inner", [False, True])
def test_a_gradient_term_is_refused_and_not_lost(affine, checkpoint8, inner):
    """A penalty on the input's gradient, which would need the second derivative: whatever requires a gradient beside the
    input, and whether or not the input is a leaf."""
    leaf, dy, w, b = make((2, 16, 4, 4), torch.float32, seed=29)
    leaf.requires_grad_(True)
    x = leaf * 2 if inner else leaf
    if affine == "none":
        w = b = None
    elif affine == "trained":
        w.requires_grad_(True), b.requires_grad_(True)
    y = groupnorm_2d(x, 4, w, b, activation="silu", checkpoint8=checkpoint8)
    first = torch.autograd.grad(y, x, dy, retain_graph=True)[0]
    (dx,) = torch.autograd.grad(y, x, dy, create_graph=True)
    assert torch.equal(dx, first)                      # the first derivative is there
    with pytest.raises(RuntimeError, match="twice"):
        (y.sum() + dx.square().sum()).backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(dx.square().sum(), leaf, allow_unused=True)


@pytest.mark.parametrize("checkpoint8", [False, True])
@pytest.mark.parametrize("create_graph", [False, True])
def test_a_tangent_of_the_output_gradient_is_refused_and_not_lost(checkpoint8, create_graph):
    """Forward over reverse: the gradients would come back without their tangents."""
    x, dy, w, b = make((2, 16, 4, 4), torch.float32, seed=32)
    y = groupnorm_2d(x.requires_grad_(True), 4, w, b, checkpoint8=checkpoint8)
    weight = torch.randn(16, 8, 3, 3, device="cuda").half().requires_grad_(True)
    c = conv2d_gw8_checkpoint8(x.detach().half(), weight, None, padding_y=1, padding_x=1, groups=2)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(dy, torch.ones_like(dy))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, x, dual, create_graph=create_graph)
        if checkpoint8:
            dual = torch.autograd.forward_ad.make_dual(dy.half(), torch.ones_like(dy).half())
            with pytest.raises(RuntimeError, match="twice" if create_graph else "forward-mode"):
                torch.autograd.grad(c, weight, dual, create_graph=create_graph)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("checkpoint8", [False, True])
def test_model_held_in_16_bits(dtype, checkpoint8):
    """A model cast to fp16 or bf16, outside autocast: parameters of the data's type are taken in fp32, their gradients
    come back in their own type (one rounding)."""
    shape, groups = (3, 64, 9, 7), 8
    x, dy, w, b = make(shape, dtype, seed=30)
    model = nn.Sequential(nn.GroupNorm(groups, 64), nn.SiLU()).cuda()
    with torch.no_grad():
        model[0].weight.copy_(w), model[0].bias.copy_(b)
    model.to(dtype)
    weight, bias = model[0].weight, model[0].bias
    ref = Reference(x, groups, weight, bias, 1e-5, "silu", dy, checkpoint8)
    for fast in (transform(model, group_norm=True, checkpoint8=checkpoint8),
                 GroupNorm2d.from_torch_module(model[0], "silu", checkpoint8)):
        xs = x.clone().requires_grad_(True)
        y = fast(xs)
        assert y.dtype == dtype
        assert_within(y, ref.y, ref.y_tol, "y")
        dx, dw, db = torch.autograd.grad(y, (xs, weight, bias), dy)
        assert_within(dx, ref.dx, ref.dx_tol, "dx")
        assert dw.dtype == db.dtype == dtype
        assert_within(dw, ref.dweight, ref.dweight_tol + half_step(ref.dweight.abs() + ref.dweight_tol, dtype), "dweight")
        assert_within(db, ref.dbias, ref.dbias_tol + half_step(ref.dbias.abs() + ref.dbias_tol, dtype), "dbias")
        with torch.inference_mode():
            assert torch.equal(fast(x), y)
        with torch.no_grad():
            assert torch.equal(fast(x), y)
    layer = GroupNorm2d(groups, 64, dtype=dtype, device="cuda")
    assert torch.equal(layer(x), groupnorm_2d(x, groups))
    assert torch.equal(groupnorm_2d(x, groups, weight, None), groupnorm_2d(x, groups, weight.float(), None))
    # neither types that differ from each other nor a 16-bit vector beside data of another type
    other = torch.bfloat16 if dtype is torch.float16 else torch.float16
    for call in (lambda: groupnorm_2d(x, groups, weight, bias.float()), lambda: groupnorm_2d(x, groups, weight.float(), bias),
                 lambda: groupnorm_2d(x.float(), groups, weight, bias), lambda: groupnorm_2d(x.to(other), groups, weight, bias),
                 lambda: groupnorm_2d(x, groups, weight.double(), bias.double())):
        with pytest.raises(ValueError, match="weight and bias"):
            call()
