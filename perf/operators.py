"""Group norm with an activation on channels_last tensors and activation checkpoints in 8 bits: the
cases they are measured on, their plain forms and their values in 64 bits.

  infer   y = act(groupnorm(x))                                  what a serving process calls
  train   the same forward and its backward pass: y, dx, dweight, dbias
  train8  the same, with the input of the norm kept for the backward pass as 8-bit codes
  pack    a tensor to 8-bit codes with one power-of-two scale per 8 channels of a pixel, and back
  conv8   the group-width-8 convolution, its input kept in that form: y, dx, dweight (and dbias)

The scale of a block of 8 values is the smallest 2^k (k >= -126) for which the largest magnitude of the
block rounds to at most 127; codes are rounded half to even, and cut where the value that they stand for
would leave the range of the type.  The backward pass of `train8` uses the values that the codes stand
for in place of the input, and the statistics of the input itself.
"""

import math

import torch

own = False

ACTIVATIONS = ("none", "silu", "gelu")
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one small latent image of a serving process: latency only
        dict(name="infer_1x256x16x16_fp16", op="infer", n=1, c=256, h=16, w=16, groups=32, type="fp16", act="silu"),
        # odd sizes, three channels a group, 32-bit data
        dict(name="infer_5x96x37x53_fp32", op="infer", n=5, c=96, h=37, w=53, groups=32, type="fp32", act="gelu"),
        # the last resolution of an image decoder, one image: few groups, each of them large
        dict(name="infer_1x128x512x512_bf16", op="infer", n=1, c=128, h=512, w=512, groups=32, type="bf16", act="silu"),
        # the 64-channel 56 x 56 layer of the repository's benchmark, a training batch
        dict(name="train_256x64x56x56_fp16", op="train", n=256, c=64, h=56, w=56, groups=8, type="fp16", act="silu"),
        # two large images: fewer images than multiprocessors
        dict(name="train_2x256x128x128_bf16", op="train", n=2, c=256, h=128, w=128, groups=32, type="bf16", act="silu"),
        # the widest and smallest stage of the example network: 7 x 7 pixels, 24 channels a group
        dict(name="train_64x768x7x7_fp16", op="train", n=64, c=768, h=7, w=7, groups=32, type="fp16", act="gelu"),
        # its 192-channel stage with the 8-bit checkpoint: 6 channels a group
        dict(name="train8_128x192x28x28_fp16", op="train8", n=128, c=192, h=28, w=28, groups=32, type="fp16", act="silu"),
        # a few odd images, no activation
        dict(name="train8_3x40x65x33_bf16", op="train8", n=3, c=40, h=65, w=33, groups=5, type="bf16", act="none"),
        # a whole layer's input packed and restored
        dict(name="pack_256x64x56x56_fp16", op="pack", n=256, c=64, h=56, w=56, type="fp16"),
        dict(name="pack_2x24x17x5_bf16", op="pack", n=2, c=24, h=17, w=5, type="bf16"),
        # the benchmark's convolution with the checkpoint, and an odd one with a larger filter
        dict(name="conv8_128x64x56x56_3x3", op="conv8", n=128, c=64, h=56, w=56, r=3, s=3, bias=True, type="fp16"),
        dict(name="conv8_7x96x29x31_5x5", op="conv8", n=7, c=96, h=29, w=31, r=5, s=5, bias=False, type="fp16"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("infer", "train", "train8", "pack", "conv8"))
    c = 8 * _spread(rng, 1, 128)
    h = _spread(rng, 3, 300)
    w = max(3, min(400, int(h * rng.uniform(0.5, 2))))
    values = _spread(rng, 1 << 14, 3 << 23)
    n = max(1, min(512, values // (c * h * w)))
    while n * c * h * w > 3 << 23:
        c = 8 * max(1, c // 16)
        h = max(3, h - h // 8)
    case = dict(op=op, n=n, c=c, h=h, w=w)
    if op == "conv8":
        return dict(case, r=rng.choice((1, 3, 3, 5)), s=rng.choice((1, 3, 3, 5)), bias=rng.random() < 0.5, type="fp16")
    if op == "pack":
        return dict(case, type=rng.choice(tuple(TYPES)))
    # groups of 16 values at least: with two or three the normalised values hardly depend on the input,
    # and the gradient is what rounding leaves
    groups = rng.choice([g for g in range(1, c + 1) if c % g == 0 and (c // g) * h * w >= 16 and g <= 64])
    # (no gradients of ReLU: its derivative jumps where the output is zero, so one value in some
    # millions depends on the last bit of the statistics)
    act = rng.choice(ACTIVATIONS + ("relu",) if op == "infer" else ACTIVATIONS)
    return dict(case, groups=groups, type=rng.choice(tuple(TYPES)), act=act)


def _values(shape, gen, dtype):
    """Activations: each channel with a scale and an offset of its own, as behind a convolution."""
    n, c, h, w = shape
    x = torch.randn((n, h, w, c), generator=gen, device="cuda")
    scale = torch.exp(0.5 * torch.randn(c, generator=gen, device="cuda"))
    shift = 0.7 * torch.randn(c, generator=gen, device="cuda")
    return (x.mul_(scale).add_(shift)).to(dtype).permute(0, 3, 1, 2)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["type"]]
    n, c, h, w = case["n"], case["c"], case["h"], case["w"]
    state = {"op": case["op"], "x": _values((n, c, h, w), gen, dtype)}
    if case["op"] == "pack":
        return state
    if case["op"] == "conv8":
        r, s = case["r"], case["s"]
        state["weight"] = (torch.randn((c, r, s, 8), generator=gen, device="cuda") / math.sqrt(8 * r * s)).to(dtype).permute(0, 3, 1, 2)
        state["bias"] = 0.1 * torch.randn(c, generator=gen, device="cuda") if case["bias"] else None
        state["pad"] = (r // 2, s // 2)
    else:
        state["weight"] = 1 + 0.2 * torch.randn(c, generator=gen, device="cuda")
        state["bias"] = 0.2 * torch.randn(c, generator=gen, device="cuda")
        state["groups"], state["act"], state["eps"] = case["groups"], case["act"], 1e-5
    if case["op"] != "infer":
        state["dy"] = _grad((n, c, h, w), gen, dtype)  # the same size as x: the filters are odd and padded
        state["leaves"] = [state[k].requires_grad_(True) for k in ("x", "weight", "bias") if state[k] is not None]
    return state


def _grad(shape, gen, dtype):
    n, c, h, w = shape
    return torch.randn((n, h, w, c), generator=gen, device="cuda").to(dtype).permute(0, 3, 1, 2)


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        op = state["op"]
        if op == "pack":
            return {"restored": _restored(state["x"])}
        if op == "conv8":
            return _plain_conv(state)
        return _plain_norm(state)


def _run_own(state):
    from spio_b200 import functional as F

    op, x = state["op"], state["x"]
    if op == "pack":
        codes, exponents = F.checkpoint8_pack(x)
        return {"restored": F.checkpoint8_unpack(codes, exponents, x.dtype)}
    if op == "conv8":
        y = F.conv2d_gw8_checkpoint8(x, state["weight"], state["bias"], padding_y=state["pad"][0],
                                     padding_x=state["pad"][1], groups=x.shape[1] // 8)
    else:
        y = F.groupnorm_2d(x, state["groups"], state["weight"], state["bias"], state["eps"],
                           activation=state["act"], checkpoint8=op == "train8")
    if op == "infer":
        return {"y": y}
    grads = torch.autograd.grad(y, state["leaves"], state["dy"])
    return dict(zip(("dx", "dweight", "dbias"), grads), y=y.detach())


# ---- plain forms, in 32 bits


def _restored(x):
    """The values of `x` after a trip through 8-bit codes, in its own type."""
    top = torch.finfo(x.dtype).max
    n, c, h, w = x.shape
    v = x.permute(0, 2, 3, 1).reshape(n, h, w, c // 8, 8).float()
    largest = v.abs().amax(-1, keepdim=True)
    exponent = torch.frexp(largest)[1] - 7  # largest = m * 2^(exponent + 6), 1 <= m < 2
    over = torch.ldexp(largest, -exponent) >= 127.5
    exponent = torch.clamp(exponent + over, min=-126)
    scale = torch.ldexp(torch.ones_like(largest), exponent)
    limit = torch.floor(top / scale)
    codes = torch.minimum(torch.maximum(torch.round(v / scale), -limit), limit)
    return (codes * scale).reshape(n, h, w, c).to(x.dtype).permute(0, 3, 1, 2)


def _activation(z, act):
    """The activation and its derivative."""
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        p = 0.5 * torch.erfc(z * -math.sqrt(0.5))
        return z * p, p + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "relu":
        return torch.clamp(z, min=0), (z > 0).to(z.dtype)
    return z, torch.ones_like(z)


def _plain_norm(state):
    x, groups = state["x"], state["groups"]
    n, c, h, w = x.shape
    grouped = lambda t: t.permute(0, 2, 3, 1).reshape(n, h * w, groups, c // groups).float()  # noqa: E731
    image = lambda t: t.reshape(n, h, w, c).to(x.dtype).permute(0, 3, 1, 2)  # noqa: E731
    v = grouped(x)
    weight, bias = (state[k].reshape(groups, c // groups) for k in ("weight", "bias"))
    mean = v.mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(((v - mean) ** 2).mean((1, 3), keepdim=True) + state["eps"])
    y = image(_activation((v - mean) * rstd * weight + bias, state["act"])[0])
    if state["op"] == "infer":
        return {"y": y}
    if state["op"] == "train8":
        v = grouped(_restored(x))
    hat = (v - mean) * rstd
    grad = grouped(state["dy"]) * _activation(hat * weight + bias, state["act"])[1]
    dbias, dweight = grad.sum((0, 1)), (grad * hat).sum((0, 1))
    grad = grad * weight
    dx = rstd * (grad - grad.mean((1, 3), keepdim=True) - hat * (grad * hat).mean((1, 3), keepdim=True))
    return {"y": y, "dx": image(dx), "dweight": dweight.reshape(c), "dbias": dbias.reshape(c)}


def _taps(t, r, s, pad):
    """`t` (n, h, w, g, 8) padded, as r * s shifted views of size (n, p, q, g, 8)."""
    p, q = t.shape[1] + 2 * pad[0] - r + 1, t.shape[2] + 2 * pad[1] - s + 1
    t = torch.nn.functional.pad(t, (0, 0, 0, 0, pad[1], pad[1], pad[0], pad[0]))
    return [t[:, i : i + p, j : j + q] for i in range(r) for j in range(s)]


def _plain_conv(state):
    x, weight, bias, pad, dy = (state[k] for k in ("x", "weight", "bias", "pad", "dy"))
    n, c, h, w = x.shape
    r, s = weight.shape[2:]
    split = lambda t: t.permute(0, 2, 3, 1).reshape(t.shape[0], t.shape[2], t.shape[3], c // 8, 8).float()  # noqa: E731
    image = lambda t: t.reshape(*t.shape[:3], c).to(x.dtype).permute(0, 3, 1, 2)  # noqa: E731
    taps = weight.float().reshape(c // 8, 8, 8, r * s).permute(3, 0, 1, 2)  # (tap, group, out, in)
    grad = split(dy)
    y = sum(torch.einsum("npqgi,goi->npqgo", v, k) for v, k in zip(_taps(split(x), r, s, pad), taps))
    if bias is not None:
        y = y + bias.reshape(c // 8, 8)
    back = (r - 1 - pad[0], s - 1 - pad[1])
    dx = sum(torch.einsum("nhwgo,goi->nhwgi", v, k) for v, k in zip(_taps(grad, r, s, back), taps.flip(0)))
    dw = [torch.einsum("npqgi,npqgo->goi", v, grad) for v in _taps(split(_restored(x)), r, s, pad)]
    dw = torch.stack(dw, -1).reshape(c, 8, r, s).to(weight.dtype)
    out = {"y": image(y), "dx": image(dx), "dweight": dw}
    if bias is not None:
        out["dbias"] = grad.sum((0, 1, 2)).reshape(c)
    return out


# ---- what one pass cannot do without


def work(case):
    size = 4 if case["type"] == "fp32" else 2
    c, values = case["c"], case["n"] * case["c"] * case["h"] * case["w"]
    op = case["op"]
    if op == "pack":  # x in, codes and exponents out and in again, the restored tensor out
        return {"bytes": values * (2 * size + 2 * 9 / 8), "flops": 4 * values}
    if op == "conv8":
        macs = values * 8 * case["r"] * case["s"]
        return {"bytes": 4 * values * size + 4 * c * 8 * case["r"] * case["s"], "flops": 3 * 2 * macs}
    if op == "infer":
        return {"bytes": 2 * values * size + 8 * c, "flops": 12 * values}
    # x and dy in, y and dx out
    return {"bytes": 4 * values * size + 16 * c, "flops": 40 * values}


# ---- the operators' definition in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "pack":
            return {"restored": _exact_restored(state["x"])}
        if case["op"] == "conv8":
            return _exact_conv(state)
    return _exact_norm(state)


def _exact_restored(x):
    v = x.detach().double()
    n, c = v.shape[:2]
    blocks = v.unflatten(1, (c // 8, 8))
    largest = blocks.abs().max(2, keepdim=True).values
    k = torch.ceil(torch.log2(torch.where(largest > 0, largest, torch.ones_like(largest)) / 127.5))
    # the logarithm may be off next to a whole number: compare, which powers of two do without rounding
    k = torch.where(largest < 127.5 * torch.exp2(k - 1), k - 1, k)
    k = torch.where(largest >= 127.5 * torch.exp2(k), k + 1, k).clamp(min=-126)
    unit = torch.exp2(k)
    most = torch.floor(torch.finfo(x.dtype).max / unit)
    return (torch.clamp(torch.round(blocks / unit), -most, most) * unit).flatten(1, 2)


def _exact_norm(state):
    x, groups, act = state["x"].detach().double(), state["groups"], state["act"]
    n, c = x.shape[:2]
    wide = lambda t: t.repeat_interleave(c // groups, 1)[:, :, None, None]  # (n, groups) to (n, c, 1, 1)  # noqa: E731
    per_group = lambda t: t.reshape(n, groups, -1)  # noqa: E731
    row = lambda t: t.detach().double().reshape(1, c, 1, 1)  # noqa: E731
    var, mean = torch.var_mean(per_group(x), dim=2, correction=0)
    rstd = (var + state["eps"]).rsqrt()
    smooth = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.nn.functional.relu,
              "none": lambda t: t}[act]
    y = smooth((x - wide(mean)) * wide(rstd) * row(state["weight"]) + row(state["bias"]))
    if state["op"] == "infer":
        return {"y": y}
    if state["op"] == "train8":
        x = _exact_restored(state["x"])
    hat = (x - wide(mean)) * wide(rstd)
    z = (hat * row(state["weight"]) + row(state["bias"])).requires_grad_(True)
    (grad,) = torch.autograd.grad(smooth(z), z, state["dy"].double())
    dweight, dbias = (grad * hat).sum((0, 2, 3)), grad.sum((0, 2, 3))
    inner = grad * row(state["weight"])
    a, b = per_group(inner).mean(2), per_group(inner * hat).mean(2)
    return {"y": y, "dx": wide(rstd) * (inner - wide(a) - hat * wide(b)), "dweight": dweight, "dbias": dbias}


def _exact_conv(state):
    """Products of whole planes, one input channel of the group and one tap at a time."""
    x, weight, dy = (state[k].detach().double().contiguous() for k in ("x", "weight", "dy"))
    kept = _exact_restored(state["x"]).contiguous()
    c, r, s = x.shape[1], weight.shape[2], weight.shape[3]
    py, px = state["pad"]
    h, w = x.shape[2:]
    p, q = dy.shape[2:]
    first = torch.arange(c, device=x.device) // 8 * 8
    y, dx, dw = torch.zeros_like(dy), torch.zeros_like(x), torch.zeros_like(weight)
    if state["bias"] is not None:
        y += state["bias"].detach().double()[:, None, None]
    for i in range(r):
        for j in range(s):
            # output rows and columns whose input pixel (row + i - py, column + j - px) exists
            p0, p1 = max(0, py - i), min(p, h + py - i)
            q0, q1 = max(0, px - j), min(q, w + px - j)
            if p0 >= p1 or q0 >= q1:
                continue
            rows, cols = slice(p0 + i - py, p1 + i - py), slice(q0 + j - px, q1 + j - px)
            for k in range(8):
                y[:, :, p0:p1, q0:q1] += x[:, first + k, rows, cols] * weight[:, k, i, j][:, None, None]
                dw[:, k, i, j] = (kept[:, first + k, rows, cols] * dy[:, :, p0:p1, q0:q1]).sum((0, 2, 3))
                # input channel first + k receives from output channel o of its group with weight[o, its place]
                dx[:, :, rows, cols] += (dy[:, first + k, p0:p1, q0:q1]
                                         * weight[first + k, torch.arange(c, device=x.device) % 8, i, j][:, None, None])
    out = {"y": y, "dx": dx, "dweight": dw}
    if state["bias"] is not None:
        out["dbias"] = dy.sum((0, 2, 3))
    return out
