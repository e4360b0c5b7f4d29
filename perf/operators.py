"""What is measured of the normalisation and 4-bit layers: their cases, plain forms and exact results.

`run` makes one pass through an operator: with `own` the calls of the framework's layers, without it the same in
elementary torch operations.  Every tensor is channels last, {N, C, H, W} in the layers' size convention; a matrix is
the tensor {1, columns, 1, rows} and a matrix product the convolution with a 1x1 filter.

Operators (`case["op"]`):
  norm    group normalisation with an activation
  trip    quantisation of rows to 4-bit blocks, and the values those stand for
  conv    convolution of a 4-bit tensor with a 4-bit filter, bias and activation
  block   group normalisation with an activation, quantised in the same pass, and the convolution that reads it
"""
import math

import torch

own = False

NONE, RELU, SILU = 0, 1, 2
EPSILON = 1e-5


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # the innermost level of a U-shaped network on a small image: latency of one small normalisation
        dict(name="norm_small", op="norm", dtype="fp16", n=1, c=512, h=16, w=16, groups=32, act=SILU),
        # a batch of the sample's 91x91 images, fp32, groups of five channels: nothing is a power of two
        dict(name="norm_odd", op="norm", dtype="fp32", n=3, c=60, h=91, w=91, groups=12, act=RELU),
        # the 64 channels of the benchmark's 1080p frame
        dict(name="norm_frame", op="norm", dtype="fp16", n=1, c=64, h=1080, w=1920, groups=32, act=SILU),
        # the same tensor to 4 bits and back
        dict(name="trip_frame", op="trip", dtype="fp16", rows=1080 * 1920, columns=64),
        # rows of an unrolled 5x5 RGB filter window over a 91x91 image: every row ends inside a block
        dict(name="trip_odd", op="trip", dtype="fp32", rows=91 * 91, columns=75),
        # one row times a large matrix: bound by the filter's bytes, and by latency
        dict(name="conv_row", op="conv", dtype="fp16", n=1, c=4096, h=1, w=1, o=4096, kh=1, kw=1, bias=True, act=NONE),
        # a pointwise layer on a batch of 128x128 images: bound by the output's bytes
        dict(name="conv_point", op="conv", dtype="fp16", n=4, c=256, h=128, w=128, o=256, kh=1, kw=1, bias=True, act=RELU),
        # 64 -> 64 channels, 3x3, on the 1080p frame (the sample network's widest layer)
        dict(name="conv_frame", op="conv", dtype="fp16", n=1, c=64, h=1080, w=1920, o=64, kh=3, kw=3, bias=True, act=RELU),
        # a wide 3x3 layer: bound by the matrix units
        dict(name="conv_wide", op="conv", dtype="fp16", n=1, c=512, h=256, w=256, o=512, kh=3, kw=3, bias=False, act=NONE),
        # fp32 results, an even filter side and odd sizes everywhere
        dict(name="conv_odd", op="conv", dtype="fp32", n=2, c=75, h=91, w=91, o=33, kh=5, kw=2, bias=True, act=SILU),
        # a pre-activation block of a residual network on one 256x256 image
        dict(name="block_wide", op="block", dtype="fp16", n=1, c=256, h=256, w=256, groups=32, o=256, kh=3, kw=3, act=SILU),
        # the same on a batch of 91x91 images with channels that end inside a block
        dict(name="block_odd", op="block", dtype="fp16", n=2, c=80, h=91, w=91, groups=16, o=96, kh=3, kw=3, act=SILU),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _image(rng, pixels):
    """n, h, w with about `pixels` pixels in all."""
    n = min(_log(rng, 1, 8), max(1, pixels))
    w = max(1, min(pixels // n, int(math.sqrt(pixels / n) * math.exp(rng.uniform(-0.7, 0.7)))))
    return n, max(1, pixels // (n * w)), w


def draw(rng):
    op = rng.choice(["norm", "trip", "conv", "conv", "block"])
    if op == "trip":
        columns = _log(rng, 1, 4096)
        rows = _log(rng, 1, max(1, min(2 << 20, (1 << 27) // columns)))
        return dict(op=op, dtype=rng.choice(["fp16", "fp32"]), rows=rows, columns=columns)
    if op in ("norm", "block"):
        groups = rng.choice([1, 2, 4, 8, 16, 32])
        c = groups * rng.randint(1, max(1, 1024 // groups)) if rng.random() < 0.5 else groups * rng.choice([1, 2, 4, 8])
        c = min(c, 1024)
    if op == "norm":
        n, h, w = _image(rng, _log(rng, 16, max(16, min(2 << 20, (1 << 26) // c))))
        return dict(op=op, dtype=rng.choice(["fp16", "fp32"]), n=n, c=c, h=h, w=w, groups=groups, act=rng.randrange(3))
    kh, kw = rng.choice([(1, 1), (1, 1), (3, 3), (3, 3), (5, 5), (2, 3), (1, 7)])
    o = _log(rng, 3, 1024) if rng.random() < 0.5 else 32 * rng.randint(1, 16)
    if op == "conv":
        c = _log(rng, 3, 4096) if kh * kw == 1 else _log(rng, 3, 512)
        c = c if rng.random() < 0.5 else -(-c // 32) * 32
    # as many pixels as keep the unrolled windows below 4 GB and the products below the largest listed case's
    most = min(2 << 20, (1 << 30) // (c * kh * kw), int(1.2e11) // (c * kh * kw * o), (1 << 27) // o)
    n, h, w = _image(rng, _log(rng, 1, max(1, most)))
    case = dict(op=op, n=n, c=c, h=h, w=w, o=o, kh=kh, kw=kw)
    if op == "conv":
        return dict(case, dtype=rng.choice(["fp16", "fp32"]), bias=rng.random() < 0.7, act=rng.randrange(3))
    return dict(case, dtype="fp16", groups=groups, act=rng.randrange(3))


def work(case):
    size = 2 if case["dtype"] == "fp16" else 4
    if case["op"] == "trip":
        values = case["rows"] * case["columns"]
        held = case["rows"] * -(-case["columns"] // 32) * 17
        return {"bytes": 2 * values * size + 2 * held, "flops": 6 * values}
    m = case["n"] * case["h"] * case["w"]
    norm_flops = 10 * m * case["c"]
    if case["op"] == "norm":
        return {"bytes": 2 * m * case["c"] * size + 2 * case["c"] * size, "flops": norm_flops}
    taps, o = case["kh"] * case["kw"], case["o"]
    blocks = -(-case["c"] // 32)
    bytes_ = o * taps * blocks * 17 + m * o * size
    flops = 2 * m * taps * case["c"] * o
    if case["op"] == "conv":
        return {"bytes": bytes_ + m * blocks * 17, "flops": flops}
    # the normalised tensor in between is written and read once in 4 bits
    return {"bytes": bytes_ + m * case["c"] * size + 2 * m * blocks * 17, "flops": flops + norm_flops}


# ---------------------------------------------------------------------------
# The plain form
# ---------------------------------------------------------------------------
def _activate(y, act):
    if act == RELU:
        return torch.clamp(y, min=0)
    return y / (1 + torch.exp(-y)) if act == SILU else y


def _normalise(x, groups, scale, bias, act):
    n, h, w, c = x.shape
    v = x.float().reshape(n, h * w, groups, c // groups)
    d = v - v.mean(dim=(1, 3), keepdim=True)
    y = d * torch.rsqrt((d * d).mean(dim=(1, 3), keepdim=True) + EPSILON)
    return _activate(y.reshape(n, h, w, c) * scale.float() + bias.float(), act)


def _quantise(x):
    """[..., columns] in fp32 -> codes [..., blocks, 16] (element 2i in the low half of byte i) and scales [..., blocks]."""
    blocks = -(-x.shape[-1] // 32)
    v = torch.nn.functional.pad(x, (0, 32 * blocks - x.shape[-1])).reshape(*x.shape[:-1], blocks, 32)
    most = v.abs().amax(dim=-1)
    exponent = torch.clamp(torch.frexp(most)[1] - 3, min=-127)      # floor(log2(most)) - 2
    exponent = torch.where(most == 0, torch.full_like(exponent, -127), exponent)
    # 2^-exponent in two factors, each a normal number
    half = torch.div(exponent, 2, rounding_mode="floor")
    v = torch.ldexp(torch.ldexp(v, -half[..., None]), (half - exponent)[..., None])
    m = v.abs()
    # the magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6 are the codes 0 .. 7; ties go to the even code
    code = torch.where(m < 2, torch.round(2 * m), torch.where(m < 4, 2 + torch.round(m), 4 + torch.round(m / 2)))
    code = torch.clamp(code, max=7).to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)
    return code[..., 0::2] | (code[..., 1::2] << 4), (exponent + 127).to(torch.uint8)


def _values(codes, scales, columns):
    """What codes and scales stand for, in fp32."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    code = torch.stack([codes & 15, codes >> 4], dim=-1).reshape(*scales.shape, 32)
    v = table[code.int()] * torch.exp2(scales.float() - 127)[..., None]
    return v.reshape(*scales.shape[:-1], -1)[..., :columns]


def _convolve(x, f, bias, act):
    """x [n, h, w, c], f [o, kh, kw, c] in fp32."""
    n, h, w, c = x.shape
    o, kh, kw, _ = f.shape
    p = torch.nn.functional.pad(x, (0, 0, kw // 2, (kw - 1) // 2, kh // 2, (kh - 1) // 2))
    windows = p.unfold(1, kh, 1).unfold(2, kw, 1).reshape(n * h * w, c * kh * kw)
    y = windows @ f.permute(3, 1, 2, 0).reshape(c * kh * kw, o)
    return _activate(y if bias is None else y + bias.float(), act).reshape(n, h, w, o)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _type(case):
    return torch.float16 if case["dtype"] == "fp16" else torch.float32


def _activations(g, n, h, w, c):
    """A convolution's output: channels of different spread and offset."""
    x = torch.randn(n, h, w, c, generator=g, device="cuda")
    spread = torch.exp2(torch.randn(c, generator=g, device="cuda"))
    return x * spread + torch.randn(c, generator=g, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype, s = _type(case), dict(case)
    if case["op"] == "trip":
        rows, columns = case["rows"], case["columns"]
        s["x"] = _activations(g, 1, 1, rows, columns).reshape(rows, columns).to(dtype)
        blocks = -(-columns // 32)
        s["codes"] = torch.empty(rows, blocks, 16, dtype=torch.uint8, device="cuda")
        s["scales"] = torch.empty(rows, blocks, dtype=torch.uint8, device="cuda")
        s["out"] = torch.empty(rows, columns, dtype=dtype, device="cuda")
        return s
    n, c, h, w = (case[k] for k in "nchw")
    x = _activations(g, n, h, w, c)
    if case["op"] in ("norm", "block"):
        s["x"] = x.to(dtype)
        s["scale"] = (1 + 0.2 * torch.randn(c, generator=g, device="cuda")).to(dtype)
        s["shift"] = (0.2 * torch.randn(c, generator=g, device="cuda")).to(dtype)
    if case["op"] == "norm":
        s["out"] = torch.empty_like(s["x"])
    else:
        o, kh, kw = case["o"], case["kh"], case["kw"]
        f = torch.randn(o, kh, kw, c, generator=g, device="cuda") / math.sqrt(c * kh * kw)
        s["filter"] = _quantise(f)
        s["bias"] = None
        if case.get("bias", True):
            s["bias"] = (0.2 * torch.randn(o, generator=g, device="cuda")).to(dtype)
        s["out"] = torch.empty(n, h, w, o, dtype=dtype, device="cuda")
        blocks = -(-c // 32)
        if case["op"] == "conv":
            s["codes"], s["scales"] = _quantise(torch.clamp(x, min=-0.25))
        else:
            s["codes"] = torch.empty(n, h, w, blocks, 16, dtype=torch.uint8, device="cuda")
            s["scales"] = torch.empty(n, h, w, blocks, dtype=torch.uint8, device="cuda")
    if "groups" in case:
        # the layers say what they need for a size; no size here asks for more than this
        s["workspace"] = torch.empty(4 << 20, dtype=torch.uint8, device="cuda")
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def _code(case):
    return 0 if case["dtype"] == "fp16" else 1


def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "norm":
        return _normalise(s["x"], s["groups"], s["scale"], s["shift"], s["act"]).to(_type(s))
    if s["op"] == "trip":
        codes, scales = _quantise(s["x"].float())
        return _values(codes, scales, s["columns"]).to(_type(s))
    f = _values(*s["filter"], s["c"])
    if s["op"] == "conv":
        x = _values(s["codes"], s["scales"], s["c"])
        return _convolve(x, f, s["bias"], s["act"]).to(_type(s))
    codes, scales = _quantise(_normalise(s["x"], s["groups"], s["scale"], s["shift"], s["act"]))
    return _convolve(_values(codes, scales, s["c"]), f, s["bias"], NONE).to(_type(s))


def _run_own(s):
    import superresolution_amd as S
    t = _code(s)
    stream = torch.cuda.current_stream().cuda_stream or None
    if s["op"] == "trip":
        S.layer_quantize_mx4(t, s["x"].data_ptr(), s["rows"], s["columns"], s["codes"].data_ptr(), s["scales"].data_ptr(), stream)
        S.layer_dequantize_mx4(t, s["codes"].data_ptr(), s["scales"].data_ptr(), s["rows"], s["columns"], s["out"].data_ptr(), stream)
        return s["out"]
    sizes = (s["n"], s["c"], s["h"], s["w"])
    if s["op"] == "norm":
        S.layer_group_norm(t, s["x"].data_ptr(), sizes, s["groups"], s["scale"].data_ptr(), s["shift"].data_ptr(), EPSILON, s["act"],
                           s["out"].data_ptr(), s["workspace"].data_ptr(), s["workspace"].numel(), stream)
        return s["out"]
    if s["op"] == "block":
        S.layer_group_norm_mx4(t, s["x"].data_ptr(), sizes, s["groups"], s["scale"].data_ptr(), s["shift"].data_ptr(), EPSILON, s["act"],
                               s["codes"].data_ptr(), s["scales"].data_ptr(), s["workspace"].data_ptr(), s["workspace"].numel(), stream)
    S.layer_conv2d_mx4(t, s["codes"].data_ptr(), s["scales"].data_ptr(), sizes, s["filter"][0].data_ptr(), s["filter"][1].data_ptr(),
                       (s["o"], s["c"], s["kh"], s["kw"]), s["bias"].data_ptr() if s["bias"] is not None else None,
                       s["act"] if s["op"] == "conv" else NONE, s["out"].data_ptr(), stream)
    return s["out"]


# ---------------------------------------------------------------------------
# The results in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _exact_act(y, act):
    return torch.relu(y) if act == RELU else y * torch.sigmoid(y) if act == SILU else y


def _exact_rounded(x):
    """Every block of 32 columns of x (float64) rounded to what its 4-bit form stands for: nearest of the eight magnitudes
    times the block's power of two, the even one of two equally near."""
    columns = x.shape[-1]
    out = torch.empty_like(x)
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    # between magnitudes i and i + 1: the middle goes down where i is even, up where it is odd
    middle = (grid[1:] + grid[:-1]) / 2
    for b in range(0, columns, 32):
        part = x[..., b:b + 32]
        top = part.abs().amax(dim=-1, keepdim=True)
        unit = torch.exp2(torch.clamp(torch.floor(torch.log2(top)) - 2, min=-127))
        # log2 rounds: put the power of two right where that passed it
        unit = torch.where(unit * 8 <= top, unit * 2, unit)
        unit = torch.where((unit * 4 > top) & (unit > 2.0 ** -127), unit / 2, unit)
        m = part.abs() / unit
        index = torch.zeros_like(m, dtype=torch.int64)
        for i, t in enumerate(middle.tolist()):
            index += (m > t) if i % 2 == 0 else (m >= t)
        out[..., b:b + 32] = torch.copysign(grid[index] * unit, part)
    return out


def _exact_norm(x, groups, scale, bias, act):
    n, h, w, c = x.shape
    y = torch.empty(n, h, w, c, dtype=torch.float64, device=x.device)
    k = c // groups
    for i in range(n):
        for j in range(groups):
            v = x[i, :, :, j * k:(j + 1) * k].double()
            var, mean = torch.var_mean(v, correction=0)
            y[i, :, :, j * k:(j + 1) * k] = (v - mean) / torch.sqrt(var + EPSILON)
    y.mul_(scale.double()).add_(bias.double())
    return _exact_act(y, act)


def _exact_held(codes, scales, columns):
    low, high = (codes & 15).long(), (codes >> 4).long()
    code = torch.empty(*codes.shape[:-1], 32, dtype=torch.int64, device=codes.device)
    code[..., 0::2], code[..., 1::2] = low, high
    e, f = (code >> 1) & 3, code & 1
    m = torch.where(e == 0, 0.5 * f.double(), (1 + 0.5 * f.double()) * torch.exp2(e.double() - 1))
    v = torch.where(code >= 8, -m, m) * torch.exp2(scales.double() - 127)[..., None]
    return v.reshape(*codes.shape[:-2], -1)[..., :columns]


def _exact_conv(x, f, bias, act):
    n, h, w, c = x.shape
    o, kh, kw, _ = f.shape
    y = torch.zeros(n, h, w, o, dtype=torch.float64, device=x.device)
    for i in range(kh):
        for j in range(kw):
            dy, dx = i - kh // 2, j - kw // 2
            top, bottom, left, right = max(0, -dy), min(h, h - dy), max(0, -dx), min(w, w - dx)
            if top >= bottom or left >= right:
                continue
            part = x[:, top + dy:bottom + dy, left + dx:right + dx, :].reshape(-1, c)
            y[:, top:bottom, left:right, :] += (part @ f[:, i, j, :].t().contiguous()).reshape(n, bottom - top, right - left, o)
    if bias is not None:
        y += bias.double()
    return _exact_act(y, act)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s["x"], case["groups"], s["scale"], s["shift"], case["act"])
    if case["op"] == "trip":
        return _exact_rounded(s["x"].double())
    f = _exact_held(*s["filter"], case["c"])
    if case["op"] == "conv":
        return _exact_conv(_exact_held(s["codes"], s["scales"], case["c"]), f, s["bias"], case["act"])
    x = _exact_rounded(_exact_norm(s["x"], case["groups"], s["scale"], s["shift"], case["act"]))
    return _exact_conv(x, f, s["bias"], NONE)
