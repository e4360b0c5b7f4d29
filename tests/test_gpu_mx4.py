"""The normalisation and 4-bit layers against their definitions in 64 bits.

Tolerances.  A result stored in fp16 / fp32 is off by half a step at most (2^-11 / 2^-24 of its value; 2^-25 absolutely
among the subnormals of fp16).  fp32 arithmetic before that is bounded where it is used.
"""
import numpy as np
import pytest
import torch

import superresolution_amd as S

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {0: torch.float16, 1: torch.float32}
GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def stream():
    return torch.cuda.current_stream().cuda_stream or None


def step(dtype, ref):
    """Half a step of the stored type."""
    return ref.abs() * (2.0 ** -11 if dtype == 0 else U) + (2.0 ** -25 if dtype == 0 else 2.0 ** -150)


class Guarded:
    """A device tensor between two rows of bytes that no kernel may touch."""

    def __init__(self, shape, dtype, fill=None):
        n = int(np.prod(shape)) * torch.empty(0, dtype=dtype).element_size()
        self.raw = torch.full((n + 512,), 0xA5, dtype=torch.uint8, device="cuda")
        self.t = self.raw[256:256 + n].view(dtype).reshape(shape)
        self.n = n
        if fill is not None:
            self.t.copy_(fill)

    def ptr(self):
        return self.t.data_ptr()

    def whole(self):
        torch.cuda.synchronize()
        assert (self.raw[:256] == 0xA5).all() and (self.raw[256 + self.n:] == 0xA5).all(), "written outside the tensor"
        return self.t.cpu()


# ---------------------------------------------------------------------------
# The definitions
# ---------------------------------------------------------------------------
def act64(y, act):
    return torch.where(y < 0, torch.zeros_like(y), y) if act == 1 else y * torch.sigmoid(y) if act == 2 else y


def norm64(x, groups, scale, bias, eps, act):
    """x [n, h, w, c]; also the mean over the deviation, the normalised value and the result before the activation."""
    n, h, w, c = x.shape
    v = x.double().reshape(n, h * w, groups, c // groups)
    mean = v.mean(dim=(1, 3), keepdim=True)
    var = ((v - mean) ** 2).mean(dim=(1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xh = ((v - mean) * rstd).reshape(n, h, w, c)
    shift = (mean.abs() * rstd).expand_as(v).reshape(n, h, w, c)
    s = torch.ones(c, dtype=torch.float64) if scale is None else scale.double()
    b = torch.zeros(c, dtype=torch.float64) if bias is None else bias.double()
    y = xh * s + b
    return act64(y, act), shift, xh, s, b, y


def norm_tolerance(shift, xh, s, b, y):
    """fp32 before the last rounding.  Sums run over at most 64 terms in a row at every level of the joins, with errors
    of at most 64 half steps of terms of the size of the spread; a joined mean has a few half steps of its own value, which
    the division by the deviation makes `shift`.  The variance's relative error is twice the mean's and its own sum's.
    The last line is (x - mean) * mul + add, and SiLU passes an error on 1.1 times and adds (|y| + 8) half steps."""
    return U * (1.1 * (80 * (shift + xh.abs() + 1) * s.abs() + 4 * b.abs()) + y.abs() * (y.abs() + 8))


def quantise64(x):
    """x [rows, columns] -> codes [rows, blocks, 16], scales [rows, blocks] (uint8), from the definition in 64 bits."""
    x = x.double()
    rows, columns = x.shape
    blocks = -(-columns // 32)
    v = torch.zeros(rows, blocks * 32, dtype=torch.float64)
    v[:, :columns] = x
    v = v.reshape(rows, blocks, 32)
    most = v.abs().amax(-1)
    bad = ~torch.isfinite(v).all(-1)
    e = torch.frexp(torch.where(bad, torch.ones_like(most), most))[1] - 1 - 2
    e = torch.where(most == 0, torch.full_like(e, -127), e.clamp(min=-127))
    code = nearest((v * torch.exp2(-e.double())[..., None]))
    code[bad] = 0
    scales = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)
    code = code.to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scales


def nearest(v):
    m = v.abs()
    i = torch.zeros(v.shape, dtype=torch.int64)
    for k in range(7):
        middle = float(GRID[k] + GRID[k + 1]) / 2
        i += (m > middle) if k % 2 == 0 else (m >= middle)
    return i + 8 * torch.signbit(v).long()


def values64(codes, scales, columns):
    code = torch.stack([codes & 15, codes >> 4], dim=-1).reshape(*scales.shape, 32).long()
    v = GRID.to(codes.device)[code & 7] * torch.where(code >= 8, -1.0, 1.0).double()
    f = torch.exp2(scales.double() - 127)
    f = torch.where(scales == 255, torch.full_like(f, float("nan")), f)
    return (v * f[..., None]).reshape(*scales.shape[:-1], -1)[..., :columns]


def conv64(x, w, bias, act):
    """x [n, h, w, c], w [o, kh, kw, c], on either side; also the sum of the magnitudes of the terms."""
    n, H, W, c = x.shape
    o, kh, kw, _ = w.shape
    p = torch.zeros(n, H + kh - 1, W + kw - 1, c, dtype=torch.float64, device=x.device)
    p[:, kh // 2:kh // 2 + H, kw // 2:kw // 2 + W] = x
    y = torch.zeros(n, H, W, o, dtype=torch.float64, device=x.device)
    size = torch.zeros_like(y)
    for i in range(kh):
        for j in range(kw):
            part = p[:, i:i + H, j:j + W].reshape(-1, c)
            f = w[:, i, j].T.contiguous()
            y += (part @ f).reshape(y.shape)
            size += (part.abs() @ f.abs()).reshape(y.shape)
    if bias is not None:
        y, size = y + bias.double().to(y.device), size + bias.double().abs().to(y.device)
    return act64(y, act), size, y


def conv_tolerance(size, y, blocks):
    """An instruction adds 64 products (exact in fp32) to the sum and may drop what is below a step (2^-23) of the largest
    term or partial sum at each of the six levels of its tree; there is one for every two blocks, and a few more additions
    join partial sums and the bias.  SiLU as above."""
    return 2 * U * size * 1.1 * (blocks / 2 + 12) + U * y.abs() * (y.abs() + 8)


def quantise(x, dtype):
    rows, columns = x.shape
    blocks = -(-columns // 32)
    src = Guarded(x.shape, TYPES[dtype], x)
    codes, scales = Guarded((rows, blocks, 16), torch.uint8), Guarded((rows, blocks), torch.uint8)
    S.layer_quantize_mx4(dtype, src.ptr(), rows, columns, codes.ptr(), scales.ptr(), stream())
    return codes, scales


def group_norm(x, dtype, groups, scale, bias, act, eps=1e-5, mx4=False, in_place=False):
    n, h, w, c = x.shape
    src = Guarded(x.shape, TYPES[dtype], x)
    sb = [None if v is None else Guarded(v.shape, TYPES[dtype], v) for v in (scale, bias)]
    ps = [None if v is None else v.ptr() for v in sb]
    need = S.layer_group_norm_workspace(dtype, (n, c, h, w), groups)
    work = Guarded((need,), torch.uint8)
    if mx4:
        blocks = -(-c // 32)
        codes, scales = Guarded((n * h * w, blocks, 16), torch.uint8), Guarded((n * h * w, blocks), torch.uint8)
        S.layer_group_norm_mx4(dtype, src.ptr(), (n, c, h, w), groups, *ps, eps, act, codes.ptr(), scales.ptr(), work.ptr(), need, stream())
        work.whole()
        return codes, scales
    out = src if in_place else Guarded(x.shape, TYPES[dtype])
    S.layer_group_norm(dtype, src.ptr(), (n, c, h, w), groups, *ps, eps, act, out.ptr(), work.ptr(), need, stream())
    work.whole()
    return out.whole()


def convolve(xc, xs, sizes, wc, ws, fsizes, bias, act, dtype):
    n, c, h, w = sizes
    out = Guarded((n, h, w, fsizes[0]), TYPES[dtype])
    b = None if bias is None else Guarded(bias.shape, TYPES[dtype], bias)
    S.layer_conv2d_mx4(dtype, xc.ptr(), xs.ptr(), sizes, wc.ptr(), ws.ptr(), fsizes, None if b is None else b.ptr(), act, out.ptr(), stream())
    return out.whole()


def rnd(shape, seed, dtype=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp2(torch.randn(shape[-1], generator=g)) + torch.randn(shape[-1], generator=g)
    return x.to(TYPES[dtype])


# ---------------------------------------------------------------------------
# 4-bit blocks
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("rows,columns", [(1, 1), (1, 31), (1, 32), (5, 33), (3, 75), (129, 64), (7, 96), (2, 1000), (1000, 3), (70, 257)])
def test_quantise_is_the_definition(dtype, rows, columns):
    x = rnd((rows, columns), rows * 1000 + columns, dtype)
    codes, scales = quantise(x, dtype)
    want, want_s = quantise64(x)
    assert torch.equal(scales.whole(), want_s) and torch.equal(codes.whole(), want)


def test_quantise_every_fp16_value():
    """Every bit pattern as the largest of a block and among others: ties, saturation, subnormals, zeros, infinities, NaN."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    v = bits.view(torch.float16)
    alone = torch.zeros(65536, 32, dtype=torch.float16)
    alone[:, 5] = v
    mixed = v.reshape(2048, 32)                                  # 32 neighbours share an exponent
    steps = torch.arange(-64, 64, dtype=torch.float32).reshape(4, 32) / 8
    ties = torch.cat([steps.half() * 2.0 ** e for e in range(-22, 12)])
    ties[:, 0] = torch.cat([torch.full((4,), 7.0) * 2.0 ** e for e in range(-22, 12)]).half()
    for x in (alone, mixed, ties):
        codes, scales = quantise(x, 0)
        want, want_s = quantise64(x)
        assert torch.equal(scales.whole(), want_s) and torch.equal(codes.whole(), want)


def test_quantise_every_fp32_exponent():
    """Blocks over the whole range of fp32, subnormals included; the smaller values of a block down to nothing."""
    g = torch.Generator().manual_seed(3)
    rows = []
    for e in range(-149, 128):
        m = torch.rand(32, generator=g, dtype=torch.float64) + 1
        rows.append(m * 2.0 ** e * torch.where(torch.rand(32, generator=g) < 0.5, -1.0, 1.0).double())
        rows.append(m * torch.exp2(e - torch.arange(32).double() / 4))
    x = torch.stack(rows)
    x = torch.where(x.abs() >= 2.0 ** 128 * (1 - 2.0 ** -25), torch.full_like(x, 3.0e38), x).float()
    special = torch.ones(8, 32)
    special[0, 3], special[1, 31], special[2, 0], special[3, :] = float("inf"), -float("inf"), float("nan"), 0
    special[4, :], special[5, 7], special[6, 9] = -0.0, 3.4028234663852886e38, 1e-45
    x = torch.cat([x, special])
    codes, scales = quantise(x, 1)
    want, want_s = quantise64(x)
    assert torch.equal(scales.whole(), want_s) and torch.equal(codes.whole(), want)


@pytest.mark.parametrize("dtype", [0, 1])
def test_dequantise_every_code_and_scale(dtype):
    scales = torch.arange(256, dtype=torch.uint8).reshape(256, 1)
    code = torch.arange(32, dtype=torch.uint8) % 16
    codes = (code[0::2] | (code[1::2] << 4)).expand(256, 1, 16).contiguous()
    for columns in (32, 27, 8, 1):
        c, s, out = Guarded(codes.shape, torch.uint8, codes), Guarded(scales.shape, torch.uint8, scales), Guarded((256, columns), TYPES[dtype])
        S.layer_dequantize_mx4(dtype, c.ptr(), s.ptr(), 256, columns, out.ptr(), stream())
        want = values64(codes, scales, columns).to(TYPES[dtype])
        got = out.whole()
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got[~want.isnan()], want[~want.isnan()])
        assert torch.equal(torch.signbit(got[:255]), torch.signbit(want[:255]))


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("rows,columns", [(1, 1), (3, 33), (129, 64), (70, 257), (1000, 3)])
def test_round_trip(dtype, rows, columns):
    x = rnd((rows, columns), 5, dtype)
    codes, scales = quantise(x, dtype)
    out = Guarded((rows, columns), TYPES[dtype])
    S.layer_dequantize_mx4(dtype, codes.ptr(), scales.ptr(), rows, columns, out.ptr(), stream())
    assert torch.equal(out.whole(), values64(*quantise64(x), columns).to(TYPES[dtype]))


def test_offsets_past_32_bits():
    """More than 2^32 values: the last rows are the same as alone, and so are rows on both sides of 2^32."""
    h, w, columns = 8200, 8192, 64                               # 2^26 and 65536 rows
    rows = h * w
    x = torch.zeros(rows, columns, dtype=torch.float16, device="cuda")
    tail = rnd((96, columns), 9)
    for at in (rows - 96, (1 << 25) - 48, (1 << 26) - 48):
        x[at:at + 96] = tail.cuda()
    codes = torch.empty(rows, 2, 16, dtype=torch.uint8, device="cuda")
    scales = torch.empty(rows, 2, dtype=torch.uint8, device="cuda")
    S.layer_quantize_mx4(0, x.data_ptr(), rows, columns, codes.data_ptr(), scales.data_ptr(), stream())
    want, want_s = quantise64(tail)
    f = Guarded((64, 64), torch.float16, rnd((64, 64), 10) / 8)
    wc, ws = quantise(f.t.cpu(), 0)
    S.layer_dequantize_mx4(0, codes.data_ptr(), scales.data_ptr(), rows, columns, x.data_ptr(), stream())
    y = torch.empty(rows, 64, dtype=torch.float16, device="cuda")
    S.layer_conv2d_mx4(0, codes.data_ptr(), scales.data_ptr(), (1, 64, 1, rows), wc.ptr(), ws.ptr(), (64, 64, 1, 1), None, 0, y.data_ptr(), stream())
    torch.cuda.synchronize()
    # as an image: other kernels, the same sums (of one step)
    z = torch.empty_like(y)
    S.layer_conv2d_mx4(0, codes.data_ptr(), scales.data_ptr(), (1, 64, h, w), wc.ptr(), ws.ptr(), (64, 64, 1, 1), None, 0, z.data_ptr(), stream())
    torch.cuda.synchronize()
    assert torch.equal(z, y)
    del z
    v = values64(want, want_s, columns)
    ref, size, raw = conv64(v.reshape(1, 1, 96, 64), values64(wc.whole(), ws.whole(), 64).reshape(64, 1, 1, 64), None, 0)
    for at in (rows - 96, (1 << 25) - 48, (1 << 26) - 48):
        assert torch.equal(codes[at:at + 96].cpu(), want) and torch.equal(scales[at:at + 96].cpu(), want_s)
        assert torch.equal(x[at:at + 96].cpu(), v.half())
        assert ((y[at:at + 96].cpu().double() - ref[0, 0]).abs() <= conv_tolerance(size, raw, 2)[0, 0] + step(0, ref)[0, 0]).all()
    assert float(y[:(1 << 25) - 48].abs().max()) == 0
    del codes, scales, y
    # a normalisation of the same tensor in place: statistics by torch in 64 bits, a part of the image at a time
    need = S.layer_group_norm_workspace(0, (1, columns, 1, rows), 4)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    total = torch.zeros(columns, dtype=torch.float64, device="cuda")
    square = torch.zeros_like(total)
    for part in x.split(1 << 22):
        total += part.double().sum(0)
        square += part.double().square().sum(0)
    total, square = total.cpu().reshape(4, 16).sum(1) / (rows * 16.0), square.cpu().reshape(4, 16).sum(1) / (rows * 16.0)
    S.layer_group_norm(0, x.data_ptr(), (1, columns, 1, rows), 4, None, None, 1e-5, 0, x.data_ptr(), work.data_ptr(), need, stream())
    torch.cuda.synchronize()
    rstd = 1 / torch.sqrt(square - total ** 2 + 1e-5)
    want = (v.half().double().reshape(96, 4, 16) - total[:, None]) * rstd[:, None]
    want = want.reshape(96, 64)
    for at in (rows - 96, (1 << 25) - 48):
        assert ((x[at:at + 96].cpu().double() - want).abs() <= step(0, want) + U * 200 * (want.abs() + 1)).all()


def test_more_threads_than_one_grid_dimension_holds():
    """2^32 rows of one value, 2^31 - 1 pixels, 2^24 images of one pixel: workgroups whose threads number 2^32 and more."""
    rows, pixels = (1 << 32) + 3, (1 << 31) - 1
    tail = rnd((40, 1), 11)
    x = torch.zeros(rows, 1, dtype=torch.float16, device="cuda")
    at = (rows - 40, (1 << 31) - 41, 12345)
    for a in at:
        x[a:a + 40] = tail.cuda()
    codes = torch.empty(rows, 16, dtype=torch.uint8, device="cuda")
    scales = torch.empty(rows, dtype=torch.uint8, device="cuda")
    S.layer_quantize_mx4(0, x.data_ptr(), rows, 1, codes.data_ptr(), scales.data_ptr(), stream())
    x.fill_(9)
    S.layer_dequantize_mx4(0, codes.data_ptr(), scales.data_ptr(), rows, 1, x.data_ptr(), stream())
    f = rnd((4, 1), 12)
    wc, ws = quantise(f, 0)
    y = torch.empty(pixels, 4, dtype=torch.float16, device="cuda")
    S.layer_conv2d_mx4(0, codes.data_ptr(), scales.data_ptr(), (1, 1, 1, pixels), wc.ptr(), ws.ptr(), (4, 1, 1, 1), None, 0, y.data_ptr(), stream())
    torch.cuda.synchronize()
    want, want_s = quantise64(tail)
    v = values64(want, want_s, 1)
    product = (v * values64(wc.whole(), ws.whole(), 1).reshape(1, 4)).half()   # 4 bits of fraction at most: exact in fp16
    for a in at:
        assert torch.equal(codes[a:a + 40].cpu(), want[:, 0]) and torch.equal(scales[a:a + 40].cpu(), want_s[:, 0])
        assert torch.equal(x[a:a + 40].cpu(), v.half())
        if a + 40 <= pixels:
            assert torch.equal(y[a:a + 40].cpu(), product)
    assert float(x[rows - 41]) == 0 and float(y[1 << 30:(1 << 30) + 4096].abs().max()) == 0
    del x, y, codes, scales
    images = (1 << 24) + 3
    x = torch.randn(images, 1, 1, 8, dtype=torch.float16, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    out = torch.empty_like(x)
    need = S.layer_group_norm_workspace(0, (images, 8, 1, 1), 2)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    S.layer_group_norm(0, x.data_ptr(), (images, 8, 1, 1), 2, None, None, 1e-5, 0, out.data_ptr(), work.data_ptr(), need, stream())
    torch.cuda.synchronize()
    for a in (0, (1 << 21) - 20, (1 << 23) - 20, images - 40):
        ref, *parts = norm64(x[a:a + 40].cpu(), 2, None, None, 1e-5, 0)
        assert ((out[a:a + 40].cpu().double() - ref).abs() <= step(0, ref) + norm_tolerance(*parts)).all()


def test_group_norm_first_value_far_from_the_others():
    """Large parts of few channels, whose sums are taken about the first value: its distance must not drown the spread."""
    n, h, w, c, d = 1, 8192, 8192, 4, 300.0
    x = torch.randn(n, h, w, c, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    x.view(-1, c)[::65536] += d
    v = x.double().view(-1, 2, 2)
    mean = v.mean(dim=(0, 2))
    v = v - mean[:, None]
    rstd = 1 / torch.sqrt((v ** 2).mean(dim=(0, 2)) + 1e-5)
    want = (v * rstd[:, None]).view(n, h, w, c)
    out = torch.empty_like(x)
    need = S.layer_group_norm_workspace(1, (n, c, h, w), 2)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    S.layer_group_norm(1, x.data_ptr(), (n, c, h, w), 2, None, None, 1e-5, 0, out.data_ptr(), work.data_ptr(), need, stream())
    torch.cuda.synchronize()
    # A thread adds up 256 values at most; the one of 256 threads whose first value is the far one adds up squares of d:
    # U * i * d^2 at term i, 256^2 / 2 in all, and twice that in the square of its sum.  Its part's variance times the part's pixels
    # is 65536 (1 + d^2 / 65536); the result has half the variance's relative error.  Its mean is off by 256 U d, the
    # part's by d U, the other sums by 80 half steps of the spread and the mean as in norm_tolerance.
    off = 1.5 * 256 ** 2 * U * d ** 2 / (65536 + d ** 2) / 2
    assert ((out.double() - want).abs() <= off * want.abs() + U * (80 * (want.abs() + 1) + d)).all()


# ---------------------------------------------------------------------------
# Group normalisation
# ---------------------------------------------------------------------------
NORMS = [(1, 1, 1, 1, 1), (2, 3, 1, 1, 3), (1, 32, 1, 7, 4), (3, 60, 9, 13, 12), (1, 64, 33, 31, 32), (2, 2056, 3, 3, 8),
         (1, 4100, 5, 3, 1), (2, 2304, 2, 2, 1152), (1, 4096, 2, 2, 4096), (1, 96, 70, 90, 3), (5, 7, 17, 3, 7), (1, 512, 16, 16, 32),
         (2, 40, 64, 48, 5), (1, 2050, 1, 40, 2), (70, 8, 2, 3, 2), (1, 256, 128, 64, 32), (1, 8, 400, 300, 2)]


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("n,c,h,w,groups", NORMS)
def test_group_norm(dtype, n, c, h, w, groups):
    for act, (with_scale, with_bias) in enumerate([(True, True), (False, True), (True, False)]):
        x = rnd((n, h, w, c), n + c + h + act, dtype)
        scale = (1 + 0.3 * rnd((c,), 1, 1)).to(TYPES[dtype]) if with_scale else None
        bias = rnd((c,), 2, dtype) if with_bias else None
        ref, *parts = norm64(x, groups, scale, bias, 1e-5, act)
        got = group_norm(x, dtype, groups, scale, bias, act, in_place=act == 1)
        assert ((got.double() - ref).abs() <= step(dtype, ref) + norm_tolerance(*parts)).all()


@pytest.mark.parametrize("n,c,h,w,groups", [(1, 32, 40, 30, 4), (2, 9, 64, 64, 3), (1, 2200, 4, 4, 1), (1, 64, 8, 8, 8)])
def test_group_norm_large_mean(n, c, h, w, groups):
    """A mean of a thousand deviations: a variance taken as avg(x^2) - mean^2 would be off by parts in ten."""
    x = torch.randn((n, h, w, c), generator=torch.Generator().manual_seed(4)) + 1000
    x[:, 0, 0, :] += 40                                          # the first values are not near the others
    ref, *parts = norm64(x, groups, None, None, 1e-5, 0)
    got = group_norm(x, 1, groups, None, None, 0)
    assert ((got.double() - ref).abs() <= step(1, ref) + norm_tolerance(*parts)).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("c,groups,h,w", [(12, 3, 8, 9), (64, 4, 60, 50)])
def test_group_norm_keeps_a_bad_value_in_its_group(bad, c, groups, h, w):
    x = rnd((2, h, w, c), 6)
    x[1, h // 2, 3, c // groups] = bad                           # image 1, group 1
    got = group_norm(x, 0, groups, None, None, 2)
    k = c // groups
    assert got[1, :, :, k:2 * k].isnan().all()
    got[1, :, :, k:2 * k] = 0
    assert got.isfinite().all()
    x[1, h // 2, 3, k] = 0
    ref, *parts = norm64(x, groups, None, None, 1e-5, 2)
    tol = step(0, ref) + norm_tolerance(*parts)
    err = (got.double() - ref).abs()
    err[1, :, :, k:2 * k] = 0
    assert (err <= tol).all()


def test_group_norm_of_a_constant_is_the_bias():
    x = torch.full((1, 9, 7, 24), 3.0)
    bias = rnd((24,), 3, 1)
    for act in range(3):
        got = group_norm(x, 1, 4, None, bias, act)
        want = act64(bias.double(), act).expand_as(got)
        assert ((got.double() - want).abs() <= U * 20 * (want.abs() + 1)).all()


def check_codes(codes, scales, ref, tol):
    """Codes and scales may be those of any value within tol of ref: the scale between the scales of the smallest and largest
    possible maximum, and each code between those of the two ends."""
    rows, columns = ref.shape
    codes, scales = codes.whole(), scales.whole()
    blocks = scales.shape[1]
    pad = lambda v: torch.nn.functional.pad(v, (0, blocks * 32 - columns)).reshape(rows, blocks, 32)  # noqa: E731
    v, t = pad(ref), pad(tol)
    low, high = (v.abs() - t).clamp(min=0).amax(-1), (v.abs() + t).amax(-1)
    scale_of = lambda m: torch.where(m == 0, torch.zeros_like(m, dtype=torch.int32), (torch.frexp(m)[1] - 3 + 127).clamp(min=0).int())  # noqa: E731
    assert (scales.int() >= scale_of(low)).all() and (scales.int() <= scale_of(high)).all()
    inv = torch.exp2(127 - scales.double())[..., None]
    signed = lambda c: GRID[c & 7] * torch.where(c >= 8, -1.0, 1.0).double()  # noqa: E731
    got = torch.stack([codes & 15, codes >> 4], dim=-1).reshape(rows, blocks, 32).long()
    assert (signed(got) >= signed(nearest((v - t) * inv))).all() and (signed(got) <= signed(nearest((v + t) * inv))).all()
    sharp = signed(nearest((v - t) * inv)) == signed(nearest((v + t) * inv))     # a zero of either sign is a zero
    assert sharp.double().mean() > 0.9                           # the check is a check


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("n,c,h,w,groups", NORMS)
def test_group_norm_mx4(dtype, n, c, h, w, groups):
    for act in range(3):
        x = rnd((n, h, w, c), n + c + h + act, dtype)
        scale, bias = (1 + 0.3 * rnd((c,), 1, 1)).to(TYPES[dtype]), rnd((c,), 2, dtype)
        ref, *parts = norm64(x, groups, scale, bias, 1e-5, act)
        codes, scales = group_norm(x, dtype, groups, scale, bias, act, mx4=True)
        check_codes(codes, scales, ref.reshape(-1, c), norm_tolerance(*parts).reshape(-1, c))


# ---------------------------------------------------------------------------
# Convolution
# ---------------------------------------------------------------------------
CONVS = [(1, 1, 1, 1, 1, 1, 1), (1, 32, 1, 1, 16, 1, 1), (1, 33, 1, 1, 5, 1, 1), (1, 4096, 1, 1, 300, 1, 1), (1, 512, 1, 2, 64, 1, 1),
         (1, 2049, 1, 17, 33, 1, 1), (1, 64, 9, 11, 64, 3, 3), (2, 75, 13, 9, 33, 5, 2), (1, 96, 20, 30, 130, 3, 3), (3, 16, 7, 7, 8, 7, 7),
         (1, 256, 24, 24, 256, 3, 3), (1, 128, 40, 33, 70, 1, 1), (1, 300, 16, 16, 200, 2, 3), (2, 64, 50, 70, 3, 3, 3), (1, 3, 21, 33, 32, 5, 5),
         (1, 8, 1, 40, 12, 1, 7), (1, 8, 40, 1, 12, 7, 1), (1, 8, 2, 2, 12, 7, 7), (1, 288, 30, 31, 512, 1, 1), (4, 160, 33, 17, 96, 3, 1),
         (1, 1024, 6, 6, 128, 3, 3), (1, 32, 130, 140, 40, 1, 1), (1, 512, 9, 15, 513, 1, 1), (1, 700, 1, 300, 260, 1, 1),
         (1, 64, 150, 170, 64, 3, 3), (1, 32, 140, 150, 70, 3, 3), (2, 96, 90, 110, 40, 3, 3), (1, 128, 130, 140, 32, 3, 3), (1, 20, 200, 160, 24, 5, 5),
         (1, 50, 150, 150, 64, 5, 5), (1, 8, 150, 170, 33, 1, 7), (1, 100, 160, 150, 20, 2, 2), (1, 30, 150, 170, 10, 7, 7), (1, 64, 16, 5000, 24, 3, 3),
         (1, 40, 3000, 17, 130, 3, 2), (1, 256, 256, 258, 256, 1, 1), (1, 130, 260, 256, 300, 1, 1), (1, 65, 150, 130, 160, 2, 2)]


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("n,c,h,w,o,kh,kw", CONVS)
def test_conv(dtype, n, c, h, w, o, kh, kw):
    x, f = rnd((n * h * w, c), c + o), rnd((o * kh * kw, c), c * o + 1) / 8
    xc, xs = quantise(x, 0)
    wc, ws = quantise(f, 0)
    x64 = values64(xc.whole(), xs.whole(), c).reshape(n, h, w, c)
    w64 = values64(wc.whole(), ws.whole(), c).reshape(o, kh, kw, c)
    for act, bias in ((0, None), (1, rnd((o,), 7, dtype)), (2, rnd((o,), 8, dtype))):
        ref, size, y = conv64(x64, w64, bias, act)
        got = convolve(xc, xs, (n, c, h, w), wc, ws, (o, c, kh, kw), bias, act, dtype)
        assert ((got.double() - ref).abs() <= step(dtype, ref) + conv_tolerance(size, y, kh * kw * -(-c // 32))).all()


LARGE = [(1, 64, 450, 450, 64, 3, 3), (1, 33, 453, 441, 40, 3, 3), (2, 32, 310, 330, 64, 3, 3), (1, 3, 451, 449, 24, 5, 5), (1, 64, 450, 443, 33, 7, 7),
         (3, 20, 270, 260, 130, 5, 5), (1, 64, 450, 450, 64, 1, 1), (1, 17, 449, 450, 3, 1, 7), (1, 60, 450, 450, 32, 7, 1), (1, 32, 9, 33000, 64, 2, 2),
         (1, 50, 6000, 33, 5, 3, 2), (1, 64, 330, 330, 200, 3, 3), (1, 30, 450, 450, 70, 7, 7)]


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("n,c,h,w,o,kh,kw", LARGE)
def test_conv_of_large_images(dtype, n, c, h, w, o, kh, kw):
    """At most 64 channels of many pixels (the 64-bit reference runs on the GPU here)."""
    x, f = rnd((n * h * w, c), c + o), rnd((o * kh * kw, c), c * o + 1) / 8
    x[(n * h * w) // 2, 1] = float("nan")                        # one pixel in the middle: its neighbours' outputs, and no others
    xc, xs = quantise(x, 0)
    wc, ws = quantise(f, 0)
    x64 = values64(xc.t, xs.t, c).reshape(n, h, w, c)
    w64 = values64(wc.t, ws.t, c).reshape(o, kh, kw, c)
    act = c % 3
    bias = rnd((o,), 7, dtype) if act else None
    ref, size, y = conv64(x64, w64, bias, act)
    got = convolve(xc, xs, (n, c, h, w), wc, ws, (o, c, kh, kw), bias, act, dtype).cuda().double()
    assert int(ref.isnan().sum()) > 0 and torch.equal(got.isnan(), ref.isnan())
    ok = (got - ref).abs() <= step(dtype, ref) + conv_tolerance(size, y, kh * kw * -(-c // 32))
    assert (ok | ref.isnan()).all()


TAPS = [(1, 96, 200, 215, 96, 3, 3), (1, 128, 203, 211, 128, 3, 3), (2, 256, 130, 160, 65, 3, 3), (1, 224, 250, 190, 33, 2, 3),
        (1, 75, 230, 215, 30, 5, 2), (1, 130, 215, 220, 100, 1, 7), (1, 170, 127, 190, 230, 3, 3), (1, 50, 215, 210, 90, 5, 5),
        (3, 7, 125, 127, 75, 7, 1), (1, 160, 8, 6000, 70, 2, 2), (1, 128, 1500, 33, 200, 4, 1), (1, 128, 900, 64, 60, 7, 7),
        (1, 250, 310, 190, 2, 3, 3), (5, 96, 91, 91, 85, 3, 3), (1, 512, 170, 160, 256, 3, 3),
        (1, 380, 210, 213, 90, 2, 2), (1, 640, 250, 190, 20, 1, 5), (2, 290, 130, 160, 60, 3, 3), (1, 1024, 160, 256, 128, 3, 2), (1, 20, 200, 220, 384, 3, 3),
        (2, 4, 130, 190, 290, 5, 5), (1, 500, 210, 213, 40, 2, 3)]


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("n,c,h,w,o,kh,kw", TAPS)
def test_conv_of_several_taps(dtype, n, c, h, w, o, kh, kw):
    """Windows with several taps: every number of blocks and channels of a tile, channels in one part and in several, with NaN in the
    first and in the last block of a pixel."""
    x, f = rnd((n * h * w, c), c + o), rnd((o * kh * kw, c), c * o + 1) / 8
    x[(n * h * w) // 2, 0] = x[(n * h * w) // 3, c - 1] = x[n * h * w - 1, c // 2] = float("nan")
    xc, xs = quantise(x, 0)
    wc, ws = quantise(f, 0)
    x64 = values64(xc.t, xs.t, c).reshape(n, h, w, c)
    w64 = values64(wc.t, ws.t, c).reshape(o, kh, kw, c)
    act = (c + o) % 3
    bias = rnd((o,), 7, dtype) if act else None
    ref, size, y = conv64(x64, w64, bias, act)
    got = convolve(xc, xs, (n, c, h, w), wc, ws, (o, c, kh, kw), bias, act, dtype).cuda().double()
    assert int(ref.isnan().sum()) > 0 and torch.equal(got.isnan(), ref.isnan())
    ok = (got - ref).abs() <= step(dtype, ref) + conv_tolerance(size, y, kh * kw * -(-c // 32))
    assert (ok | ref.isnan()).all()


@pytest.mark.parametrize("c,h,w,o,kh,kw", [(128, 203, 211, 128, 3, 3), (256, 150, 190, 200, 3, 2), (128, 310, 190, 20, 3, 3), (64, 450, 450, 64, 3, 3)])
def test_conv_scales_at_odd_addresses(c, h, w, o, kh, kw):
    """Scales that cannot be read in words: the same results, bit for bit."""
    xc, xs = quantise(rnd((h * w, c), 1), 0)
    wc, ws = quantise(rnd((o * kh * kw, c), 2) / 30, 0)
    ref = convolve(xc, xs, (1, c, h, w), wc, ws, (o, c, kh, kw), None, 2, 0)
    b = c // 32
    for by in (1, 3):
        ms, mf = Guarded((h * w * b + 4,), torch.uint8), Guarded((o * kh * kw * b + 4,), torch.uint8)
        ms.t[by:by + h * w * b], mf.t[by:by + o * kh * kw * b] = xs.t.view(-1), ws.t.view(-1)
        out = Guarded((1, h, w, o), torch.float16)
        S.layer_conv2d_mx4(0, xc.ptr(), ms.ptr() + by, (1, c, h, w), wc.ptr(), mf.ptr() + by, (o, c, kh, kw), None, 2, out.ptr(), stream())
        assert torch.equal(out.whole(), ref)


@pytest.mark.parametrize("c,h,w,o,kh,kw", [(1 << 20, 2, 1400, 2, 3, 1), (4000, 2, 360000, 8, 3, 1), (64, 2, 15000000, 3, 2, 2)])
def test_conv_taps_far_apart(c, h, w, o, kh, kw):
    """Rows of pixels so long that a window's taps are more than 2^31 bytes of codes apart."""
    b = -(-c // 32)
    g = torch.Generator(device="cuda")
    g.manual_seed(c)
    codes = torch.randint(0, 256, (h, w, b, 16), generator=g, device="cuda", dtype=torch.uint8)
    if c % 32:
        codes[:, :, -1, (c % 32) // 2:] = 0                       # what a block is filled up with
    scales = torch.randint(120, 130, (h, w, b), generator=g, device="cuda", dtype=torch.uint8)
    fc = torch.randint(0, 256, (o, kh, kw, b, 16), generator=g, device="cuda", dtype=torch.uint8)
    fs = torch.randint(115, 120, (o, kh, kw, b), generator=g, device="cuda", dtype=torch.uint8)
    out = torch.empty(h, w, o, device="cuda")
    S.layer_conv2d_mx4(1, codes.data_ptr(), scales.data_ptr(), (1, c, h, w), fc.data_ptr(), fs.data_ptr(), (o, c, kh, kw), None, 0, out.data_ptr(), stream())
    torch.cuda.synchronize()
    f64 = values64(fc, fs, c)
    for x0 in (0, w // 2 - 3, w - 7):                             # seven columns and a border of one on either side
        x1, left = x0 + 7, 1 if x0 else 0
        right = 1 if x1 < w else 0
        part = values64(codes[:, x0 - left:x1 + right].contiguous(), scales[:, x0 - left:x1 + right].contiguous(), c)
        ref, size, y = conv64(part[None], f64, None, 0)
        ref, size, y = (v[0, :, left:left + 7] for v in (ref, size, y))
        got = out[:, x0:x1].double()
        assert ((got - ref).abs() <= step(1, ref) + conv_tolerance(size, y, kh * kw * b)).all()


@pytest.mark.parametrize("dtype", [0, 1])
def test_tensors_anywhere(dtype):
    """Tensors at multiples of their element, scales at odd addresses: the same results as aligned ones, bit for bit."""
    n, c, h, w, o, groups = 1, 128, 40, 33, 70, 8
    t = TYPES[dtype]
    size = t.itemsize

    def moved(v, by):
        raw = torch.zeros(v.numel() * v.element_size() + 512, dtype=torch.uint8, device="cuda")
        part = raw[by:by + v.numel() * v.element_size()]
        part.copy_(v.contiguous().view(-1).view(torch.uint8))
        return raw, part, raw.data_ptr() + by

    x, scale, bias, cb = (rnd(s, k, dtype).cuda() for k, s in enumerate([(n, h, w, c), (c,), (c,), (o,)]))
    wc, ws = quantise((rnd((o * 9, c), 9) / 30).to(t), dtype)
    need = S.layer_group_norm_workspace(dtype, (n, c, h, w), groups)
    work = torch.empty(need + 8, dtype=torch.uint8, device="cuda")
    results = []
    for by, odd in ((0, 0), (size, 1), (3 * size, 3)):
        keep = [moved(v, by) for v in (x, scale, bias, cb)]
        px, ps, pb, pc = (k[2] for k in keep)
        y, out, back = (torch.zeros(m * size + 512, dtype=torch.uint8, device="cuda") for m in (x.numel(), n * h * w * o, x.numel()))
        codes, xs = torch.empty(n * h * w * 4, 16, dtype=torch.uint8, device="cuda"), torch.empty(n * h * w * 4 + 8, dtype=torch.uint8, device="cuda")
        fs = torch.empty(o * 36 + 8, dtype=torch.uint8, device="cuda")
        fs[odd:odd + o * 36] = ws.t.view(-1)
        S.layer_group_norm(dtype, px, (n, c, h, w), groups, ps, pb, 1e-5, 2, y.data_ptr() + by, work.data_ptr(), need, stream())
        S.layer_group_norm_mx4(dtype, px, (n, c, h, w), groups, ps, pb, 1e-5, 2, codes.data_ptr(), xs.data_ptr() + odd, work.data_ptr(), need, stream())
        S.layer_conv2d_mx4(dtype, codes.data_ptr(), xs.data_ptr() + odd, (n, c, h, w), wc.ptr(), fs.data_ptr() + odd, (o, c, 3, 3), pc, 1, out.data_ptr() + by, stream())
        S.layer_dequantize_mx4(dtype, codes.data_ptr(), xs.data_ptr() + odd, n * h * w, c, back.data_ptr() + by, stream())
        torch.cuda.synchronize()
        results.append([v[by:by + m * size].clone() for v, m in ((y, x.numel()), (out, n * h * w * o), (back, x.numel()))] + [codes, xs[odd:odd + n * h * w * 4].clone()])
        S.layer_quantize_mx4(dtype, back.data_ptr() + by, n * h * w, c, codes.data_ptr(), xs.data_ptr() + odd, stream())
        torch.cuda.synchronize()
        results[-1][-2] = codes.clone()
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


@pytest.mark.parametrize("m,o", [(1, 40), (5, 64), (700, 150)])
def test_conv_scales_over_their_range(m, o):
    """Scales from 2^-127 to 2^120 whose products stay within fp32, zeros of any scale, and results below fp32."""
    c = 128
    g = torch.Generator().manual_seed(m)
    code = lambda *s: torch.randint(0, 256, s, generator=g, dtype=torch.uint8)  # noqa: E731
    xc, wc = code(m, 4, 16), code(o, 4, 16)
    for sx, sw in ((0, 240), (240, 0), (127, 127), (120, 200), (3, 251), (1, 60), (0, 0)):
        xs, ws = torch.full((m, 4), sx, dtype=torch.uint8), torch.full((o, 4), sw, dtype=torch.uint8)
        xs[:, 1] = 254 - sw if sw > 0 else 200
        G = [Guarded(t.shape, torch.uint8, t) for t in (xc, xs, wc, ws)]
        ref, size, y = conv64(values64(xc, xs, c).reshape(1, 1, m, c), values64(wc, ws, c).reshape(o, 1, 1, c), None, 0)
        got = convolve(G[0], G[1], (1, c, 1, m), G[2], G[3], (o, c, 1, 1), None, 0, 1)
        # below the normal numbers of fp32 every addition may lose 2^-126
        assert ((got.double() - ref).abs() <= step(1, ref) + conv_tolerance(size, y, 4) + 256 * 2.0 ** -126).all(), (sx, sw)
    # zeros stay zeros whatever their scales
    G = [Guarded(t.shape, torch.uint8, t) for t in (torch.zeros_like(xc), torch.full((m, 4), 254, dtype=torch.uint8), wc, torch.full((o, 4), 250, dtype=torch.uint8))]
    assert float(convolve(G[0], G[1], (1, c, 1, m), G[2], G[3], (o, c, 1, 1), None, 0, 1).abs().max()) == 0


@pytest.mark.parametrize("h,w,c,o", [(1, 3, 64, 40), (12, 15, 96, 70), (40, 40, 64, 64)])
def test_conv_nan_blocks(h, w, c, o):
    """A NaN block of a pixel makes NaN of the outputs whose window holds that pixel, one of a filter of its output channel."""
    kh = kw = 3
    x, f = rnd((h * w, c), 1), rnd((o * 9, c), 2) / 8
    x[(h // 2) * w + 1, 40] = float("nan")
    f[5 * 9 + 4, 2] = float("inf")                               # the middle tap of output 5: every pixel uses it
    xc, xs = quantise(x, 0)
    wc, ws = quantise(f, 0)
    got = convolve(xc, xs, (1, c, h, w), wc, ws, (o, c, kh, kw), None, 0, 0)[0]
    want = torch.zeros(h, w, o, dtype=torch.bool)
    want[max(0, h // 2 - 1):h // 2 + 2, 0:3] = True
    want[:, :, 5] = True
    assert torch.equal(got.isnan(), want)


def test_conv_is_the_generic_convolution():
    """Values that 4 bits hold exactly: the same result as srx_layer_conv2d on the same tensors (bias and ReLU)."""
    n, c, h, w, o, k = 1, 32, 19, 23, 48, 3
    g = torch.Generator().manual_seed(2)
    pick = lambda s: GRID[torch.randint(0, 8, s, generator=g)].half() * torch.where(torch.rand(s, generator=g) < 0.5, -1, 1)  # noqa: E731
    x, f = pick((n, h, w, c)), pick((o, k, k, c)) / 16
    x[..., 0], f[..., 0] = 6, 6 / 16                             # every block has the same scale
    bias = rnd((o,), 3)
    dx, df, db = x.cuda(), f.cuda(), bias.cuda()
    dense = torch.empty(n, h, w, o, dtype=torch.float16, device="cuda")
    S.layer_conv2d(0, 1, dx.data_ptr(), (n, c, h, w), df.data_ptr(), (o, c, k, k), db.data_ptr(), dense.data_ptr(), stream())
    xc, xs = quantise(x.reshape(-1, c), 0)
    wc, ws = quantise(f.reshape(-1, c), 0)
    got = convolve(xc, xs, (n, c, h, w), wc, ws, (o, c, k, k), bias, 1, 0)
    want = dense.cpu()
    # both sums are exact here (multiples of 2^-6 below 2^14); what is left is the bias addition and the rounding to fp16
    assert ((got.double() - want.double()).abs() <= 2 * step(0, want.double()) + 2.0 ** -20).all()


# ---------------------------------------------------------------------------
# Together, streams, graphs
# ---------------------------------------------------------------------------
def block(x, groups, scale, bias, wc, ws, o, k, cb, bufs, s):
    n, h, w, c = x.shape
    codes, scales, out, work = bufs
    S.layer_group_norm_mx4(0, x.data_ptr(), (n, c, h, w), groups, scale.data_ptr(), bias.data_ptr(), 1e-5, 2, codes.data_ptr(),
                           scales.data_ptr(), work.data_ptr(), work.numel(), s)
    S.layer_conv2d_mx4(0, codes.data_ptr(), scales.data_ptr(), (n, c, h, w), wc.data_ptr(), ws.data_ptr(), (o, c, k, k), cb.data_ptr(), 0,
                       out.data_ptr(), s)


def block_buffers(n, h, w, c, o, groups):
    b = -(-c // 32)
    return (torch.empty(n * h * w, b, 16, dtype=torch.uint8, device="cuda"), torch.empty(n * h * w, b, dtype=torch.uint8, device="cuda"),
            torch.empty(n, h, w, o, dtype=torch.float16, device="cuda"),
            torch.empty(S.layer_group_norm_workspace(0, (n, c, h, w), groups), dtype=torch.uint8, device="cuda"))


def residual_setup(seed, n, h, w, c, groups):
    x = rnd((n, h, w, c), seed)
    scale, bias, cb = (1 + 0.2 * rnd((c,), seed + 1, 1)).half(), rnd((c,), seed + 2), rnd((c,), seed + 3)
    wc, ws = quantise((rnd((c * 9, c), seed + 4) / (3 * c ** 0.5)).half(), 0)
    return x, scale, bias, cb, wc, ws


def residual64(x, scale, bias, cb, wc, ws, groups, codes, scales):
    """The block's output from the 4-bit tensor in between, which is checked on its own."""
    n, h, w, c = x.shape
    x64 = values64(codes, scales, c).reshape(n, h, w, c)
    return conv64(x64, values64(wc, ws, c).reshape(c, 3, 3, c), cb, 0)


@pytest.mark.parametrize("n,h,w,c,groups", [(1, 9, 13, 64, 8), (2, 31, 17, 80, 16), (1, 64, 64, 96, 3)])
def test_residual_block(n, h, w, c, groups):
    """x + conv(silu(norm(x))): the layers one after another, and the addition of the framework's own layer."""
    x, scale, bias, cb, wc, ws = residual_setup(c, n, h, w, c, groups)
    dx = x.cuda()
    bufs = block_buffers(n, h, w, c, c, groups)
    d = [t.cuda() for t in (scale, bias, cb)]
    block(dx, groups, d[0], d[1], wc.t, ws.t, c, 3, d[2], bufs, stream())
    out = torch.empty_like(dx)
    S.layer_add(0, dx.data_ptr(), bufs[2].data_ptr(), out.data_ptr(), dx.numel(), stream())
    torch.cuda.synchronize()
    ref, *parts = norm64(x, groups, scale, bias, 1e-5, 2)
    G = [Guarded(b.shape, torch.uint8, b) for b in bufs[:2]]
    check_codes(*G, ref.reshape(-1, c), norm_tolerance(*parts).reshape(-1, c))
    y, size, raw = residual64(x, scale, bias, cb, wc.whole(), ws.whole(), groups, bufs[0].cpu(), bufs[1].cpu())
    tol = step(0, y) + conv_tolerance(size, raw, 9 * -(-c // 32))
    assert ((bufs[2].cpu().double() - y).abs() <= tol).all()
    assert ((out.cpu().double() - (x.double() + y)).abs() <= tol + step(0, x.double().abs() + y.abs() + tol)).all()


def test_two_streams_and_a_foreign_default_stream():
    """Two blocks at once on streams of their own, each with its own buffers, give what they give alone, bit for bit."""
    shapes = [(1, 90, 70, 64, 8), (2, 33, 41, 96, 6)]
    runs = []
    for k, (n, h, w, c, g) in enumerate(shapes):
        x, scale, bias, cb, wc, ws = residual_setup(50 + k, n, h, w, c, g)
        args = (x.cuda(), g, scale.cuda(), bias.cuda(), wc.t, ws.t, c, 3, cb.cuda())
        alone = block_buffers(n, h, w, c, c, g)
        block(*args, alone, stream())
        torch.cuda.synchronize()
        runs.append((args, alone, block_buffers(n, h, w, c, c, g), torch.cuda.Stream(), (wc, ws)))
    for _ in range(5):
        for args, _, bufs, s, _ in runs:
            block(*args, bufs, s.cuda_stream)
    torch.cuda.synchronize()
    for _, alone, bufs, _, _ in runs:
        assert all(torch.equal(a, b) for a, b in zip(alone[:3], bufs[:3]))


def test_captured_and_replayed():
    """Every layer in one graph; replayed with new inputs, eager work in between, equal to the eager calls bit for bit."""
    n, h, w, c, g = 1, 60, 50, 64, 8
    x, scale, bias, cb, wc, ws = residual_setup(90, n, h, w, c, g)
    dx, d = x.cuda(), [t.cuda() for t in (scale, bias, cb)]
    bufs, eager = block_buffers(n, h, w, c, c, g), block_buffers(n, h, w, c, c, g)
    y, ey = torch.empty_like(dx), torch.empty_like(dx)

    def run(b, o, s):
        block(dx, g, d[0], d[1], wc.t, ws.t, c, 3, d[2], b, s)
        S.layer_quantize_mx4(0, b[2].data_ptr(), n * h * w, c, b[0].data_ptr(), b[1].data_ptr(), s)
        S.layer_dequantize_mx4(0, b[0].data_ptr(), b[1].data_ptr(), n * h * w, c, o.data_ptr(), s)
        S.layer_group_norm(0, o.data_ptr(), (n, c, h, w), g, None, None, 1e-5, 0, o.data_ptr(), b[3].data_ptr(), b[3].numel(), s)

    run(eager, ey, stream())                                     # kernels are loaded before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(bufs, y, torch.cuda.current_stream().cuda_stream)
    for k in range(4):
        dx.copy_(rnd((n, h, w, c), 200 + k).cuda())
        graph.replay()
        run(eager, ey, stream())
        torch.cuda.synchronize()
        assert torch.equal(y, ey) and torch.equal(bufs[2], eager[2])
