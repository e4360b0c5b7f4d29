"""Group normalisation of fp32 values at the end of their range, and of values far from the others, against the definition in
64 bits.  Helpers and tolerances are those of test_gpu_mx4."""
import pytest
import torch

import superresolution_amd as S
from test_gpu_mx4 import Guarded, U, check_codes, group_norm, norm64, norm_tolerance, step, stream

pytestmark = pytest.mark.gpu

# n, c, h, w, groups: one workgroup holds one group, several groups; parts joined by the output kernel, by a kernel of their own
SHAPES = [(2, 64, 8, 9, 2), (2, 96, 16, 16, 12), (2, 64, 120, 100, 2), (2, 64, 600, 500, 4)]
WIDE = (2, 4224, 5, 3, 1)                                        # a group wider than a workgroup


def moments(v):
    """Mean and variance of a matrix of many rows on the GPU, in 64 bits.  Rows are summed up there and joined on the host: one
    result of many blocks, as torch's mean() of it all, has been wrong here once in 1e5 times."""
    mean = float(v.sum(1).cpu().sum() / v.numel())
    return mean, float(((v - mean) ** 2).sum(1).cpu().sum() / v.numel())


def every(ok):
    return bool(ok.reshape(ok.shape[0], -1).all(1).cpu().all())


def noise(shape, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("size", [3e38, 1e20, None])
@pytest.mark.parametrize("n,c,h,w,groups", SHAPES + [WIDE])
def test_squares_past_the_range_make_nan(size, n, c, h, w, groups):
    """Of image 1, group 0: squares that pass the range of fp32, and squares a 64th of it whose sum passes it."""
    k = c // groups
    x = noise((n, h, w, c), 1)
    sign = torch.where(torch.arange(h * w * k) % 2 == 0, 1.0, -1.0).reshape(h, w, k)
    ref, *parts = norm64(x, groups, None, None, 1e-5, 2)
    x[1, :, :, :k] = sign * (size or 2.0 ** 61)
    got = group_norm(x, 1, groups, None, None, 2)
    assert got[1, :, :, :k].isnan().all()
    other = torch.ones(n, h, w, c, dtype=torch.bool)
    other[1, :, :, :k] = False
    assert ((got.double() - ref).abs() <= step(1, ref) + norm_tolerance(*parts))[other].all()
    codes, scales = group_norm(x, 1, groups, None, None, 2, mx4=True)
    blocks = -(-c // 32)
    bad = torch.zeros(n, h * w, blocks, dtype=torch.bool)
    bad[1, :, :-(-k // 32)] = True                               # blocks that hold a value of the group
    assert torch.equal((scales.whole() == 255).reshape(bad.shape), bad)
    assert (codes.whole().reshape(*bad.shape, 16)[bad] == 0).all()


@pytest.mark.parametrize("n,c,h,w,groups", SHAPES + [WIDE])
def test_squares_within_the_range_are_normalised(n, c, h, w, groups):
    """The squared deviations' sum is a quarter of fp32's range."""
    k = c // groups
    x = noise((n, h, w, c), 2) * (2.0 ** 126 / (h * w * k)) ** 0.5
    ref, *parts = norm64(x, groups, None, None, 1e-5, 0)
    got = group_norm(x, 1, groups, None, None, 0)
    assert ((got.double() - ref).abs() <= step(1, ref) + norm_tolerance(*parts)).all()
    check_codes(*group_norm(x, 1, groups, None, None, 0, mx4=True), ref.reshape(-1, c), norm_tolerance(*parts).reshape(-1, c))


@pytest.mark.parametrize("n,c,h,w,groups", SHAPES + [WIDE, (1, 1 << 18, 3, 1, 2)])
def test_one_value_takes_half_the_range(n, c, h, w, groups):
    """The first value of every group is 2^63.5 and the others are small against it: the squared deviations' sum is half the range
    of fp32, but squares about that value pass it from the third on."""
    x = noise((n, h, w, c), 3)
    x[:, 0, 0, ::c // groups] = 2.0 ** 63.5
    ref, *parts = norm64(x, groups, None, None, 1e-5, 0)
    got = group_norm(x, 1, groups, None, None, 0)
    assert ((got.double() - ref).abs() <= step(1, ref) + norm_tolerance(*parts)).all()


def test_a_sum_whose_square_passes_the_range():
    """256 values of a thread about a first one 1e17 away: the square of their sum passes the range of fp32, nothing else does."""
    n, h, w, c, d = 1, 8192, 8192, 4, 1e17
    x = torch.randn(n, h, w, c, device="cuda", generator=torch.Generator("cuda").manual_seed(2)) * 1e10
    x.view(-1, c)[65536] = d                                     # the first pixel of a part
    want = x.double().view(h, w, 2, 2)
    for group in range(2):
        mean, var = moments(want[:, :, group].reshape(1 << 16, -1))
        want[:, :, group] = (want[:, :, group] - mean) / (var + 1e-5) ** 0.5
    want = want.view(n, h, w, c)
    out = torch.empty_like(x)
    need = S.layer_group_norm_workspace(1, (n, c, h, w), 2)
    work = Guarded((need,), torch.uint8)
    S.layer_group_norm(1, x.data_ptr(), (n, c, h, w), 2, None, None, 1e-5, 0, out.data_ptr(), work.ptr(), need, stream())
    torch.cuda.synchronize()
    # A difference of the 255 is off by U d at most, and counts with the d / 256 that it is off their mean: 2 U d^2 of the sum of
    # squared deviations, which is d^2, and half of that in the result; 80 half steps for the rest, as in norm_tolerance.
    assert every(((out.double() - want).abs() <= U * (want.abs() + 80 * (want.abs() + 1)))[0])


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("n,c,h,w", [(1, 1 << 20, 2, 1), (1, 4100, 5, 3), (2, 100003, 3, 1), (8, 2064, 64, 64)])
def test_wide_group_first_values_far_from_the_others(dtype, n, c, h, w):
    """A group wider than a workgroup, whose threads add up thousands of values (2^20 channels: 4096) about the first one."""
    x = noise((n, h, w, c), 4)
    x[:, 0, 0, :2048:8] += 300                                   # the first value of each of 256 threads
    x = x.to(torch.float32 if dtype else torch.float16)
    ref, *parts = norm64(x, 1, None, None, 1e-5, 0)
    got = group_norm(x, dtype, 1, None, None, 0)
    assert ((got.double() - ref).abs() <= step(dtype, ref) + norm_tolerance(*parts)).all()


def test_wide_group_in_parts_of_many_values():
    """So many images that a workgroup takes 241 pixels of one: threads add up 1928 to 3856 values, the first of which is far."""
    n, c, h, w = 64, 2064, 64, 64
    x = torch.randn(n, h * w, c, device="cuda", generator=torch.Generator("cuda").manual_seed(5))
    x[:, ::241, :2048:8] += 300
    out = torch.empty_like(x)
    need = S.layer_group_norm_workspace(1, (n, c, h, w), 1)
    assert need == n * -(-h * w // 241) * 8
    work = Guarded((need,), torch.uint8)
    S.layer_group_norm(1, x.data_ptr(), (n, c, h, w), 1, None, None, 1e-5, 0, out.data_ptr(), work.ptr(), need, stream())
    work.whole()
    for i in range(n):
        v = x[i].double()
        mean, var = moments(v)
        rstd = 1 / (var + 1e-5) ** 0.5
        v = (v - mean) * rstd
        assert every((out[i].double() - v).abs() <= U * (v.abs() + 80 * (abs(mean) * rstd + v.abs() + 1)))


@pytest.mark.parametrize("dtype", [0, 1])
def test_one_row_of_threads_first_values_far_from_the_others(dtype):
    """1032 channels: 129 threads a pixel, so that one row of them adds up a part's pixels, the first of which is far."""
    n, c, h, w, d = 64, 1032, 64, 64, 300.0
    x = torch.randn(n, h * w, c, device="cuda", generator=torch.Generator("cuda").manual_seed(6))
    x[:, ::256] += d
    x = x.to(torch.float32 if dtype else torch.float16)
    out = torch.empty_like(x)
    need = S.layer_group_norm_workspace(dtype, (n, c, h, w), 1)
    assert need == n * 16 * 8                                    # 16 parts of 256 pixels
    work = Guarded((need,), torch.uint8)
    S.layer_group_norm(dtype, x.data_ptr(), (n, c, h, w), 1, None, None, 1e-5, 0, out.data_ptr(), work.ptr(), need, stream())
    work.whole()
    # fp16: sums in 32 bits, as in test_group_norm_first_value_far_from_the_others, but every channel of every part has a far value
    off = 1.5 * 256 ** 2 * U * d ** 2 / (256 + d ** 2) / 2 if dtype == 0 else 0
    for i in range(n):
        v = x[i].double()
        mean, var = moments(v)
        rstd = 1 / (var + 1e-5) ** 0.5
        v = (v - mean) * rstd
        tol = off * v.abs() + U * (80 * (abs(mean) * rstd + v.abs() + 1) + d * rstd)
        if dtype == 0:
            tol += v.abs() * 2.0 ** -11 + 2.0 ** -25 + 256 * U * d * rstd        # and each part's mean
        else:
            tol += U * v.abs()
        assert every((out[i].double() - v).abs() <= tol)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("n,c,h,w,groups", [(1, 64, 256, 190, 64), (1, 128, 128, 190, 128), (1, 512, 60, 90, 512), (2, 90, 150, 210, 45)])
def test_many_groups_of_many_parts(dtype, n, c, h, w, groups):
    """The output kernel joins up to 64 parts of a group by four lanes and fewer: 16 to 64 parts a lane."""
    x = noise((n, h, w, c), 7) * torch.exp2(noise((c,), 8)) + noise((c,), 9)
    x = x.to(torch.float32 if dtype else torch.float16)
    parts = S.layer_group_norm_workspace(dtype, (n, c, h, w), groups) // (n * groups * 8)
    assert parts == 64
    ref, *rest = norm64(x, groups, None, None, 1e-5, 2)
    got = group_norm(x, dtype, groups, None, None, 2)
    assert ((got.double() - ref).abs() <= step(dtype, ref) + norm_tolerance(*rest)).all()
    blocks = group_norm(x, dtype, groups, None, None, 2, mx4=True)
    check_codes(*blocks, ref.reshape(-1, c), norm_tolerance(*rest).reshape(-1, c))


def test_more_parts_than_a_wave_keeps():
    """1040 parts of an image, joined by the 64 lanes of a wave."""
    n, c, h, w, groups = 1, 1032, 520, 512, 8
    x = torch.randn(h * w, groups, c // groups, device="cuda", generator=torch.Generator("cuda").manual_seed(8)).half()
    x[:, 3] += torch.linspace(-3, 3, h * w, device="cuda")[:, None].half()      # parts with means of their own
    need = S.layer_group_norm_workspace(0, (n, c, h, w), groups)
    assert need == (1040 + 1) * groups * 8
    out, work = torch.empty_like(x), Guarded((need,), torch.uint8)
    S.layer_group_norm(0, x.data_ptr(), (n, c, h, w), groups, None, None, 1e-5, 0, out.data_ptr(), work.ptr(), need, stream())
    work.whole()
    for g in range(groups):
        v = x[:, g].double()
        mean, var = moments(v)
        rstd = 1 / (var + 1e-5) ** 0.5
        v = (v - mean) * rstd
        assert every((out[:, g].double() - v).abs() <= v.abs() * 2.0 ** -11 + 2.0 ** -25 + U * 80 * (abs(mean) * rstd + v.abs() + 1))


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("n,c,h,w,groups", [(1, 399, 4, 9, 133), (2, 144, 8, 8, 3), (3, 120, 5, 5, 5), (1, 205, 9, 9, 41), (2, 112, 16, 16, 7), (3, 33, 5, 5, 33)])
def test_last_tile_of_groups_narrower_than_the_others(dtype, n, c, h, w, groups):
    """Images held in registers, whose groups come in tiles of whole blocks and a rest: nothing is written behind the rest's blocks,
    where the next pixel's are."""
    x = noise((n, h, w, c), 10).to(torch.float32 if dtype else torch.float16)
    assert S.layer_group_norm_workspace(dtype, (n, c, h, w), groups) == 0
    for act in range(3):
        ref, *rest = norm64(x, groups, None, None, 1e-5, act)
        blocks = group_norm(x, dtype, groups, None, None, act, mx4=True)
        check_codes(*blocks, ref.reshape(-1, c), norm_tolerance(*rest).reshape(-1, c))
        got = group_norm(x, dtype, groups, None, None, act)
        assert ((got.double() - ref).abs() <= step(dtype, ref) + norm_tolerance(*rest)).all()
