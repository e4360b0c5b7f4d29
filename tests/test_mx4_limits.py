"""Sizes and arguments of the normalisation and 4-bit layers at the ends of their ranges, without a GPU."""
import pytest

import superresolution_amd as S

P = 1 << 20          # an address no refused call looks at
INVALID = 1


def refused(call, *args):
    with pytest.raises(S.SrxError) as e:
        call(*args)
    assert e.value.status == INVALID
    return str(e.value)


@pytest.mark.parametrize("sizes", [
    (1 << 16,) * 4,                                     # 2^64 values: none, in 64 bits
    ((1 << 32) - 1,) * 4, (1 << 20, 1 << 20, 1 << 20, 1 << 4), (3, 1 << 20, (1 << 32) - 1, 1 << 31), (1, 1 << 10, 1 << 15, 1 << 15)])
def test_values_are_counted_past_64_bits(sizes):
    refused(S.layer_group_norm_workspace, 0, sizes, 1)
    assert "sizes" in refused(S.layer_group_norm, 0, P, sizes, 1, None, None, 1e-5, 0, P, P, 1 << 60)
    refused(S.layer_plan, 0, 0, sizes, (1, sizes[1], 1, 1))
    refused(S.layer_plan, 2, 0, sizes, (1, 1, 1, 1))
    refused(S.layer_plan, 0, 0, (1, sizes[1], 1, 1), sizes)


@pytest.mark.parametrize("n,h,w", [(1 << 22, 1 << 21, 1 << 21), (1 << 31, 1 << 31, 4), ((1 << 32) - 1,) * 3, (1, 1 << 16, 1 << 15)])
def test_pixels_are_counted_past_64_bits(n, h, w):
    """(2^64 pixels are none in 64 bits, and rows and columns of 2^42 pixels none in 32.)"""
    for c in (1, 32):
        assert "sizes" in refused(S.layer_conv2d_mx4, 0, P, P, (n, c, h, w), P, P, (1, c, 1, 1), None, 0, P)


def test_the_largest_tensor_is_taken():
    assert S.layer_plan(2, 0, (1, 1, (1 << 20) - 1, (1 << 20) + 1), (1, 1, 1, 1))[0] == (1, 1, (1 << 20) - 1, (1 << 20) + 1)
    refused(S.layer_plan, 2, 0, (1, 1, 1 << 20, 1 << 20), (1, 1, 1, 1))


@pytest.mark.parametrize("by", [1 << 32, -(1 << 32), 1 << 64])
def test_numbers_past_their_type_are_refused(by):
    """Not taken for what their low bits are."""
    sizes = (1, 8, 4, 4)
    for i in range(4):
        far = tuple(v + by * (k == i) for k, v in enumerate(sizes))
        refused(S.layer_group_norm_workspace, 0, far, 2)
        assert "32 bits" in refused(S.layer_conv2d_mx4, 0, P, P, far, P, P, (5, 8, 3, 3), None, 0, P)
        assert "32 bits" in refused(S.layer_conv2d_mx4, 0, P, P, sizes, P, P, far, None, 0, P)
        assert "32 bits" in refused(S.layer_plan, 0, 0, far, (5, 8, 3, 3))
    refused(S.layer_group_norm_workspace, 0, sizes, 2 + by)
    refused(S.layer_group_norm_workspace, by, sizes, 2)
    for call in (S.layer_group_norm, lambda *a: S.layer_group_norm_mx4(*a[:8], P, *a[8:])):
        for dtype, groups, act, nbytes in ((by, 2, 0, 1 << 20), (0, 2 + by, 0, 1 << 20), (0, 2, by, 1 << 20), (0, 2, 0, -1), (0, 2, 0, (1 << 64) + (1 << 20))):
            assert "out of range" in refused(call, dtype, P, sizes, groups, P, P, 1e-5, act, P, P, nbytes)
    assert "out of range" in refused(S.layer_conv2d_mx4, by, P, P, sizes, P, P, (5, 8, 3, 3), None, 0, P)
    assert "out of range" in refused(S.layer_conv2d_mx4, 0, P, P, sizes, P, P, (5, 8, 3, 3), None, by, P)


@pytest.mark.parametrize("rows,columns", [((1 << 64) + 3, 32), (3, (1 << 64) + 32), (3 - (1 << 64), 32), (-1, 32), (3, -32)])
def test_rows_and_columns_past_64_bits_are_refused(rows, columns):
    refused(S.layer_mx4_sizes, rows, columns)
    assert "out of range" in refused(S.layer_quantize_mx4, 0, P, rows, columns, P, P)
    assert "out of range" in refused(S.layer_dequantize_mx4, 0, P, P, rows, columns, P)


@pytest.mark.parametrize("sizes", [(1, 8, 4), (1, 8, 4, 4, 1)])
def test_sizes_are_four(sizes):
    with pytest.raises((S.SrxError, IndexError)):
        S.layer_group_norm_workspace(0, sizes, 2)


@pytest.mark.parametrize("n,c,h,w,groups", [
    (1024, 1032, 20, 25, 1), (64, 1032, 128, 128, 1), (64, 2040, 128, 128, 8), (64, 696, 200, 200, 3), (256, 2048, 64, 64, 4),
    (64, 5000, 64, 64, 50), (1, 4, 8192, 8192, 2), (1024, 8, 256, 256, 2), (2, 520, 2048, 2048, 1)])
def test_parts_are_short_enough_for_sums_in_32_bits(n, c, h, w, groups):
    """The statistics of an image come in parts (a mean and a sum of squares of 4 bytes each, and once more where there are over
    64), whose pixels 256 threads of eight channels share: no thread may add up more than 256 of them."""
    need = S.layer_group_norm_workspace(0, (n, c, h, w), groups)
    parts = need // (n * groups * 8)
    assert need == parts * n * groups * 8
    parts -= parts > 64
    pixels = -(-h * w // parts)
    k = c // groups
    vecs = -(-k * min(groups, 2048 // k) // 8)                   # of a workgroup's whole groups
    assert vecs <= 256 and -(-pixels // (256 // vecs)) <= 256
