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
