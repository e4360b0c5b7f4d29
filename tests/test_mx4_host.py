"""The normalisation and 4-bit layers without a GPU: sizes, and calls that are refused before anything is launched."""
import ctypes as C

import pytest

import superresolution_amd as S

P = 1 << 20          # an address no refused call looks at
INVALID = 1


def refused(call, *args):
    with pytest.raises(S.SrxError) as e:
        call(*args)
    assert e.value.status == INVALID
    return str(e.value)


@pytest.mark.parametrize("rows,columns,codes,scales", [(1, 1, 16, 1), (1, 32, 16, 1), (3, 33, 96, 6), (7, 64, 224, 14),
                                                       (1 << 31, 64, 1 << 36, 1 << 32)])
def test_block_form_sizes(rows, columns, codes, scales):
    assert S.layer_mx4_sizes(rows, columns) == (codes, scales)


@pytest.mark.parametrize("rows,columns", [(0, 1), (1, 0), (1 << 40, 1), (1, (1 << 20) + 1), (1 << 38, 32)])
def test_block_form_sizes_refused(rows, columns):
    refused(S.layer_mx4_sizes, rows, columns)
    refused(S.layer_quantize_mx4, 0, P, rows, columns, P, P)
    refused(S.layer_dequantize_mx4, 0, P, P, rows, columns, P)


def test_block_form_arguments_refused():
    refused(S.layer_quantize_mx4, 2, P, 1, 1, P, P)              # data type
    refused(S.layer_quantize_mx4, 0, None, 1, 1, P, P)
    refused(S.layer_quantize_mx4, 0, P, 1, 1, None, P)
    refused(S.layer_quantize_mx4, 0, P, 1, 1, P, None)
    refused(S.layer_quantize_mx4, 0, P + 1, 1, 1, P, P)          # fp16 at an odd address
    refused(S.layer_quantize_mx4, 1, P + 2, 1, 1, P, P)          # fp32 at half its size
    refused(S.layer_quantize_mx4, 0, P, 1, 1, P + 8, P)          # codes at a multiple of 16
    refused(S.layer_dequantize_mx4, -1, P, P, 1, 1, P)
    refused(S.layer_dequantize_mx4, 0, None, P, 1, 1, P)
    refused(S.layer_dequantize_mx4, 0, P, None, 1, 1, P)
    refused(S.layer_dequantize_mx4, 0, P, P, 1, 1, None)
    refused(S.layer_dequantize_mx4, 0, P, P, 1, 1, P + 1)


def norm(dtype=0, x=P, sizes=(1, 8, 300, 200), groups=2, scale=P, bias=P, epsilon=1e-5, act=0, out=P, work=P, nbytes=1 << 20):
    return (dtype, x, sizes, groups, scale, bias, epsilon, act, out, work, nbytes)


@pytest.mark.parametrize("change", [
    dict(dtype=2), dict(dtype=-1), dict(x=None), dict(out=None), dict(sizes=(0, 8, 4, 4)), dict(sizes=(1, 0, 4, 4)),
    dict(sizes=(1, 8, 0, 4)), dict(sizes=(1, 8, 4, 0)), dict(groups=0), dict(groups=3), dict(groups=16), dict(epsilon=0.0),
    dict(epsilon=-1.0), dict(epsilon=1e-40), dict(epsilon=float("nan")), dict(epsilon=float("inf")), dict(act=3), dict(act=-1), dict(work=None),
    dict(nbytes=8), dict(work=P + 4), dict(x=P + 1), dict(scale=P + 1), dict(bias=P + 1), dict(out=P + 1),
    dict(dtype=1, x=P + 2), dict(sizes=(1, (1 << 20) + 2, 1, 1)), dict(sizes=(1 << 20, 1 << 10, 1 << 10, 1 << 5))])
def test_group_norm_arguments_refused(change):
    args = norm(**change)
    refused(S.layer_group_norm, *args)
    dtype, x, sizes, groups, scale, bias, epsilon, act, out, work, nbytes = args
    codes = out if out != P + 1 else P + 8
    refused(S.layer_group_norm_mx4, dtype, x, sizes, groups, scale, bias, epsilon, act, codes, P, work, nbytes)


def test_group_norm_counts_groups_in_31_bits():
    refused(S.layer_group_norm, *norm(sizes=(1 << 31, 1, 1, 1), groups=1))
    refused(S.layer_group_norm, *norm(sizes=(1 << 28, 8, 1, 1), groups=8))
    refused(S.layer_group_norm_workspace, 0, (1 << 28, 8, 1, 1), 8)
    assert S.layer_group_norm_workspace(0, ((1 << 28) - 1, 8, 1, 1), 8) == 0


def test_group_norm_mx4_needs_both_outputs():
    refused(S.layer_group_norm_mx4, 0, P, (1, 8, 4, 4), 2, P, P, 1e-5, 0, P, None, P, 1 << 20)


def test_group_norm_workspace():
    need = S.layer_group_norm_workspace(0, (2, 64, 300, 200), 32)
    assert 0 < need < 1 << 20
    assert "%d bytes" % need in refused(S.layer_group_norm, *norm(sizes=(2, 64, 300, 200), groups=32, nbytes=need - 1))
    refused(S.layer_group_norm_workspace, 0, (2, 64, 300, 200), 5)
    refused(S.layer_group_norm_workspace, 3, (2, 64, 300, 200), 4)
    assert S.lib().srx_layer_group_norm_workspace(0, C.byref((C.c_uint32 * 4)(1, 8, 4, 4)), 2, None) == INVALID


def conv(dtype=0, codes=P, scales=P, sizes=(1, 8, 4, 4), fc=P, fs=P, fsizes=(5, 8, 3, 3), bias=P, act=0, out=P):
    return (dtype, codes, scales, sizes, fc, fs, fsizes, bias, act, out)


@pytest.mark.parametrize("change", [
    dict(dtype=2), dict(codes=None), dict(scales=None), dict(fc=None), dict(fs=None), dict(out=None), dict(act=3), dict(act=-1),
    dict(fsizes=(5, 9, 3, 3)), dict(fsizes=(5, 8, 8, 3)), dict(fsizes=(5, 8, 3, 8)), dict(fsizes=(0, 8, 3, 3)),
    dict(fsizes=(5, 8, 0, 3)), dict(sizes=(0, 8, 4, 4)), dict(sizes=(1, 8, 4, 0)), dict(codes=P + 8), dict(fc=P + 4),
    dict(out=P + 1), dict(bias=P + 1), dict(dtype=1, out=P + 2), dict(sizes=(2, 8, 1 << 15, 1 << 15)),
    dict(sizes=(1, (1 << 20) + 32, 1, 1), fsizes=(1, (1 << 20) + 32, 1, 1)), dict(fsizes=((1 << 20) + 1, 8, 1, 1)),
    dict(sizes=(1, 1 << 20, 4, 4), fsizes=(1, 1 << 20, 4, 4))])
def test_conv_arguments_refused(change):
    refused(S.layer_conv2d_mx4, *conv(**change))


def test_host_memory_is_refused():
    """Memory of the host (and, without a GPU, any memory) is refused, not read by a kernel."""
    buf = (C.c_uint8 * 4096)()
    p = (C.addressof(buf) + 15) & ~15
    assert "not device memory" in refused(S.layer_quantize_mx4, 0, p, 1, 32, p + 1024, p + 2048)
    assert "not device memory" in refused(S.layer_dequantize_mx4, 0, p, p + 1024, 1, 32, p + 2048)
    need = S.layer_group_norm_workspace(0, (1, 8, 4, 4), 2)
    assert "not device memory" in refused(S.layer_group_norm, *norm(x=p, sizes=(1, 8, 4, 4), out=p, scale=None, bias=None, work=p + 2048, nbytes=need))
    assert "not device memory" in refused(S.layer_conv2d_mx4, *conv(codes=p, scales=p, fc=p, fs=p, bias=None, out=p))
