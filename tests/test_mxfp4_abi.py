"""What the MXFP4 entry points refuse before they touch CUDA, what they answer without work to do, and the sizes they give. CPU only."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def L():
    from flashrt_b200 import lib
    return lib


P = C.c_void_p(4096)        # an address that no refused call reads


def with_(args, i, v):
    a = list(args)
    a[i] = v
    return a


def test_sizes(L):
    f = L.lib.frx_mxfp4_packed_bytes
    assert f(128, 128) == 8704 and f(1, 128) == 8704 and f(129, 256) == 4 * 8704 and f(2048, 512) == 2048 * 512 * 17 // 32
    for bad in ((0, 128), (128, 0), (128, 64), (128, 130), (-1, 128)):
        assert f(*bad) == 0
    g = L.lib.frx_mxfp4_moe_layer_workspace_bytes
    assert g(1, 10, 2048, 512, 512) > 0 and g(16384, 10, 2048, 512, 512) > 163840 * 2048 * 2
    assert g(0, 1, 128, 128, 1) > 0
    for bad in ((-1, 1, 128, 128, 1), (1, 0, 128, 128, 1), (1, 33, 128, 128, 64), (1, 1, 64, 128, 1), (1, 1, 128, 100, 1), (1, 1, 128, 128, 0), (1, 1, 128, 128, 4097), (2 ** 27, 32, 128, 128, 64)):
        assert g(*bad) == 0


def test_quantize_refusals(L):
    ok = [None, P, 64, 0, 4, 64, P, P]
    for i, v, rc in ((1, None, L.ERR_ARG), (1, C.c_void_p(4098), L.ERR_ARG), (2, 63, L.ERR_ARG), (3, 3, L.ERR_ARG), (4, -1, L.ERR_ARG), (5, -32, L.ERR_ARG), (5, 48, L.ERR_SHAPE),
                     (6, None, L.ERR_ARG), (6, C.c_void_p(4104), L.ERR_ARG), (7, None, L.ERR_ARG)):
        assert L.lib.frx_mxfp4_quantize(*with_(ok, i, v)) == rc, (i, v)
    assert L.lib.frx_mxfp4_quantize(None, P, 2 ** 30, 0, 2 ** 20, 2 ** 20, P, P) == L.ERR_SHAPE
    assert L.lib.frx_mxfp4_quantize(None, None, 64, 0, 0, 64, None, None) == L.OK
    back = [None, P, P, 4, 64, 1, P, 64]
    for i, v, rc in ((1, None, L.ERR_ARG), (1, C.c_void_p(4097), L.ERR_ARG), (2, None, L.ERR_ARG), (3, -1, L.ERR_ARG), (4, 40, L.ERR_SHAPE), (5, 2, L.ERR_ARG), (6, None, L.ERR_ARG),
                     (6, C.c_void_p(4097), L.ERR_ARG), (7, 60, L.ERR_ARG)):
        assert L.lib.frx_mxfp4_dequantize(*with_(back, i, v)) == rc, (i, v)
    assert L.lib.frx_mxfp4_dequantize(None, None, None, 0, 64, 0, None, 64) == L.OK


def test_pack_refusals(L):
    ok = [None, P, P, 2, 130, 256, P]
    for i, v, rc in ((1, None, L.ERR_ARG), (1, C.c_void_p(4100), L.ERR_ARG), (2, C.c_void_p(4098), L.ERR_ARG), (3, -1, L.ERR_ARG), (4, 0, L.ERR_SHAPE), (5, 200, L.ERR_SHAPE), (6, None, L.ERR_ARG),
                     (3, 2 ** 30, L.ERR_SHAPE)):
        assert L.lib.frx_mxfp4_pack(*with_(ok, i, v)) == rc, (i, v)
    assert L.lib.frx_mxfp4_unpack(None, None, 2, 130, 256, P, P) == L.ERR_ARG
    assert L.lib.frx_mxfp4_unpack(None, P, 2, 130, 192, P, P) == L.ERR_SHAPE
    assert L.lib.frx_mxfp4_pack(None, None, None, 0, 130, 256, None) == L.OK


def test_product_refusals(L):
    ok = [None, P, P, 4, 256, P, 100, P, 100, 1]
    for i, v, rc in ((1, None, L.ERR_ARG), (1, C.c_void_p(4104), L.ERR_ARG), (2, C.c_void_p(4098), L.ERR_ARG), (3, -1, L.ERR_ARG), (4, 96, L.ERR_SHAPE), (4, 0, L.ERR_SHAPE), (5, None, L.ERR_ARG),
                     (5, C.c_void_p(4104), L.ERR_ARG), (6, 0, L.ERR_SHAPE), (7, None, L.ERR_ARG), (7, C.c_void_p(4097), L.ERR_ARG), (8, 99, L.ERR_ARG), (9, 4, L.ERR_ARG)):
        assert L.lib.frx_mxfp4_matmul(*with_(ok, i, v)) == rc, (i, v)
    assert L.lib.frx_mxfp4_matmul(None, None, None, 0, 256, None, 100, None, 100, 0) == L.OK
    moe = [None, P, P, 4, 256, P, 8, 100, P, P, 2, 8, P, 100, 0]
    for i, v, rc in ((1, None, L.ERR_ARG), (3, -1, L.ERR_ARG), (4, 64, L.ERR_SHAPE), (5, None, L.ERR_ARG), (6, 0, L.ERR_SHAPE), (6, 4097, L.ERR_SHAPE), (7, 0, L.ERR_SHAPE), (8, None, L.ERR_ARG),
                     (10, 0, L.ERR_ARG), (11, -1, L.ERR_ARG), (12, None, L.ERR_ARG), (13, 99, L.ERR_ARG), (14, -1, L.ERR_ARG)):
        assert L.lib.frx_mxfp4_moe_matmul(*with_(moe, i, v)) == rc, (i, v)
    # without slot_of there is a row of x for every row of y
    assert L.lib.frx_mxfp4_moe_matmul(None, P, P, 7, 256, P, 8, 100, P, None, 1, 8, P, 100, 0) == L.ERR_ARG
    assert L.lib.frx_mxfp4_moe_matmul(None, P, P, 8, 256, P, 8, 100, P, None, 2, 8, P, 100, 0) == L.ERR_ARG
    assert L.lib.frx_mxfp4_moe_matmul(None, None, None, 0, 256, None, 8, 100, None, None, 1, 0, None, 100, 0) == L.OK


def test_layer_refusals(L):
    n, ff, E = 256, 128, 8
    need = L.lib.frx_mxfp4_moe_layer_workspace_bytes(4, 2, n, ff, E)
    ok = [None, P, P, P, E, n, ff, P, n, 0, P, P, 4, 2, P, n, 1, P, need]
    odd = C.c_void_p(4097)
    for i, v, rc in ((1, None, L.ERR_ARG), (2, None, L.ERR_ARG), (3, None, L.ERR_ARG), (1, C.c_void_p(4100), L.ERR_ARG), (4, 0, L.ERR_SHAPE), (5, 200, L.ERR_SHAPE), (6, 64, L.ERR_SHAPE),
                     (7, None, L.ERR_ARG), (7, odd, L.ERR_ARG), (8, n - 1, L.ERR_ARG), (9, 3, L.ERR_ARG), (10, None, L.ERR_ARG), (11, None, L.ERR_ARG), (12, -1, L.ERR_ARG), (13, 33, L.ERR_SHAPE),
                     (14, None, L.ERR_ARG), (14, odd, L.ERR_ARG), (15, n - 1, L.ERR_ARG), (16, -1, L.ERR_ARG), (17, None, L.ERR_ARG), (17, C.c_void_p(4100), L.ERR_ARG), (18, need - 1, L.ERR_WORKSPACE)):
        assert L.lib.frx_mxfp4_moe_layer(*with_(ok, i, v)) == rc, (i, v)
    assert L.lib.frx_mxfp4_moe_layer(*with_(with_(ok, 12, 0), 7, None)) == L.OK


@pytest.mark.parametrize("bad", ["short", "type", "strides", "experts"])
def test_a_packed_matrix_that_is_not_whole_is_refused(L, bad):
    import torch

    from flashrt_b200 import mxfp4
    data = torch.zeros(2 * mxfp4.packed_bytes(200, 256), dtype=torch.uint8)
    assert data.numel() == 2 * 4 * 8704
    mxfp4._whole(mxfp4.Packed(data, 2, 200, 256))
    w = {"short": (data[:-1], 2, 200, 256), "type": (data.view(torch.int8), 2, 200, 256), "strides": (data.repeat(2)[::2], 2, 200, 256), "experts": (data, 3, 200, 256)}[bad]
    with pytest.raises(L.FrxError):
        mxfp4._whole(mxfp4.Packed(*w))
    with pytest.raises(L.FrxError):
        mxfp4._columns(mxfp4.Packed(*w), 256)
    with pytest.raises(L.FrxError):
        mxfp4._columns(mxfp4.Packed(data, 2, 200, 256), 128)


def test_more_rows_than_an_expert_holds_are_refused(L):
    # an expert's blocks of 112 rows are counted in 24 bits
    most = 112 * (2 ** 24 - 1)
    assert L.lib.frx_mxfp4_matmul(None, P, P, most + 1, 128, P, 1, P, 1, 0) == L.ERR_SHAPE


def test_layer_rows_in_bfloat16_are_for_a_bfloat16_output(L):
    n, ff, E = 256, 128, 8
    need = L.lib.frx_mxfp4_moe_layer_workspace_bytes(4, 2, n, ff, E)
    ok = [None, P, P, P, E, n, ff, P, n, 0, P, P, 4, 2, P, n, 1, P, need]
    for out_dtype in (16, 18, 32, 33):              # float32 or float16 with the flag, flags that there are not
        assert L.lib.frx_mxfp4_moe_layer(*with_(ok, 16, out_dtype)) == L.ERR_ARG
    assert L.lib.frx_mxfp4_moe_layer(*with_(with_(ok, 16, 17), 18, need - 1)) == L.ERR_WORKSPACE     # taken; what is short is the workspace
