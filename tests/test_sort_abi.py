"""What the entry points of the sort refuse before they touch CUDA, and what they answer without work to do. CPU only."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def L():
    from flashrt_b200 import lib
    return lib


P = C.c_void_p(4096)        # an address that no refused call reads


def test_workspace_sizes(L):
    f = L.lib.frx_moe_sort_workspace_bytes
    assert f(1, 10, 512) == 256 and f(0, 1, 1) == 256
    assert f(16384, 10, 512) >= 256 + 161 * 512 * 4
    for bad in ((-1, 1, 1), (1, 0, 1), (1, 33, 64), (1, 1, 0), (1, 1, 4097), (2 ** 30, 2, 8)):
        assert f(*bad) == 0


def test_sort_refusals(L):
    f = L.lib.frx_moe_sort
    assert f(None, P, -1, 2, 8, P, P, P, P, 4096) == L.ERR_ARG
    assert f(None, P, 4, 33, 8, P, P, P, P, 4096) == L.ERR_SHAPE
    assert f(None, P, 4, 2, 4097, P, P, P, P, 4096) == L.ERR_SHAPE
    assert f(None, P, 4, 2, 8, P, P, P, P, 255) == L.ERR_WORKSPACE
    assert f(None, P, 4, 2, 8, P, P, P, C.c_void_p(4100), 4096) == L.ERR_ARG
    for i in (1, 5, 6, 7, 8):
        args = [None, P, 513, 2, 8, P, P, P, P, 4096]
        args[i] = None
        assert f(*args) == L.ERR_ARG


def test_row_refusals(L):
    lib = L.lib
    ok = [None, P, 64, 1, P, 4, 2, 64, P, 64, 8]
    for i, v, rc in ((1, None, L.ERR_ARG), (2, 63, L.ERR_ARG), (3, 3, L.ERR_ARG), (3, -1, L.ERR_ARG), (4, None, L.ERR_ARG), (5, -1, L.ERR_ARG), (6, 0, L.ERR_SHAPE),
                     (6, 33, L.ERR_SHAPE), (7, -1, L.ERR_ARG), (8, None, L.ERR_ARG), (9, 63, L.ERR_ARG), (1, C.c_void_p(4097), L.ERR_ARG)):
        a = list(ok)
        a[i] = v
        assert lib.frx_moe_sort_rows(*a) == rc, (i, v)
    assert lib.frx_moe_sort_rows(None, P, 64, 1, P, 2 ** 27, 32, 64, P, 64, 8) == L.ERR_SHAPE
    # nothing to do: no launch
    assert lib.frx_moe_sort_rows(None, None, 64, 1, None, 0, 2, 64, None, 64, 8) == L.OK
    assert lib.frx_moe_sort_rows(None, None, 0, 1, None, 4, 2, 0, None, 0, 8) == L.OK
    back = [None, P, 64, 8, 0, P, 4, 2, 64, P, 64]
    for i, v, rc in ((1, None, L.ERR_ARG), (2, 63, L.ERR_ARG), (4, 9, L.ERR_ARG), (5, None, L.ERR_ARG), (7, 33, L.ERR_SHAPE), (9, None, L.ERR_ARG), (10, 63, L.ERR_ARG)):
        a = list(back)
        a[i] = v
        assert lib.frx_moe_sort_rows_backward(*a) == rc, (i, v)
    un = [None, P, 64, 8, 2, P, P, 4, 2, 64, P, 64]
    for i, v, rc in ((1, None, L.ERR_ARG), (4, 5, L.ERR_ARG), (5, None, L.ERR_ARG), (6, None, L.ERR_ARG), (8, 0, L.ERR_SHAPE), (10, C.c_void_p(4097), L.ERR_ARG), (11, 1, L.ERR_ARG)):
        a = list(un)
        a[i] = v
        assert lib.frx_moe_unsort_rows(*a) == rc, (i, v)
    ub = [None, P, 64, P, 64, 8, 0, P, P, 4, 2, 64, P, 64, P]
    for i, v, rc in ((1, None, L.ERR_ARG), (2, 1, L.ERR_ARG), (3, None, L.ERR_ARG), (4, 1, L.ERR_ARG), (6, 7, L.ERR_ARG), (7, None, L.ERR_ARG), (8, None, L.ERR_ARG),
                     (10, 40, L.ERR_SHAPE), (12, None, L.ERR_ARG), (13, 1, L.ERR_ARG), (14, None, L.ERR_ARG)):
        a = list(ub)
        a[i] = v
        assert lib.frx_moe_unsort_rows_backward(*a) == rc, (i, v)


def test_route_backward_refusals(L):
    f = L.lib.frx_route_topk_backward
    assert f(None, P, P, P, -1, 8, 2, P) == L.ERR_ARG
    for E, k in ((0, 1), (1025, 1), (8, 0), (8, 9), (64, 33)):
        assert f(None, P, P, P, 4, E, k, P) == L.ERR_SHAPE
    assert f(None, None, None, None, 0, 8, 2, None) == L.OK
    for i in (1, 2, 3, 7):
        a = [None, P, P, P, 4, 8, 2, P]
        a[i] = None
        assert f(*a) == L.ERR_ARG
