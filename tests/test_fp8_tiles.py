"""Which tile a call of the 8-bit float products takes, asked of the library without a launch: no GPU."""
import ctypes as C

import pytest

from quantised_bayesian_nets_amd import _lib

AT = 1 << 20      # an address that nothing reads


def linear(M, N, K, S=1, y_type=1, shared=False):
    kp = -(-K // 128) * 128
    sp = -(-kp // 512) * 4
    v = _lib.lib().qbnn_linear_f8_tile(_lib.F8_LINEAR.pack(0, 0, 0, AT, AT, 0 if shared else M * kp, 0 if shared else M * sp, AT, AT, N * kp, -(-N // 128) * sp, 0, 0, AT, AT,
                                                         M, N, K, S, 0, y_type, 0))
    return (v >> 16, v & 65535) if v > 0 else v


def experts(S, T, E, k, D, H, N, y_type=1, exact=0):
    tiles = (C.c_int32 * 2)()
    rc = _lib.lib().qbnn_experts_f8_tiles(_lib.F8_EXPERTS.pack(*[0] * 3, AT, AT, *[AT] * 3, AT, AT, 1024, 4, 0, 0, AT, AT, 1024, 4, 0, 0, AT, AT, AT, AT,
                                                             S, T, E, k, S * T, D, H, N, E, E, exact, 0, y_type), tiles)
    return [(t >> 16, t & 65535) for t in tiles] if rc == 0 else rc


def test_the_forms_of_dense_calls():
    assert linear(1, 1024, 1024) == (16, 16) and linear(20, 1024, 1024) == (32, 64) and linear(20, 1024, 1024, y_type=3) == (32, 128) and linear(9, 64, 64, y_type=3) == (16, 128)
    assert linear(33, 100, 100) == (64, 128) and linear(128, 500, 800, S=100, y_type=0) == (128, 128) and linear(8192, 8192, 8192) == (256, 256)
    assert linear(4096, 4096, 4096, y_type=0) == (128, 256)           # the exact form has no 256 x 256
    assert linear(0, 4, 4) == 0 and linear(4, 4, 0) == -1


def test_no_form_is_chosen_that_cannot_take_the_call():
    """More tiles than one axis of a grid holds, and rows past the first 4 GiB."""
    assert experts(64, 1024, 1024, 1, 64, 64, 64) == [(16, 128), (16, 64)]        # 69632 row tiles
    assert linear(2, 64, 64, S=1 << 20) == (16, 16) and linear(20, 64, 64, S=1 << 20, y_type=3) == (32, 128)
    for T in (1 << 17, 1 << 19, 1 << 21, 1 << 23):                                    # 8 GiB of hidden rows and more: still through LDS, as fewer rows are
        # gathered rows of 4 GiB and more (4096 columns from 2^20 rows on): the form for few rows, up to 2^20 tiles of it
        assert experts(1, T, 8, 4, 1024, 4096, 1024) == [(256, 256) if T << 10 < 1 << 32 else (32, 128), (256, 256)]
        assert experts(1, T, 8, 4, 4096, 1024, 1024) == [(256, 256) if T << 12 < 1 << 32 else (32, 128), (256, 256)]
    assert linear(1 << 27, 128, 8192) == (256, 256)


def test_a_call_that_fits_no_grid_is_refused_before_anything_runs():
    assert linear(1 << 30, 1, 128, y_type=0) == (128, 256)            # 2^31 threads of 2^32
    L, call = _lib.lib(), _lib.F8_LINEAR.pack(AT, 0, 0, AT, AT, 0, 0, AT, AT, 0, 0, 0, 0, AT, AT, 1 << 30, 1, 128, 4, 0, 0, 0)
    assert linear(1 << 30, 1, 128, S=4, y_type=0) == -1 and b"do not fit a grid" in L.qbnn_last_error()
    assert L.qbnn_linear_f8_mc(call, None) == -1 and b"do not fit a grid" in L.qbnn_last_error()
    assert linear(1, 64, 64, S=(1 << 31) - 1) == -1
    assert linear((1 << 31) - 1, (1 << 31) - 300, 128, S=1 << 30, shared=True) == -1 and b"do not fit a grid" in L.qbnn_last_error()      # 2^78 tiles: not lost in 64 bits
    assert linear((1 << 31) - 1, 64, 128, y_type=3) == (256, 256)
