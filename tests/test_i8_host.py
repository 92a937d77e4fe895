"""Refusals of the 8-bit integer entries that come back before any device work, and without a device the loud failure."""
import ctypes as C

import numpy as np
import pytest

from cudapp_b200 import api
from tests.conftest import HAVE_GPU

L = api.lib
V = 0x10000                                                                   # an aligned address that nothing reads: the refusals come first


def cfg(E=64, topk=4, score=0, groups=1, kept=0, rank=1, norm=1, scale=1.0):
    return api.MoeRouteConfig(E, topk, score, groups, kept, rank, norm, scale)


@pytest.mark.parametrize("bad", [cfg(E=0), cfg(E=1025), cfg(topk=0), cfg(topk=33), cfg(E=3, topk=4), cfg(score=2), cfg(groups=7), cfg(E=1024, groups=64), cfg(groups=4, kept=5), cfg(rank=3),
                                 cfg(groups=64, kept=2, rank=2), cfg(E=64, groups=16, kept=1, topk=5), cfg(scale=float("nan")), cfg(scale=float("inf")), cfg(E=8, groups=8, kept=4, rank=2, topk=2)])
def test_route_refuses(bad):
    assert L.omega_gpu_moe_route_async(bad, 1, V, 0, 0, 0, V, V, 0) == api.BAD_ARGS
    assert api.moe_route(bad, np.zeros((1, max(bad.experts, 1)), np.float32))[0] == api.BAD_ARGS
    h = C.c_void_p(5)
    assert L.omega_gpu_moe_i8_layer_create(C.c_void_p(V), C.c_void_p(V), C.byref(bad), None, C.c_uint32(1), C.byref(h)) == api.BAD_ARGS and not h.value


@pytest.mark.parametrize("args", [(0, V, 0, 0, 0, V, V), (1, 0, 0, 0, 0, V, V), (1, V, 0, 0, 0, 0, V), (1, V, 0, 0, 0, V, 0), (1, V + 2, 0, 0, 0, V, V), (1, V + 1, 1, 0, 0, V, V), (1, V, 0, 252, 0, V, V),
                                  (1, V, 0, 258, 0, V, V), (1, V, 1, 127, 0, V, V), (1, V, 0, 0, V + 2, V, V)])
def test_route_refuses_buffers(args):
    assert L.omega_gpu_moe_route_async(cfg(), *args, 0) == api.BAD_ARGS


def test_row_refusals():
    norm, quant, gate = L.omega_gpu_residual_norm_q8_async, L.omega_gpu_quant_q8_async, L.omega_gpu_swiglu_q8_async
    good = [2, 64, 1e-6, V, 0, 0, 0, 0, 0, 0, V, V, 0]
    for at, v in ((0, 0), (1, 0), (1, 24), (1, 16400), (2, -1.0), (2, float("nan")), (3, 0), (6, V), (3, V + 8), (4, V + 4), (7, V + 8), (8, V + 4), (9, V + 2), (10, 0), (10, V + 4), (11, 0), (11, V + 2)):
        assert norm(*[v if i == at else a for i, a in enumerate(good)]) == api.BAD_ARGS, (at, v)
    good = [2, 64, V, 1, 0, V, V, 0]
    for at, v in ((0, 0), (1, 0), (1, 40), (1, 16400), (2, 0), (2, V + 8), (4, 112), (4, 136), (5, 0), (5, V + 8), (6, 0), (6, V + 1)):
        assert quant(*[v if i == at else a for i, a in enumerate(good)]) == api.BAD_ARGS, (at, v)
    good = [2, 64, V, 1, V, V, 0]
    for at, v in ((0, 0), (1, 8), (1, 16400), (2, 0), (2, V + 8), (4, 0), (4, V + 8), (5, 0), (5, V + 2)):
        assert gate(*[v if i == at else a for i, a in enumerate(good)]) == api.BAD_ARGS, (at, v)
    assert api.swiglu_q8_f32(np.zeros((1, 24), np.float32))[0] == api.BAD_ARGS and api.residual_norm_q8_f32(np.zeros((1, 24), np.float32))[0] == api.BAD_ARGS


class Tensor(C.Structure):
    """the library's own record, for the checks that come before its pointers are used"""
    _fields_ = [("n", C.c_uint32), ("k", C.c_uint32), ("rest", C.c_uint8 * 1024)]


def test_upload_and_product_refusals():
    w = np.zeros((4, 32), np.int8)
    assert api.i8_upload(np.zeros((4, 24), np.int8), np.ones(4))[0] == api.BAD_ARGS and api.i8_upload(np.zeros((1, 32784), np.int8), np.ones(1))[0] == api.TOO_LARGE
    assert api.i8_upload(w, [1, np.nan, 1, 1])[0] == api.NAN_WEIGHT and "scale 1" in api.last_error()
    assert api.i8_upload(w, [1, 1, np.inf, 1])[0] == api.BAD_ARGS and "scale 2" in api.last_error()
    h = C.c_void_p(7)
    assert L.omega_gpu_i8_upload(C.c_uint32(4), C.c_uint32(32), None, None, C.byref(h)) == api.BAD_ARGS and not h.value
    assert api.i8_upload_dev(0, 32, V, V)[0] == api.BAD_ARGS and api.i8_upload_dev(4, 32, 0, V)[0] == api.BAD_ARGS and api.i8_upload_dev(4, 1 << 16, V, V)[0] == api.TOO_LARGE
    t = C.pointer(Tensor(64, 32))
    good = [t, 3, V, 0, V, V, 0, 0]
    for at, v in ((0, None), (1, 0), (2, 0), (2, V + 8), (3, 16), (3, 40), (4, 0), (4, V + 2), (5, 0), (5, V + 8), (6, V + 4)):
        assert L.omega_gpu_i8_gemm_async(*[v if i == at else a for i, a in enumerate(good)]) == api.BAD_ARGS, (at, v)
    assert L.omega_gpu_i8_gemm_async(t, (1 << 30) + 1, V, 0, V, V, 0, 0) == api.TOO_LARGE and api.i8_upload_dev((1 << 30) + 1, 16, V, V)[0] == api.TOO_LARGE
    assert L.omega_gpu_i8_gemm_grouped_async(t, 4, 16, 5, V, V, 0, 0, V, (1 << 30) + 1, V, V, 0, 0) == api.TOO_LARGE
    good = [t, 4, 16, 5, V, V, 0, 0, V, 3, V, V, 0, 0]
    for at, v in ((0, None), (1, 0), (1, 5), (2, 0), (2, 257), (3, 0), (4, 0), (4, V + 8), (5, 0), (5, V + 2), (6, V + 2), (7, V + 1), (8, 0), (8, V + 4), (9, 0), (10, 0), (11, 0), (12, V + 8)):
        assert L.omega_gpu_i8_gemm_grouped_async(*[v if i == at else a for i, a in enumerate(good)]) == api.BAD_ARGS, (at, v)


def test_too_many_rows():
    many = (1 << 30) + 1
    assert L.omega_gpu_moe_route_async(cfg(), many, V, 0, 0, 0, V, V, 0) == api.TOO_LARGE
    assert L.omega_gpu_residual_norm_q8_async(many, 64, 1e-6, V, 0, 0, 0, 0, 0, 0, V, V, 0) == api.TOO_LARGE
    assert L.omega_gpu_quant_q8_async(many, 64, V, 1, 0, V, V, 0) == api.TOO_LARGE and L.omega_gpu_swiglu_q8_async(many, 64, V, 1, V, V, 0) == api.TOO_LARGE


def test_status_of_nothing():
    assert L.omega_gpu_i8_status(None, 0) == api.BAD_ARGS and L.omega_gpu_moe_i8_layer_status(None, 0) == api.BAD_ARGS


def test_layer_refusals():
    make = lambda gu, dn, c, bias=None, most=4: api.moe_i8_layer_create(C.pointer(Tensor(*gu)), C.pointer(Tensor(*dn)), c, bias, most)[0]      # noqa: E731
    c = cfg(E=4, topk=2)
    assert make((4 * 64, 64), (4 * 64, 48), c) == api.BAD_ARGS and make((4 * 64, 64), (4 * 48, 32), c) == api.BAD_ARGS and make((250, 64), (4 * 64, 32), c) == api.BAD_ARGS
    assert make((4 * 64, 64), (4 * 64, 32), c, most=0) == api.BAD_ARGS and make((4 * 64, 64), (4 * 64, 32), c, bias=[0, np.nan, 0, 0]) == api.BAD_ARGS
    assert make((4 * 64, 64), (4 * 64, 32), c, most=1 << 31) == api.TOO_LARGE and make((4 * 64, 16640), (4 * 16640, 32), c) == api.BAD_ARGS
    for fn, n in ((L.omega_gpu_moe_i8_layer_async, 6), (L.omega_gpu_moe_i8_layer_q8_async, 7)):
        assert fn(None, *([1] + [V] * (n - 2)), 0) == api.BAD_ARGS


@pytest.mark.skipif(HAVE_GPU, reason="checks the no-device behaviour")
def test_no_device_fails_loudly():
    assert api.i8_upload(np.zeros((4, 32), np.int8), np.ones(4))[0] == api.CHIP_FAIL and "CUDA" in api.last_error()
    assert L.omega_gpu_moe_route_async(cfg(), 1, V, 0, 0, 0, V, V, 0) == api.CHIP_FAIL
    assert L.omega_gpu_swiglu_q8_async(1, 64, V, 1, V, V, 0) == api.CHIP_FAIL
    assert api.moe_route(cfg(), np.zeros((2, 64), np.float32))[0] == api.CHIP_FAIL


def test_too_many_blocks_of_a_plan():
    t, call = C.pointer(Tensor(4 * 1024, 32)), L.omega_gpu_i8_gemm_grouped_async
    assert call(t, 4, 16, 1 << 30, V, V, 0, 0, V, 3, V, V, 0, 0) == api.TOO_LARGE and "blocks of 128" in api.last_error()
    assert call(t, 4, 16, 1 << 28, V, V, 0, 0, V, 3, V, V, 0, 0) == api.TOO_LARGE
