"""Sizes that no GPU holds are refused by the C entries of layer norm before the plan's products can overflow. (Without a
GPU: every call here is refused first.)"""
import ctypes

import pytest

from nablaengine_b200 import capi

INVALID = 1  # cudaErrorInvalidValue
NUL = ctypes.c_void_p(0)
AT = ctypes.c_void_p(1 << 20)  # an address that nothing reads
LONGEST = (1 << 63) - 1


def _forward(rows, cols, stride):
    return capi.load().nb_g1_layer_norm_forward(NUL, rows, cols, stride, 0, AT, 0, NUL, NUL, 1e-5, AT, AT, AT)


def _backward(rows, cols, g_stride, stride):
    return capi.load().nb_g1_layer_norm_backward(NUL, rows, cols, g_stride, stride, 0, AT, AT, AT, AT, 0, AT, AT, AT, AT,
                                                 AT)


@pytest.mark.parametrize("rows,cols", [(1 << 62, 36), (LONGEST, 1), ((1 << 40) + 1, 1), ((1 << 34) + 1, 64)])
def test_more_values_than_any_gpu_holds(rows, cols):
    assert _forward(rows, cols, 0) == INVALID and _forward(rows, cols, cols) == INVALID
    assert _backward(rows, cols, 0, 0) == INVALID and _backward(rows, cols, cols, cols) == INVALID
    assert capi.load().nb_g1_layer_norm_work_bytes(rows, cols) < 0


@pytest.mark.parametrize("rows,stride", [(1, (1 << 40) + 1), (3, LONGEST), (4, 1 << 62), (1 << 20, (1 << 20) + 1)])
def test_rows_further_apart_than_any_gpu_holds(rows, stride):
    assert _forward(rows, 36, stride) == INVALID
    assert _backward(rows, 36, stride, 36) == INVALID and _backward(rows, 36, 36, stride) == INVALID


def test_the_work_of_the_longest_calls():
    work = capi.load().nb_g1_layer_norm_work_bytes
    assert work(1 << 40, 1) > 0 and work(1 << 33, 100) > 0 and work(0, 1) == 0  # (no rows need none)
