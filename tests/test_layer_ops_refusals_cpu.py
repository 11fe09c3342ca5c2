"""Refusals of the layer operators' wrappers that need no GPU."""
import ctypes as C

import pytest
import torch

import a11spec
from a11spec import _lib
from a11spec._lib import lib


@pytest.mark.parametrize("x", [None, [1.0], 3])
def test_check_status_refuses_as_the_plain_call(x):
    """The status word's workspace is made only for tensors: the refusal stays an A11Error."""
    t = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(a11spec.A11Error, match="tensor"):
        a11spec.linear(x, t, check_status=True)
    with pytest.raises(a11spec.A11Error, match="tensor"):
        a11spec.chunk_attention(x, t, t, t, t, check_status=True)


@pytest.mark.parametrize("a,words", [((0, 64, 64, 64), "dtype"), ((1, 0, 64, 64), "sizes"), ((1, 64, 0, 64), "sizes"),
                                     ((2, 64, 64, 2 ** 30 + 8), "sizes")])
def test_linear_plan_refuses(a, words):
    tile, split = C.c_int32(), C.c_int32()
    assert lib.a11s_linear_plan(*a, 0, C.byref(tile), C.byref(split)) == _lib.EINVAL
    assert words in lib.a11s_last_error().decode()
    assert lib.a11s_linear_plan(1, 64, 64, 64, 0, None, C.byref(split)) == _lib.EINVAL


def test_linear_plan_without_a_device():
    """The 148 SMs assumed without a device: few rows stream the weights, large sizes take CTA pairs."""
    tile, split = C.c_int32(), C.c_int32()
    for rows, want in ((1, 0), (32, 0), (64, None), (8192, 256)):
        assert lib.a11s_linear_plan(_lib.BF16, rows, 2048, 8192, 0, C.byref(tile), C.byref(split)) == _lib.OK
        assert tile.value == want if want is not None else tile.value in (32, 64, 128)
