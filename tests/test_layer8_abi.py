"""The 8-bit layer's entry points without a GPU: what they answer where there is no context, and their Python binding."""
import ctypes as C
import inspect

import numpy as np
import pytest

from intel_gaudi3_software_b200 import Calculator, abi


@pytest.fixture(scope="module")
def lib():
    return abi.load_library()


def tensor(shape, dtype):
    a = np.zeros(shape, abi.NP_DTYPE[dtype])
    return abi.make_tensor(a, dtype, list(reversed(shape)))


def test_calls_without_a_context_are_refused(lib):
    x, q, s = tensor((2, 8), abi.BF16), tensor((2, 8), abi.INT8), tensor((2,), abi.FP32)
    assert lib.mmeb200_rms_norm(None, q, s, None, x, None, None, 1e-6, abi.SCALE_ROW) < 0
    assert lib.mmeb200_rms_norm_grad(None, x, None, x, x, None, None, 1e-6, None) < 0
    assert lib.mmeb200_quantize(None, q, s, x, abi.OP_MEMCPY, abi.SCALE_ROW) < 0
    assert lib.mmeb200_scaled_gemm(None, x, q, s, q, s, None, abi.OP_ABT) < 0
    assert lib.mmeb200_rms_norm_grad_workspace(None, 4, 8) == 0


def test_the_calculator_offers_them():
    for name, needs in (("rms_norm", ["out", "x", "gamma", "eps"]), ("rms_norm_grad", ["dx", "dgamma", "dy", "x", "gamma", "eps"]),
                        ("quantize", ["out", "scale", "x"]), ("scaled_gemm", ["out", "x", "x_scale", "w", "w_scale"])):
        assert list(inspect.signature(getattr(Calculator, name)).parameters)[1:1 + len(needs)] == needs


def test_int8_tensors_are_described():
    t = tensor((3, 5), abi.INT8)
    assert t.dtype == abi.INT8 == 64 and list(t.sizes)[:2] == [5, 3] and list(t.strides)[:2] == [1, 5]
    assert C.sizeof(C.c_int8) == np.dtype(abi.NP_DTYPE[abi.INT8]).itemsize
