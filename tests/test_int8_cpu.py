"""The 8-bit (W8A8) entry points' refusals: the C ABI validates before any launch, the Python entry
points before any call, and the native host path declines what it does not take.  No GPU needed."""
import ctypes

import pytest
import torch

from rocketllm_b200 import _lib, kernels

P = ctypes.c_void_p(256)       # never dereferenced: validation fails first
ODD = ctypes.c_void_p(257)
BF16 = _lib.RW4_BF16


def status(name, *args):
    return getattr(_lib.lib(), name)(*args)


@pytest.mark.parametrize("args, word", [
    ((P, 64, None, 0, 7, 1, 64, P, P, None), "dtype"),
    ((P, 64, None, 0, BF16, -1, 64, P, P, None), "rows"),
    ((P, 64, None, 0, BF16, 1, 0, P, P, None), "values"),
    ((P, 64, None, 0, BF16, 1, 131057, P, P, None), "values"),
    ((P, 64, None, 0, BF16, 1 << 40, 64, P, P, None), "rows"),
    ((P, 64, None, 0, BF16, 1 << 27, 1 << 16, P, P, None), "rows"),
    ((None, 64, None, 0, BF16, 1, 64, P, P, None), "null"),
    ((P, 64, None, 0, BF16, 1, 64, None, P, None), "null"),
    ((P, 64, None, 0, BF16, 1, 64, P, None, None), "null"),
    ((ODD, 64, None, 0, BF16, 1, 64, P, P, None), "aligned"),
    ((P, 64, ODD, 64, BF16, 1, 64, P, P, None), "aligned"),
    ((P, 64, None, 0, BF16, 1, 64, P, ODD, None), "aligned"),
    ((P, -64, None, 0, BF16, 2, 64, P, P, None), "stride"),
    ((P, 64, P, -64, BF16, 2, 64, P, P, None), "stride"),
])
def test_quantize_refuses(args, word):
    assert status("rw4_int8_quantize", *args) == _lib.RW4_EINVAL
    assert word in _lib.last_error()


@pytest.mark.parametrize("args, word", [
    ((P, 64, None, 0, P, 9, 1, 64, 1e-5, None, P, P, None), "dtype"),
    ((P, 64, None, 0, P, BF16, 1, 64, -1.0, None, P, P, None), "eps"),
    ((P, 64, None, 0, P, BF16, 1, 64, float("nan"), None, P, P, None), "eps"),
    ((P, 64, None, 0, None, BF16, 1, 64, 1e-5, None, P, P, None), "null"),
    ((P, 64, P, 64, P, BF16, 1, 64, 1e-5, None, P, P, None), "come together"),
    ((P, 64, None, 0, P, BF16, 1, 64, 1e-5, P, P, P, None), "come together"),
    ((P, 64, P, 64, ODD, BF16, 1, 64, 1e-5, P, P, P, None), "aligned"),
    ((P, 64, P, -1, P, BF16, 2, 64, 1e-5, P, P, P, None), "stride"),
])
def test_rmsnorm_refuses(args, word):
    assert status("rw4_int8_rmsnorm", *args) == _lib.RW4_EINVAL
    assert word in _lib.last_error()


@pytest.mark.parametrize("args, word", [
    ((P, P, 1, 64, P, 3, None), "dtype"),
    ((P, P, -1, 64, P, BF16, None), "rows"),
    ((P, P, 1, 0, P, BF16, None), "values"),
    ((None, P, 1, 64, P, BF16, None), "null"),
    ((P, P, 1, 64, ODD, BF16, None), "aligned"),
    ((P, ODD, 1, 64, P, BF16, None), "aligned"),
])
def test_dequantize_refuses(args, word):
    assert status("rw4_int8_dequantize", *args) == _lib.RW4_EINVAL
    assert word in _lib.last_error()


@pytest.mark.parametrize("args, word", [
    ((P, P, 1, 100, P, P, 8, None, None, P, BF16, 0, None), "multiple of 16"),
    ((P, P, 1, 0, P, P, 8, None, None, P, BF16, 0, None), "multiple of 16"),
    ((P, P, 1, 131072, P, P, 8, None, None, P, BF16, 0, None), "multiple of 16"),
    ((P, P, -1, 64, P, P, 8, None, None, P, BF16, 0, None), "M="),
    ((P, P, 1, 64, P, P, -8, None, None, P, BF16, 0, None), "N="),
    ((P, P, 1 << 30, 64, P, P, 1 << 30, None, None, P, BF16, 0, None), "too large"),
    ((P, P, 1, 64, P, P, 8, None, None, P, 5, 0, None), "out_dtype"),
    ((P, P, 1, 64, P, P, 8, None, None, P, BF16, 3, None), "path"),
    ((P, P, 1, 64, P, P, 8, None, None, P, BF16, -1, None), "path"),
    ((None, P, 1, 64, P, P, 8, None, None, P, BF16, 0, None), "null"),
    ((P, P, 1, 64, P, None, 8, None, None, P, BF16, 0, None), "null"),
    ((P, P, 1, 64, P, P, 8, None, None, None, BF16, 0, None), "null"),
    ((ctypes.c_void_p(264), P, 1, 64, P, P, 8, None, None, P, BF16, 0, None), "16-byte"),
    ((P, P, 1, 64, ctypes.c_void_p(260), P, 8, None, None, P, BF16, 0, None), "16-byte"),
    ((P, P, 1, 64, P, P, 8, ODD, None, P, BF16, 0, None), "aligned"),
    ((P, P, 1, 64, P, P, 8, None, ODD, P, BF16, 0, None), "aligned"),
    ((P, P, 1, 64, P, P, 8, None, None, ctypes.c_void_p(258), _lib.RW4_F32, 0, None), "aligned"),
])
def test_linear_refuses(args, word):
    assert status("rw4_int8_linear", *args) == _lib.RW4_EINVAL
    assert word in _lib.last_error()


def test_empty_calls_do_nothing():
    assert status("rw4_int8_quantize", None, 64, None, 0, BF16, 0, 64, None, None, None) == 0
    assert status("rw4_int8_rmsnorm", None, 64, None, 0, None, BF16, 0, 64, 1e-5, None, None, None,
                  None) == 0
    assert status("rw4_int8_dequantize", None, None, 0, 64, None, BF16, None) == 0
    assert status("rw4_int8_linear", None, None, 0, 64, None, None, 8, None, None, None, BF16, 0,
                  None) == 0
    assert status("rw4_int8_linear", None, None, 8, 64, None, None, 0, None, None, None, BF16, 0,
                  None) == 0


@pytest.mark.parametrize("native", [True, False])
def test_cpu_tensors_are_refused(native, monkeypatch):
    """No CPU path, with and without the native host path."""
    if not native:
        monkeypatch.setattr(kernels, "_native", None)
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    codes, scale = torch.zeros(2, 64, dtype=torch.int8), torch.zeros(2)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        kernels.int8_quantize(x)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        kernels.int8_quantize(x, gate=x)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        kernels.int8_rmsnorm(x, x[0], 1e-5, residual=x)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        kernels.int8_dequantize(codes, scale)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        kernels.int8_linear(codes, scale, codes, scale)


def test_native_host_path_is_built():
    """The library ships with its host fast path (built beside librw4.so)."""
    assert kernels._native is not None
    for name in ("int8_quantize", "int8_rmsnorm", "int8_dequantize", "int8_linear"):
        assert callable(getattr(kernels._native, name))


def test_native_host_path_declines_what_it_does_not_take():
    n = kernels._native
    x, codes, scale = torch.zeros(2, 64), torch.zeros(2, 64, dtype=torch.int8), torch.zeros(2)
    assert n.int8_quantize(x, None) is None
    assert n.int8_quantize(x) is None
    assert n.int8_quantize(3, None) is None
    assert n.int8_rmsnorm(x, x[0], 1e-5, None) is None
    assert n.int8_dequantize(codes, scale, torch.bfloat16) is None
    assert n.int8_dequantize(codes, scale, "bf16") is None
    assert n.int8_linear(codes, scale, codes, scale, None, None, torch.bfloat16) is None
