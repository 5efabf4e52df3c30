"""Outputs of the 8-bit entry points that overlap another operand are refused before any launch.  No
GPU needed: only calls that must be refused are made, and no pointer is read."""
import ctypes

import pytest

from rocketllm_b200 import _lib

BF16, F32 = _lib.RW4_BF16, _lib.RW4_F32
M, K = 4, 64
BASE = 1 << 20


def at(offset):
    return ctypes.c_void_p(BASE + offset)


FAR = [at(1 << (24 + i)) for i in range(6)]   # operands out of the way


def refused(name, *args):
    assert getattr(_lib.lib(), name)(*args, None) == _lib.RW4_EINVAL
    assert "overlap" in _lib.last_error()


@pytest.mark.parametrize("codes, scale", [
    (at(0), FAR[0]),                     # x itself
    (at(M * K * 2 - 1), FAR[0]),         # its last byte
    (at(-M * K + 1), FAR[0]),            # its first byte
    (FAR[0], at(8)), (FAR[0], at(-4 * M + 4)), (FAR[0], at(M * K * 2 - 4)),
    (FAR[0], ctypes.c_void_p(FAR[0].value + M * K - 4)),         # each other
])
@pytest.mark.parametrize("gated", [False, True])
def test_codes_over_the_rows_they_are_taken_from(codes, scale, gated):
    if gated:
        refused("rw4_int8_quantize", FAR[5], K, at(0), K, BF16, M, K, codes, scale)
    else:
        refused("rw4_int8_quantize", at(0), K, None, 0, BF16, M, K, codes, scale)
    refused("rw4_int8_rmsnorm", at(0), K, None, 0, FAR[4], BF16, M, K, 1e-5, None, codes, scale)
    refused("rw4_int8_rmsnorm", FAR[3], K, at(0), K, FAR[4], BF16, M, K, 1e-5, FAR[2], codes, scale)
    refused("rw4_int8_rmsnorm", FAR[3], K, FAR[5], K, FAR[4], BF16, M, K, 1e-5, at(0), codes, scale)


@pytest.mark.parametrize("row", range(M))
@pytest.mark.parametrize("stride", [K, 3 * K, 1000])
def test_codes_over_one_of_strided_rows(row, stride):
    """Any one of the rows, at its first and its last byte."""
    for offset in (row * stride * 2 - M * K + 1, (row * stride + K) * 2 - 1):
        refused("rw4_int8_quantize", at(0), stride, None, 0, BF16, M, K, at(offset), FAR[0])
    refused("rw4_int8_quantize", at(0), 0, None, 0, BF16, M, K, at(K * 2 - 1), FAR[0])


@pytest.mark.parametrize("offset", [2, -2, K * 2, (M * K - 1) * 2, -(M * K - 1) * 2])
def test_hidden_beside_an_input(offset):
    """The hidden rows may be x or the residual, not rows a little further on."""
    for x, r in ((at(0), FAR[0]), (FAR[0], at(0))):
        refused("rw4_int8_rmsnorm", x, K, r, K, FAR[1], BF16, M, K, 1e-5, at(offset), FAR[2],
                FAR[3])


def test_hidden_over_other_operands():
    # the same address, other rows: broadcast, apart
    for stride in (0, K - 1, K + 1, 2 * K):
        refused("rw4_int8_rmsnorm", at(0), stride, FAR[0], K, FAR[1], BF16, M, K, 1e-5, at(0),
                FAR[2], FAR[3])
        refused("rw4_int8_rmsnorm", FAR[0], K, at(0), stride, FAR[1], BF16, M, K, 1e-5, at(0),
                FAR[2], FAR[3])
    # the weight
    refused("rw4_int8_rmsnorm", FAR[4], K, FAR[0], K, at(0), BF16, M, K, 1e-5, at(0), FAR[2],
            FAR[3])
    # codes over the weight
    refused("rw4_int8_rmsnorm", FAR[4], K, None, 0, at(0), BF16, M, K, 1e-5, None, at(0), FAR[3])


@pytest.mark.parametrize("out, dtype", [(at(0), BF16), (at(M * K - 4), F32),
                                        (at(-M * K * 2 + 2), BF16)])
def test_values_over_their_codes(out, dtype):
    refused("rw4_int8_dequantize", at(0), FAR[0], M, K, out, dtype)
    refused("rw4_int8_dequantize", FAR[0], at(0), M, K, at(4), dtype)


N = 96


@pytest.mark.parametrize("which", ["codes", "scale", "weight", "weight_scale", "bias", "residual"])
@pytest.mark.parametrize("end", [False, True])
def test_a_product_over_its_operands(which, end):
    sizes = {"codes": M * K, "scale": 4 * M, "weight": N * K, "weight_scale": 4 * N, "bias": 2 * N,
             "residual": M * N * 2}
    ops = dict(zip(sizes, FAR))
    ops[which] = at(0)
    out = at(sizes[which] - 2) if end else at(-M * N * 2 + 2)
    refused("rw4_int8_linear", ops["codes"], ops["scale"], M, K, ops["weight"],
            ops["weight_scale"], N, ops["bias"], ops["residual"], out, BF16, 0)
