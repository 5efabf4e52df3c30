"""The modules of an RW8 model: what they compute beside the kernels they call."""
from types import SimpleNamespace

import pytest
import torch

from rocketllm_b200.quant import Int8Rows, RW8Linear, rw8_layers
from test_int8_gpu import BF, F16, F32, check_linear, check_rows, operands, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F16])
def test_wider_norm_weights_are_not_rounded(cuda, dtype):
    """A stream in 16 bits beside norm weights in 32: they are used as they are."""
    x, r, w = randn(1, 5, 512, dtype=dtype), randn(2, 5, 512, dtype=dtype), randn(3, 512, dtype=F32)
    norm = SimpleNamespace(weight=w, variance_epsilon=1e-5)

    def normed(h):
        h = h.double()
        return h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-5) * w.double()

    check_rows(*rw8_layers._norm(norm, x), normed(x), e=2.0 ** -19)
    codes, scale, h = rw8_layers._norm(norm, x, residual=r)
    assert h.dtype == dtype and torch.equal(h, (x.double() + r.double()).to(dtype))
    check_rows(codes, scale, normed(h), e=2.0 ** -19)


@pytest.mark.parametrize("dtype", [BF, F16])
def test_wider_biases_are_not_rounded(cuda, dtype):
    """Rows in 16 bits beside a bias in 32: one rounding, of the whole sum."""
    q, qs, wq, wsc, _, res = operands(4, 5, 512, 320, dtype, residual=True)
    m = RW8Linear(512, 320, bias=True, device=cuda, dtype=F32)
    m.weight.data, m.weight_scale.data = wq, wsc[:, None]
    m.bias.data = randn(5, 320, dtype=F32) * 100
    y = m(Int8Rows(q, qs, dtype))
    assert y.dtype == dtype
    check_linear(y, q, qs, wq, wsc, m.bias)
    y = m(Int8Rows(q, qs, dtype), residual=res)
    assert y.dtype == dtype
    check_linear(y, q, qs, wq, wsc, m.bias, res)
