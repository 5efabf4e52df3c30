"""What the 8-bit operators promise at the ends of their ranges and at ties, against formulas.

Tolerances, derived (u = 2^-24, half a step of fp32; the row checks are those of test_int8_gpu.py):

* codes of a tensor are rint(y * (127 / a)) with both operations rounded to fp32: the same bits as
  the same two operations of IEEE arithmetic anywhere, and the scale those of a / 127.
* silu(g) * v for g down to -120: a = |g| log2(e) / 2 <= 86.6 is rounded (half a step: 2^-18; its
  constant is off by 2^-26.2: 2^-19.7 here), which moves h = 2^-a by ln 2 of that and h^2 by twice as
  much: 7 * 2^-20; the approximate exponential is off by 2^-22, twice, the reciprocal by 2^-23, five
  roundings by u each.  e <= 8.1 * 2^-20 < 2^-16.
* a product of scales and a sum, as in test_int8_gpu.py, and half a step of fp32's subnormal numbers
  (2^-150) more where it is one.
"""
import numpy as np
import pytest
import torch

from rocketllm_b200 import kernels
from test_int8_gpu import BF, F16, F32, check_rows, operands, randn

pytestmark = pytest.mark.gpu


# a warp, a CTA or a cluster a row, one and several vectors a thread; the rings, with whole rows, any
# rows, and rows in pieces over a cluster
SHAPES = [(1, 8), (9, 509), (3, 1000), (2, 4096), (20, 14336), (2, 16385), (2, 53248), (2500, 4096),
          (640, 14336), (310, 28672), (640, 14335), (170, 33001)]


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("m,k", SHAPES)
def test_codes_are_the_rounded_product(cuda, m, k, dtype):
    """16-bit rows hold many values at an exact half of a code, each row's factor 127 / a rounded:
    the product is rounded to fp32 before it is rounded to a code."""
    x = randn(m + k, m, k, dtype=dtype)
    x[0, 0], x[0, k - 1] = 2.03125, 1.015625      # 63.5 of 127: to 64
    x[0].clamp_(-2.03125, 2.03125)
    codes, scale = kernels.int8_quantize(x)
    y = x.float().cpu().numpy()
    a = np.abs(y).max(1, keepdims=True)
    want = np.rint(y * (np.float32(127) / a))
    assert np.array_equal(codes.cpu().numpy(), want)
    assert np.array_equal(scale.cpu().numpy(), (a / np.float32(127))[:, 0])
    assert codes[0, k - 1].item() == 64


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m,k", SHAPES)
def test_gates_far_below_zero(cuda, m, k, dtype):
    """Rows whose gates all lie where exp(g) is near the end of fp32 or past it, beside ordinary ones:
    their products are far above the smallest scale."""
    g = torch.Generator(device="cuda").manual_seed(m + k)
    gate = -20 - 67 * torch.rand(m, k, generator=g, device="cuda")
    gate[::3] = -87.5 - torch.rand(gate[::3].shape, generator=g, device="cuda")
    gate[1::3] = torch.randn(gate[1::3].shape, generator=g, device="cuda") * 30
    up = randn(k, m, k, dtype=F32) * 1e12
    gate[0], up[0] = -88, 1e6
    if m > 1:
        gate[m - 1] = -92 - 28 * torch.rand(k, generator=g, device="cuda")
        up[m - 1] = 1e36
    gate, up = gate.to(dtype), up.to(dtype)
    codes, scale = kernels.int8_quantize(up, gate=gate)
    assert (codes[0] == -127).all()
    gd = gate.double()
    check_rows(codes, scale, gd * torch.sigmoid(gd) * up.double(), e=2.0 ** -16)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("eps", [0.0, 1e-5])
@pytest.mark.parametrize("m,k", SHAPES)
def test_norms_whose_squares_leave_fp32(cuda, m, k, eps, residual, dtype):
    """Finite rows whose squares, or whose products with the weight, are above fp32's largest number
    or below its smallest, among ordinary ones, a NaN and an infinite one."""
    sizes = torch.tensor([1e25, 1.0, 1e37, 1e-15, 1e18, 1e-22, 1e-30, 1e-37], device="cuda")
    x = (randn(m + k, m, k, dtype=F32) * sizes[torch.arange(m, device="cuda") % 8, None]).to(dtype)
    odd = torch.zeros(m, dtype=torch.bool, device="cuda")
    if m > 8:
        x[5, k // 2], x[6, k - 1] = float("nan"), float("inf")
        odd[5] = odd[6] = True
    for big in (1.0, 1e20):
        w = (randn(k, k, dtype=F32) * big).to(dtype)
        h = x
        if residual:
            r = x / 2
            want = (x.double() + r.double()).to(dtype)
            codes, scale, h = kernels.int8_rmsnorm(x, w, eps, residual=r, hidden=r)
            assert torch.equal(h[~odd], want[~odd]) and h is r
        else:
            codes, scale = kernels.int8_rmsnorm(x, w, eps)
        assert scale[odd].isnan().all() and not codes[odd].any()
        hd = h[~odd].double()
        y = hd * torch.rsqrt(hd.square().mean(-1, keepdim=True) + eps) * w.double()
        check_rows(codes[~odd], scale[~odd], y, e=2.0 ** -19)
    # the largest finite rows, and a weight that is not finite
    x[:] = torch.finfo(dtype).min
    w = torch.ones(k, dtype=dtype, device="cuda")
    codes, scale = kernels.int8_rmsnorm(x, w, eps)
    assert (codes == -127).all() and ((scale * 127 - 1).abs() < 2.0 ** -19).all()
    w[k // 2] = float("inf")
    codes, scale = kernels.int8_rmsnorm(x, w, eps)
    assert scale.isnan().all() and not codes.any()
    torch.cuda.synchronize()
    assert kernels.device_status() == 0


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("m,k,n", [(1, 1024, 300), (40, 4096, 512), (300, 512, 264)])
def test_scales_whose_product_is_small(cuda, m, k, n, path, dtype):
    """Scales whose product lies below 2^-126 beside results that do not, and scales far apart: no
    bits are lost on the way."""
    q, qs, w, ws, b, r = operands(m + k, m, k, n)
    f = torch.finfo(dtype)

    def check(y, q, ss, tt):
        ref = q.double() @ w.double().t() * ss.double()[:, None] * tt.double()
        err32 = 2.0 ** -22 * ref.abs() + 2.0 ** -150
        bound = err32 + f.eps / 2 * (ref.abs() + err32).clamp_min(f.smallest_normal)
        assert ((y.double() - ref).abs() <= bound).all()

    for s, t in ((2.0 ** -100, 2.0 ** -40), (2.0 ** -40, 2.0 ** -100), (2.0 ** -70, 2.0 ** -70),
                 (2.0 ** 110, 2.0 ** -120), (2.0 ** -120, 2.0 ** 90)):
        for both in (False, True):      # every token, or every other
            ss = qs.clone()
            ss[::1 if both else 2] *= s
            tt = ws * k * t
            y = kernels.int8_linear(q, ss, w, tt, dtype=dtype, path=path)
            check(y, q, ss, tt)
    # (zero, huge and NaN scales keep to themselves)
    ss, tt = qs.clone(), ws * 2.0 ** -60
    ss[0], tt[n // 2] = 2.0 ** 120, 0
    ss[m // 2] = 0
    ss[m - 1] = float("nan")
    y = kernels.int8_linear(q, ss, w, tt, dtype=dtype, path=path)
    assert y[m - 1].isnan().all()
    if m > 1:
        check(y[:m - 1], q[:m - 1], ss[:m - 1], tt)
        assert not y[m // 2].any() and not y[:m - 1, n // 2].any()


def test_outputs_beside_their_operands_are_taken(cuda):
    """Operands side by side in one buffer, outputs between strided rows, and in place: none of them
    overlaps.  Outputs that do are refused through the Python calls, too."""
    m, k = 5, 128
    buf = torch.zeros(1 << 16, dtype=BF, device="cuda")
    x = buf[:m * k].view(m, k)
    x.copy_(randn(1, m, k))
    want = kernels.int8_quantize(x.clone())
    after = buf[m * k:].view(torch.int8)
    codes = after[:m * k].view(m, k)
    scale = after[m * k:m * k + 4 * m].view(F32)
    assert all(torch.equal(a, b) for a, b in zip(kernels.int8_quantize(x, out=(codes, scale)), want))
    # rows far apart, the outputs in the gap between the first two
    apart = buf.as_strided((m, k), (4096, 1), 8192)
    apart.copy_(x)
    gap = buf[8192 + k:8192 + 4096].view(torch.int8)
    out = (gap[:m * k].view(m, k), gap[m * k:m * k + 4 * m].view(F32))
    assert all(torch.equal(a, b) for a, b in zip(kernels.int8_quantize(apart, out=out), want))
    w, r = randn(2, k), randn(3, m, k)
    want = kernels.int8_rmsnorm(x.clone(), w, 1e-5, residual=r)
    xx = x.clone()
    assert all(torch.equal(a, b) for a, b in
               zip(kernels.int8_rmsnorm(xx, w, 1e-5, residual=r, hidden=xx), want))
    both = x.clone()      # x, residual and hidden in one
    want = kernels.int8_rmsnorm(x.clone(), w, 1e-5, residual=x.clone())
    assert all(torch.equal(a, b) for a, b in
               zip(kernels.int8_rmsnorm(both, w, 1e-5, residual=both, hidden=both), want))
    flat = torch.zeros(m * k + 1, dtype=BF, device="cuda")
    for call in (lambda: kernels.int8_rmsnorm(flat[1:].view(m, k), w, 1e-5, residual=r,
                                              hidden=flat[:-1].view(m, k)),
                 lambda: kernels.int8_rmsnorm(flat[:k].expand(m, k), w, 1e-5, residual=r,
                                              hidden=flat[:-1].view(m, k)),
                 lambda: kernels.int8_quantize(x, out=(x.view(torch.int8).flatten()[:m * k].view(m, k),
                                                  scale))):
        with pytest.raises(RuntimeError, match="overlap"):
            call()
    q, s, wq, ws, _, res = operands(4, m, k, 96, residual=True)
    flat = torch.zeros(m * 96 + 1, dtype=BF, device="cuda")
    with pytest.raises(RuntimeError, match="overlap"):
        kernels.int8_linear(q, s, wq, ws, residual=flat[1:].view(m, 96), out=flat[:-1].view(m, 96))


@pytest.mark.parametrize("path,m", [(1, 4), (1, 100), (2, 64), (2, 600)])
def test_products_read_what_the_launches_before_them_wrote(cuda, path, m):
    """Weights and activations quantized into the same buffers again and again, their codes other
    ones each time, and multiplied at once: launches overlap their prologues, and each product
    gives what it gives alone."""
    n, k = 2048, 4096
    weights = [randn(s, n, k) for s in range(4)]
    xs = [randn(10 + s, m, k) for s in range(3)]
    w = (torch.empty(n, k, dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda"))
    q = (torch.empty(m, k, dtype=torch.int8, device="cuda"), torch.empty(m, device="cuda"))
    res = randn(20, m, n)

    def product(i, out=None):
        kernels.int8_quantize(xs[i % 3], out=q)
        kernels.int8_quantize(weights[i % 4], out=w)
        return kernels.int8_linear(*q, *w, residual=res, path=path, out=out)

    want = []
    for i in range(12):
        want.append(product(i).clone())
        torch.cuda.synchronize()
    assert not any(torch.equal(want[i], want[j]) for i in range(12) for j in range(i))
    got = [torch.empty_like(res) for _ in range(48)]
    for i in range(48):        # the weights last
        product(i, got[i])
    for i in range(48):
        assert torch.equal(got[i], want[i % 12])
    for i in range(48):        # the activations last
        kernels.int8_quantize(weights[i % 4], out=w)
        kernels.int8_quantize(xs[i % 3], out=q)
        kernels.int8_linear(*q, *w, residual=res, path=path, out=got[i])
    for i in range(48):
        assert torch.equal(got[i], want[i % 12])
    # in a graph, whose launches follow one another without the host
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for i in range(48):
            product(i, got[i])
    for g in got:
        g.zero_()
    graph.replay()
    for i in range(48):
        assert torch.equal(got[i], want[i % 12])


def test_native_path_takes_rows_of_any_dimension(cuda):
    """Views of three and four dimensions with one stride between their rows are not declined, others
    are, and both give what compact copies give."""
    gu = randn(1, 2, 3, 4, 512)
    w = randn(2, 256)
    one = [gu[..., :256], gu[..., 256:], gu[:1, :, :, :256], gu[:, :, :, 8:264], gu[:, :1, :1, :256],
           gu[:1, :1, :1, 5:261], gu[:1, :1, ::2, :256], gu[:0, :, :, :256], gu[:, :0, :, :256],
           gu[:1, :1, :1, :256].expand(2, 3, 4, 256)]
    many = [gu[:, :, ::3, :256], gu[:, :2, :, :256], gu.transpose(0, 1)[..., :256],
            gu[:, :, :1, :256].expand(2, 3, 4, 256)]
    for i, v in enumerate(one + many):
        c = v.clone(memory_format=torch.contiguous_format)
        calls = [(kernels._native.int8_quantize, (v, v), kernels.int8_quantize, (c, c)),
                 (kernels._native.int8_rmsnorm, (v, w, 1e-5, v), kernels.int8_rmsnorm,
                  (c, w, 1e-5, c))]
        for native, args, plain, copies in calls:
            got = native(*args)
            assert (got is not None) == (i < len(one))
            want = plain(*copies)
            for g in (got, plain(*args)):
                if g is not None:
                    assert all(a.shape == b.shape and torch.equal(a, b) for a, b in zip(g, want))
