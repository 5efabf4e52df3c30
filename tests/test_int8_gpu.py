"""The 8-bit (W8A8) operators against their formulas in 64 bits.

Tolerances, derived (u = 2^-24, half a step of fp32):

* a quantized row y with a = max |y|: the kernel rounds 127 / a and the product y * (127 / a), so
  what it rounds to a code is off by at most 127 * 2 u (1 + u); a code is therefore within
  1/2 + 127 * 2^-22 of y * 127 / a, and the scale within u of a / 127.  Where y itself is
  off by a relative e (the product silu(gate) * up, the normed row), y and a both move: 2 e more.
* silu(gate) * up for |gate| <= 16: exp's argument is rounded (16 u relative in exp) and the
  approximate exponential and division are within 2 steps each (4 u), the sum and the product round
  once: e <= (16 + 4 + 4 + 2) u < 2^-19.
* the normed row: a thread sums at most 32 squares, the tree joins 5 + 4 + 7 sums: 48 u on the mean,
  half of it on its root, rsqrt 2 steps, three roundings: e <= (24 + 4 + 3) u < 2^-19.
* a product p = s_m t_n S (S the exact integer sum), bias b, residual r: S to fp32, s_m t_n, the
  fused multiply-add and the last sum round once each: 2^-22 (|p| + |b| + |r|) covers the four;
  then one rounding to the output's type, eps / 2 of the value (below the smallest normal number:
  of that number).
"""
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from rocketllm_b200 import kernels

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
TINY = 2.0 ** -119


def check_rows(codes, scale, y, e=0.0):
    """codes, scale of finite rows y (64 bits), each off by at most a relative e."""
    y = y.reshape(-1, y.shape[-1]).double()
    codes, scale = codes.reshape(y.shape).double(), scale.reshape(-1).double()
    a = y.abs().amax(-1)
    live = a >= TINY
    v = torch.where(live[:, None], y * 127 / a.clamp_min(TINY)[:, None], torch.zeros_like(y))
    assert ((codes - v).abs().max() <= 0.5 + 127 * (2.0 ** -22 + 2 * e)).item()
    want = torch.where(live, a / 127, torch.zeros_like(a))
    assert ((scale - want).abs() <= (2.0 ** -24 + e) * want).all()
    # the row's largest value always has code 127 or -127
    assert torch.equal(codes.abs().amax(-1), torch.where(live, 127.0, 0.0).to(codes))


def randn(seed, *shape, dtype=BF):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


ROWS = [(1, 1), (1, 8), (3, 7), (5, 65), (300, 33), (2, 4095), (4, 4096), (3, 4104), (3, 5632),
        (2, 8200), (2, 14336), (2, 16384), (2, 16385), (3, 32776), (1, 53248), (2, 65543),
        (1, 131049), (1, 131056), (65, 250), (65, 264), (9, 509), (9, 1017), (7, 1018), (7, 1023)]


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("m,k", ROWS)
def test_quantize_and_back(cuda, m, k, dtype):
    x = randn(m + k, m, k, dtype=dtype)
    codes, scale = kernels.int8_quantize(x)
    assert codes.shape == x.shape and scale.shape == (m,)
    check_rows(codes, scale, x)
    for out in (BF, F16, F32):
        back = kernels.int8_dequantize(codes, scale, dtype=out)
        assert torch.equal(back, (codes.float() * scale[:, None]).to(out))


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("m,k", ROWS)
def test_quantize_gated(cuda, m, k, dtype):
    gu = randn(m * 3 + k, m, 2 * k, dtype=dtype)
    gate, up = (gu[:, :k] * 3).clamp(-16, 16), gu[:, k:]
    codes, scale = kernels.int8_quantize(up, gate=gate)
    g = gate.double()
    check_rows(codes, scale, g * torch.sigmoid(g) * up.double(), e=2.0 ** -19)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("m,k", ROWS)
def test_rmsnorm(cuda, m, k, residual, dtype):
    x, w = randn(m + 7 * k, m, k, dtype=dtype), randn(k, k, dtype=dtype)
    h = x
    if residual:
        r = randn(m + 5 * k, m, k, dtype=dtype) * 4
        codes, scale, h = kernels.int8_rmsnorm(x, w, 1e-5, residual=r)
        assert torch.equal(h, (x.double() + r.double()).to(dtype))
    else:
        codes, scale = kernels.int8_rmsnorm(x, w, 1e-5)
    hd = h.double()
    y = hd * torch.rsqrt(hd.square().mean(-1, keepdim=True) + 1e-5) * w.double()
    check_rows(codes, scale, y, e=2.0 ** -19)


# enough rows for every multiprocessor to take several in turn: whole 16-byte rows, odd ones, rows
# in pieces over a cluster
MANY = [(2500, 4096), (5100, 1032), (640, 14336), (310, 28672), (5100, 1037), (1900, 4099),
        (640, 14335), (310, 20001), (170, 33001), (90, 65539), (90, 131056), (1900, 4100)]


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("m,k", MANY)
def test_many_rows(cuda, m, k, dtype):
    """Each operator over many rows, some of them zero, NaN or infinite, the first and last among
    the ordinary ones; the residual stream in place."""
    x = randn(m + k, m, k, dtype=dtype)
    x[3], x[m // 2, k - 1], x[m - 2, 0] = 0, float("nan"), float("inf")
    odd = torch.zeros(m, dtype=torch.bool, device="cuda")
    odd[m // 2] = odd[m - 2] = True

    def check(codes, scale, y, e):
        assert scale[odd].isnan().all() and codes[odd].abs().max() == 0
        check_rows(codes[~odd], scale[~odd], y[~odd], e)

    check(*kernels.int8_quantize(x), x.double(), 0.0)
    gu = randn(m + k + 1, m, 2 * k, dtype=dtype)
    gate = gu[:, :k].double()
    codes, scale = kernels.int8_quantize(gu[:, k:], gate=gu[:, :k])
    check_rows(codes, scale, gate * torch.sigmoid(gate) * gu[:, k:].double(), 2.0 ** -19)
    w = randn(k, k, dtype=dtype)
    hd = x.double()
    y = hd * torch.rsqrt(hd.square().mean(-1, keepdim=True) + 1e-5) * w.double()
    check(*kernels.int8_rmsnorm(x, w, 1e-5), y, 2.0 ** -19)
    r = gu[:, :k].contiguous()
    h = (x.double() + r.double()).to(dtype)
    codes, scale, got = kernels.int8_rmsnorm(x, w, 1e-5, residual=r, hidden=r)
    assert got is r and torch.equal(got[~odd], h[~odd])
    hd = h.double()
    y = hd * torch.rsqrt(hd.square().mean(-1, keepdim=True) + 1e-5) * w.double()
    check(codes, scale, y, 2.0 ** -19)
    torch.cuda.synchronize()
    assert kernels.device_status() == 0


@pytest.mark.parametrize("m,k,ox,os,oc", [(1900, 4096, 1, 0, 0), (1900, 4096, 0, 3, 0),
                                          (1900, 4096, 0, 0, 5), (1900, 4099, 2, 7, 1),
                                          (90, 40000, 3, 5, 7)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_many_rows_of_every_alignment(cuda, m, k, ox, os, oc, dtype):
    """Strided inputs that start anywhere, codes and hidden rows that start anywhere; the bytes
    around the outputs stay as they were."""
    x = randn(1, m, k + 11, dtype=dtype)[:, ox:ox + k]
    second = randn(2, m, k + 8, dtype=dtype)[:, os:os + k]
    w = randn(3, k + 7, dtype=dtype)[oc:oc + k]
    flat = torch.full((m * k + 64,), 77, dtype=torch.int8, device="cuda")
    codes = flat[16 + oc:16 + oc + m * k].view(m, k)
    hflat = torch.full((m * k + 64,), 77, dtype=dtype, device="cuda")
    hidden = hflat[16 + os:16 + os + m * k].view(m, k)
    out = (codes, torch.empty(m, device="cuda"))
    kernels.int8_quantize(x, out=out)
    check_rows(*out, x)
    kernels.int8_quantize(x, gate=second, out=out)
    g = second.double()
    check_rows(*out, g * torch.sigmoid(g) * x.double(), e=2.0 ** -19)
    kernels.int8_rmsnorm(x, w, 1e-5, residual=second, out=out, hidden=hidden)
    assert torch.equal(hidden, (x.double() + second.double()).to(dtype))
    hd = hidden.double()
    check_rows(*out, hd * torch.rsqrt(hd.square().mean(-1, keepdim=True) + 1e-5) * w.double(),
               e=2.0 ** -19)
    for f, o in ((flat, oc), (hflat, os)):
        assert (f[:16 + o] == 77).all() and (f[16 + o + m * k:] == 77).all()
    torch.cuda.synchronize()
    assert kernels.device_status() == 0


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("stride", [0, 1, 8])
def test_many_overlapping_rows(cuda, stride, dtype):
    """Broadcast rows and rows a few values apart, from an unaligned start, enough of them for every
    path of the row kernels."""
    for m, k in ((700, 20003), (700, 33001), (2000, 4099), (2000, 4096)):
        flat = randn(k + stride, 3 + k + stride * m, dtype=dtype)
        x = flat[3:].as_strided((m, k), (stride, 1), 3)
        want = kernels.int8_quantize(x.contiguous())
        assert all(torch.equal(a, b) for a, b in zip(kernels.int8_quantize(x), want))
        want = kernels.int8_quantize(x.contiguous(), gate=x.contiguous())
        assert all(torch.equal(a, b) for a, b in zip(kernels.int8_quantize(x, gate=x), want))
        w = randn(1, k, dtype=dtype)
        want = kernels.int8_rmsnorm(x.contiguous(), w, 1e-5, residual=x.contiguous())
        got = kernels.int8_rmsnorm(x, w, 1e-5, residual=x)
        assert torch.equal(got[2], want[2]) and torch.equal(got[0], want[0])
        # (another path may sum the squares in another order)
        assert ((got[1] - want[1]).abs() <= 2.0 ** -19 * want[1]).all()


def test_ties_round_to_even(cuda):
    """max |y| = 127 makes the factor exactly 1: halves are ties."""
    y = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5]], device="cuda")
    codes, scale = kernels.int8_quantize(y)
    assert codes.tolist() == [[127, 0, 2, 2, 0, -2, -2, 126]] and scale.item() == 1.0


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("k", [100, 4096, 20000])
def test_rows_without_finite_values(cuda, k, dtype):
    """Zero, all but zero, NaN and infinite rows, each beside ordinary ones that stay as they are."""
    x = randn(k, 9, k, dtype=dtype)
    x[1] = 0
    x[2, k // 2] = float("nan")
    x[3, k - 1] = float("inf")
    x[4, 0] = -float("inf")
    x[5] = float("nan")
    x[6, 3], x[6, 4] = float("nan"), float("inf")
    x[7] = torch.finfo(dtype).min
    codes, scale = kernels.int8_quantize(x)
    check_rows(codes[[0, 1, 8]], scale[[0, 1, 8]], x[[0, 1, 8]])
    assert codes[1:7].abs().max() == 0 and scale[1] == 0 and scale[2:7].isnan().all()
    assert (codes[7] == -127).all() and torch.isfinite(scale[7])
    back = kernels.int8_dequantize(codes, scale, dtype=F32)
    assert (back[1] == 0).all() and back[2:7].isnan().all()
    w = torch.ones(k, dtype=dtype, device="cuda")
    codes, scale, h = kernels.int8_rmsnorm(x, w, 1e-5, residual=torch.zeros_like(x))
    assert torch.equal(h[[0, 8]], x[[0, 8]]) and scale[2:7].isnan().all()
    assert codes[1:7].abs().max() == 0 and scale[1] == 0
    hd = x[[0, 8]].double()
    check_rows(codes[[0, 8]], scale[[0, 8]],
               hd * torch.rsqrt(hd.square().mean(-1, keepdim=True) + 1e-5), e=2.0 ** -19)


def test_rows_near_the_smallest_scale(cuda):
    """Just below 2^-119 a row is stored as zeros, from there on as codes; an all-zero row normed
    with eps 0 is 0 * infinity."""
    x = torch.zeros(4, 64, device="cuda")
    x[0, 5], x[1, 5] = TINY, TINY * (1 - 2.0 ** -24)
    x[2, 5], x[2, 6] = TINY * 3, -TINY
    x[3] = 2.0 ** -149
    codes, scale = kernels.int8_quantize(x)
    check_rows(codes, scale, x)
    assert scale[1] == 0 and scale[3] == 0 and scale[0] > 0
    codes, scale = kernels.int8_rmsnorm(torch.zeros(1, 64, device="cuda"),
                                        torch.ones(64, device="cuda"), 0.0)
    assert scale.isnan().all() and codes.abs().max() == 0


def test_gate_of_extreme_values(cuda):
    """silu(g) = g / (1 + exp(-g)): 0 far below zero, g far above, NaN at -infinity."""
    gate = torch.tensor([[-200.0, 200.0, -1e30, 0.0], [1.0, 1.0, -float("inf"), 1.0],
                         [3e38, 1.0, 1.0, 1.0]], device="cuda")
    up = torch.ones_like(gate)
    codes, scale = kernels.int8_quantize(up, gate=gate)
    assert codes[0].tolist() == [0, 127, 0, 0] and abs(scale[0].item() * 127 - 200) < 1e-4
    assert scale[1].isnan() and codes[1].abs().max() == 0
    assert codes[2].tolist() == [127, 0, 0, 0] and torch.isfinite(scale[2])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_row_layouts(cuda, dtype):
    """Strided halves, unaligned starts, overlapping and broadcast rows, transposed, 1-D, 3-D and
    empty tensors give what compact copies give."""
    base = randn(3, 12, 1000, dtype=dtype)
    views = [base[:, :504], base[:, 496:], base[:, 1:801], base[::2, 3:300], base[:1].expand(5, -1),
             base.t(), base[0], base.view(3, 4, 1000), base.view(3, 4, 1000)[:, 1:3, 7:900],
             base.as_strided((9, 64), (8, 1)), base[:0], base[:, 5:6]]
    views += [base[:, s:s + n] for s in range(1, 9) for n in (600, 601, 604, 33)]
    for v in views:
        codes, scale = kernels.int8_quantize(v)
        c2, s2 = kernels.int8_quantize(v.clone(memory_format=torch.contiguous_format))
        assert codes.shape == v.shape and codes.is_contiguous()
        assert torch.equal(codes, c2) and torch.equal(scale, s2)
        w = randn(v.shape[-1], v.shape[-1], dtype=dtype)
        got = kernels.int8_rmsnorm(v, w, 1e-6, residual=v)
        want = kernels.int8_rmsnorm(v.contiguous(), w, 1e-6, residual=v.contiguous())
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        got = kernels.int8_quantize(v, gate=v)
        want = kernels.int8_quantize(v.contiguous(), gate=v.contiguous())
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_rows_of_every_alignment(cuda, dtype):
    """Both inputs, the codes and the hidden rows at every offset from a 16-byte boundary; the bytes
    around the outputs stay as they were."""
    m, k = 5, 1037
    for ox, os, oc in ((0, 0, 0), (1, 2, 3), (3, 0, 5), (0, 5, 8), (7, 7, 7), (2, 4, 6), (4, 1, 1)):
        x = randn(ox, m, k + 40, dtype=dtype)[:, ox:ox + k]
        second = randn(os + 50, m, k + 24, dtype=dtype)[:, os:os + k]
        w = randn(oc + 90, k + 16, dtype=dtype)[oc:oc + k]
        flat = torch.full((m * k + 64,), 77, dtype=torch.int8, device="cuda")
        codes = flat[16 + oc:16 + oc + m * k].view(m, k)
        hflat = torch.full((m * k + 64,), 77, dtype=dtype, device="cuda")
        hidden = hflat[16 + os:16 + os + m * k].view(m, k)
        out = (codes, torch.empty(m, device="cuda"))
        kernels.int8_quantize(x, out=out)
        check_rows(*out, x)
        kernels.int8_quantize(x, gate=second, out=out)
        g = second.double()
        check_rows(*out, g * torch.sigmoid(g) * x.double(), e=2.0 ** -19)
        kernels.int8_rmsnorm(x, w, 1e-5, residual=second, out=out, hidden=hidden)
        assert torch.equal(hidden, (x.double() + second.double()).to(dtype))
        hd = hidden.double()
        check_rows(*out, hd * torch.rsqrt(hd.square().mean(-1, keepdim=True) + 1e-5) * w.double(),
                   e=2.0 ** -19)
        assert (flat[:16 + oc] == 77).all() and (flat[16 + oc + m * k:] == 77).all()
        assert (hflat[:16 + os] == 77).all() and (hflat[16 + os + m * k:] == 77).all()
        # and back, from codes and to values at these offsets
        back = hflat[16 + os:16 + os + m * k].view(m, k)
        kernels.int8_dequantize(*out, out=back)
        assert torch.equal(back, (codes.float() * out[1][:, None]).to(dtype))
        assert (hflat[:16 + os] == 77).all() and (hflat[16 + os + m * k:] == 77).all()


def test_given_outputs(cuda):
    x, r = randn(1, 5, 256), randn(2, 5, 256)
    w = randn(3, 256)
    want = kernels.int8_rmsnorm(x, w, 1e-5, residual=r)
    out = (torch.empty(5, 256, dtype=torch.int8, device="cuda"), torch.empty(5, device="cuda"))
    for into in (torch.empty_like(x), x.clone(), r.clone()):
        xi = into if torch.equal(into, x) else x
        ri = into if torch.equal(into, r) else r
        c, s, h = kernels.int8_rmsnorm(xi, w, 1e-5, residual=ri, out=out, hidden=into)
        assert h is into and c is out[0] and s is out[1]
        assert all(torch.equal(a, b) for a, b in zip((c, s, h), want))
    c, s = kernels.int8_quantize(x, out=out)
    assert c is out[0] and all(torch.equal(a, b) for a, b in zip((c, s), kernels.int8_quantize(x)))
    y = torch.empty(5, 256, dtype=F32, device="cuda")
    assert kernels.int8_dequantize(c, s, out=y) is y
    assert torch.equal(y, kernels.int8_dequantize(c, s, dtype=F32))


# ---- the matrix product --------------------------------------------------------------------------

def operands(seed, m, k, n, dtype=BF, bias=False, residual=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(-127, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-128, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    qs = torch.rand(m, generator=g, device="cuda") + 0.1
    ws = (torch.rand(n, generator=g, device="cuda") + 0.1) / k
    b = torch.randn(n, generator=g, device="cuda").to(dtype) if bias else None
    r = torch.randn(m, n, generator=g, device="cuda").to(dtype) if residual else None
    return q, qs, w, ws, b, r


def check_linear(y, q, qs, w, ws, b=None, r=None):
    p = q.double() @ w.double().t() * qs.double()[:, None] * ws.double()
    ref, size = p.clone(), p.abs()
    for t in (b, r):
        if t is not None:
            ref += t.double()
            size += t.double().abs()
    f = torch.finfo(y.dtype)
    err32 = 2.0 ** -22 * size
    bound = err32 + f.eps / 2 * (ref.abs() + err32).clamp_min(f.smallest_normal)
    assert ((y.double() - ref).abs() <= bound).all()


@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 32, 33, 64, 65, 128, 129, 256, 257, 300])
@pytest.mark.parametrize("k,n", [(16, 1), (128, 128), (144, 129), (1040, 333), (4096, 512)])
def test_linear_tiles(cuda, m, k, n, path):
    """Token counts around every tile width, K and N with ends inside a tile."""
    q, qs, w, ws, b, r = operands(m + k + n, m, k, n)
    y = kernels.int8_linear(q, qs, w, ws, path=path)
    torch.cuda.synchronize()
    assert kernels.device_status() == 0
    check_linear(y, q, qs, w, ws)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True),
                                           (True, True)])
@pytest.mark.parametrize("m,k,n", [(1, 4096, 301), (7, 512, 4096), (100, 1024, 200),
                                   (515, 640, 777)])
def test_linear_epilogues(cuda, m, k, n, bias, residual, dtype):
    q, qs, w, ws, b, r = operands(m * n + k, m, k, n, dtype, bias, residual)
    got = [kernels.int8_linear(q, qs, w, ws, bias=b, residual=r, dtype=dtype, path=p)
           for p in (None, 1, 2)]
    check_linear(got[0], q, qs, w, ws, b, r)
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    if residual:   # in place
        into = r.clone()
        assert kernels.int8_linear(q, qs, w, ws, bias=b, residual=into, dtype=dtype,
                                   out=into) is into
        assert torch.equal(into, got[0])


@pytest.mark.parametrize("m,k,n", [(1, 4096, 6144), (16, 14336, 4096), (333, 2048, 5632),
                                   (2048, 4096, 1024), (1024, 8192, 8192), (4099, 1024, 4096),
                                   (1500, 512, 4096), (2100, 256, 5000), (530, 384, 20000),
                                   (1111, 640, 9999), (700, 512, 8200)])
def test_linear_at_model_sizes(cuda, m, k, n):
    q, qs, w, ws, b, r = operands(k, m, k, n, residual=True)
    y = kernels.int8_linear(q, qs, w, ws, residual=r)
    torch.cuda.synchronize()
    assert kernels.device_status() == 0
    check_linear(y, q, qs, w, ws, r=r)


@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("m", [1, 40, 300])
def test_linear_sums_are_exact_at_the_longest_k(cuda, m, path):
    """Every product at its largest: 131056 * 128 * 127 (and 128 * 128) stay inside 32 bits."""
    k, n = 131056, 130
    q = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
    w = torch.full((n, k), -128, dtype=torch.int8, device="cuda")
    w[1] = 127
    one_m, one_n = torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
    y = kernels.int8_linear(q, one_m, w, one_n, dtype=F32, path=path)
    want = torch.full((n,), 128 * 128 * k, dtype=torch.float64)
    want[1] = -128 * 127 * k
    assert torch.equal(y.cpu(), want.float().expand(m, n))


@pytest.mark.parametrize("path", [1, 2])
def test_linear_rows_do_not_depend_on_the_batch(cuda, path):
    q, qs, w, ws, _, _ = operands(9, 300, 1056, 260)
    whole = kernels.int8_linear(q, qs, w, ws, path=path)
    for m in (1, 16, 33, 100, 257):
        assert torch.equal(kernels.int8_linear(q[:m], qs[:m], w, ws, path=1), whole[:m])


def test_linear_of_nan_and_zero_rows(cuda):
    """A row quantized from non-finite values gives NaN in its own output row alone; a zero row
    gives the bias."""
    x = randn(4, 40, 512)
    x[7, 100], x[8] = float("inf"), 0
    codes, scale = kernels.int8_quantize(x)
    _, _, w, ws, b, _ = operands(5, 1, 512, 200, bias=True)
    for path in (1, 2):
        y = kernels.int8_linear(codes, scale, w, ws, bias=b, path=path)
        assert y[7].isnan().all() and torch.equal(y[8], b)
        assert torch.isfinite(y[torch.arange(40, device="cuda") != 7]).all()


def test_linear_shapes(cuda):
    q, qs, w, ws, b, r = operands(6, 24, 256, 96, bias=True, residual=True)
    want = kernels.int8_linear(q, qs, w, ws, bias=b, residual=r)
    y = kernels.int8_linear(q.view(2, 3, 4, 256), qs.view(2, 3, 4), w, ws[:, None], bias=b,
                            residual=r.view(2, 3, 4, 96))
    assert y.shape == (2, 3, 4, 96) and torch.equal(y.view(24, 96), want)
    y = kernels.int8_linear(q.view(2, 12, 256), qs.view(2, 12, 1), w, ws, bias=b,
                            residual=r.view(2, 12, 96))
    assert torch.equal(y.view(24, 96), want)
    y = kernels.int8_linear(q[0], qs[0], w, ws, bias=b, residual=r[0])
    assert y.shape == (96,) and torch.equal(y, want[0])
    assert kernels.int8_linear(q[:0], qs[:0], w, ws).shape == (0, 96)
    assert kernels.int8_linear(q, qs, w[:0], ws[:0]).shape == (24, 0)


@pytest.mark.parametrize("m,k,n", [(1, 2048, 1024), (60, 2048, 1024), (700, 512, 9000)])
def test_linear_repeats_bit_for_bit(cuda, m, k, n):
    q, qs, w, ws, _, _ = operands(m, m, k, n)
    first = kernels.int8_linear(q, qs, w, ws)
    for _ in range(30):
        y = kernels.int8_linear(q, qs, w, ws)
        torch.cuda.synchronize()
        assert torch.equal(y, first)


def test_more_outputs_than_32_bits_count(cuda):
    """Output and row offsets past 2^31 elements: the last rows are right, and the first."""
    m, k, n = 70001, 16, 32768
    q, qs, w, ws, _, _ = operands(8, m, k, n)
    y = kernels.int8_linear(q, qs, w, ws)
    for rows in (slice(0, 3), slice(65530, 65545), slice(m - 3, m)):
        check_linear(y[rows], q[rows], qs[rows], w, ws)
    codes, scale = kernels.int8_quantize(y)
    for rows in (slice(0, 3), slice(65530, 65545), slice(m - 3, m)):
        check_rows(codes[rows], scale[rows], y[rows])
    back = kernels.int8_dequantize(codes, scale, out=y)
    for rows in (slice(0, 3), slice(65530, 65545), slice(m - 3, m)):
        assert torch.equal(back[rows], (codes[rows].float() * scale[rows, None]).to(BF))


# ---- together ------------------------------------------------------------------------------------

def mlp(x, res, norm_w, gate_up, down):
    """One MLP half of a layer as a user runs it; returns the new residual stream."""
    codes, scale, h = kernels.int8_rmsnorm(x, norm_w, 1e-5, residual=res)
    gu = kernels.int8_linear(codes, scale, *gate_up)
    i = gu.shape[-1] // 2
    codes, scale = kernels.int8_quantize(gu[..., i:], gate=gu[..., :i])
    return kernels.int8_linear(codes, scale, *down, residual=h)


def mlp_weights(seed, h, i):
    gate_up = kernels.int8_quantize(randn(seed, 2 * i, h) * h ** -0.5)
    down = kernels.int8_quantize(randn(seed + 1, h, i) * i ** -0.5)
    return randn(seed + 2, h).abs() + 0.5, gate_up, down


@pytest.mark.parametrize("m", [1, 5, 130, 600])
def test_mlp_matches_the_dequantized_model(cuda, m):
    """The whole half layer, each kernel's own 8-bit rows in 64-bit arithmetic between: only the
    roundings of its bf16 outputs separate the two."""
    h, i = 512, 1408
    norm_w, gate_up, down = mlp_weights(m, h, i)
    x, res = randn(m + 3, m, h), randn(m + 4, m, h)
    got = mlp(x, res, norm_w, gate_up, down)
    codes, scale, hid = kernels.int8_rmsnorm(x, norm_w, 1e-5, residual=res)
    gu = kernels.int8_linear(codes, scale, *gate_up)
    check_linear(gu, codes, scale, *gate_up)
    c2, s2 = kernels.int8_quantize(gu[:, i:], gate=gu[:, :i])
    g = gu[:, :i].double()
    check_rows(c2, s2, g * torch.sigmoid(g) * gu[:, i:].double(), e=2.0 ** -19)
    check_linear(got, c2, s2, *down, r=hid)


@pytest.mark.parametrize("m", [1, 200])
def test_mlp_in_a_graph_and_on_another_stream(cuda, m):
    """Captured once and replayed on new inputs, two graphs alive at once, and eagerly on a side
    stream: the same bits as on the default stream."""
    h, i = 512, 1408
    weights = mlp_weights(11, h, i)
    xs = [(randn(20 + s, m, h), randn(30 + s, m, h)) for s in range(4)]
    want = [mlp(x, r, *weights) for x, r in xs]
    bufs = [[t.clone() for t in xs[0]] for _ in range(2)]
    graphs, outs = [], []
    for x, r in bufs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(mlp(x, r, *weights))
        graphs.append(g)
    for s in range(0, 4, 2):
        for b in range(2):
            for dst, src in zip(bufs[b], xs[s + b]):
                dst.copy_(src)
        graphs[0].replay()
        graphs[1].replay()
        assert torch.equal(outs[0], want[s]) and torch.equal(outs[1], want[s + 1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [mlp(x, r, *weights) for x, r in xs]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_weights_written_just_before_they_are_read(cuda):
    """Back-to-back launches that overlap their prologues: a product reads the codes, scales and
    weights that the launch before it wrote."""
    big = randn(1, 4096, 4096)
    small = randn(2, 4, 4096)
    want = None
    for it in range(8):
        w, ws = kernels.int8_quantize(big * (it % 2 + 1))
        q, qs = kernels.int8_quantize(small)
        y = kernels.int8_linear(q, qs, w, ws, dtype=F32)
        if it == 0:
            want = y
        elif it % 2 == 0:
            assert torch.equal(y, want)


def test_calls_at_once(cuda):
    """Threads on streams of their own: products of both kinds, the 4-bit product's tensor-core
    kernel and the row kernels at the same time give what they give alone."""
    from rocketllm_b200.synthetic import make_activation, make_weight
    pair, split = operands(1, 600, 512, 9000), operands(2, 40, 2048, 1024)
    rows = randn(3, 2500, 4096)
    packed = make_weight(4096, 1024, device=cuda, seed=4)
    x4 = make_activation(200, 1024, device=cuda, seed=5)

    def calls():
        return [kernels.int8_linear(*pair[:4]), kernels.int8_linear(*split[:4]),
                *kernels.int8_quantize(rows), kernels.linear(x4, *packed)]

    want = calls()
    torch.cuda.synchronize()
    bad = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(25):
                got = calls()[::-1 if i % 2 else 1]
                stream.synchronize()
                bad.extend(k for k, (a, b) in enumerate(zip(got, want[::-1 if i % 2 else 1]))
                           if not torch.equal(a, b))

    with ThreadPoolExecutor(4) as pool:
        for done in [pool.submit(work, i) for i in range(4)]:
            done.result()
    assert not bad and kernels.device_status() == 0


def _linear_calls():
    q, qs, w, ws = operands(1, 40, 2048, 1024)[:4]
    q2, qs2, w2, ws2 = operands(2, 600, 512, 9000)[:4]
    return [lambda out=None: kernels.int8_linear(q, qs, w, ws, out=out),
            lambda out=None: kernels.int8_linear(q2, qs2, w2, ws2, out=out)]


def _packed_calls():
    from rocketllm_b200.synthetic import make_activation, make_weight
    packed = make_weight(4096, 1024, device="cuda", seed=4)
    few, many = (make_activation(m, 1024, device="cuda", seed=5) for m in (1, 200))
    return [lambda out=None: kernels.linear(few, *packed, out=out),
            lambda out=None: kernels.linear(many, *packed, out=out)]


@pytest.mark.parametrize("make", [_linear_calls, _packed_calls])
@pytest.mark.parametrize("captured", [False, True])
def test_first_call_of_a_thread(cuda, make, captured):
    """A product can be the first CUDA call that a thread makes: its results in memory that the
    allocator holds already, or given, on a stream that is captured."""
    for call in make():
        want, stream = call(), torch.cuda.Stream()
        out = torch.zeros_like(want) if captured else None
        with torch.cuda.stream(stream):
            call()                 # leaves its memory with the stream
        torch.cuda.synchronize()

        def work():
            torch.cuda.set_stream(stream)
            return call(out)

        with ThreadPoolExecutor(1) as pool:
            if captured:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream, capture_error_mode="relaxed"):
                    got = pool.submit(work).result()
                graph.replay()
            else:
                got = pool.submit(work).result()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_native_and_ctypes_calls_agree(cuda, monkeypatch):
    x, r, w = randn(1, 6, 512), randn(2, 6, 512), randn(3, 512)
    q, qs, wq, wsc, b, res = operands(4, 6, 512, 320, bias=True, residual=True)

    def all_calls():
        c, s = kernels.int8_quantize(x)
        return [c, s, *kernels.int8_quantize(x, gate=r), *kernels.int8_rmsnorm(x, w, 1e-5),
                *kernels.int8_rmsnorm(x, w, 1e-5, residual=r), kernels.int8_dequantize(c, s),
                kernels.int8_linear(q, qs, wq, wsc),
                kernels.int8_linear(q, qs, wq, wsc, bias=b, residual=res)]

    fast = all_calls()
    calls = []
    real = kernels._native
    assert real is not None

    class Spy:
        def __getattr__(self, name):
            def f(*a):
                out = getattr(real, name)(*a)
                calls.append((name, out is not None))
                return out
            return f

    monkeypatch.setattr(kernels, "_native", Spy())
    all_calls()
    assert len(calls) == 7 and all(took for _, took in calls)   # no plain call is declined
    monkeypatch.setattr(kernels, "_native", None)
    slow = all_calls()
    assert all(torch.equal(a, b) for a, b in zip(fast, slow))


@pytest.mark.parametrize("native", [True, False])
def test_refusals(cuda, native, monkeypatch):
    if not native:
        monkeypatch.setattr(kernels, "_native", None)
    x = randn(1, 4, 256)
    q, qs, w, ws, b, r = operands(2, 4, 256, 96, bias=True, residual=True)
    bad = [
        (TypeError, lambda: kernels.int8_quantize(x.double())),
        (TypeError, lambda: kernels.int8_quantize(q)),
        (ValueError, lambda: kernels.int8_quantize(x[:, :0])),
        (ValueError, lambda: kernels.int8_quantize(torch.zeros((), device="cuda"))),
        (ValueError, lambda: kernels.int8_quantize(torch.zeros(1, 131057, device="cuda"))),
        (ValueError, lambda: kernels.int8_quantize(x, gate=x[:, :128])),
        (ValueError, lambda: kernels.int8_quantize(x, gate=x.float())),
        (ValueError, lambda: kernels.int8_quantize(x, gate=x.cpu())),
        (ValueError, lambda: kernels.int8_quantize(x, out=(q[:2], qs))),
        (TypeError, lambda: kernels.int8_quantize(x, out=(q, qs.half()))),
        (ValueError, lambda: kernels.int8_rmsnorm(x, x[0, :128], 1e-5)),
        (ValueError, lambda: kernels.int8_rmsnorm(x, x[0].float(), 1e-5)),
        (ValueError, lambda: kernels.int8_rmsnorm(x, x[0], 1e-5, residual=x[:2])),
        (ValueError, lambda: kernels.int8_rmsnorm(x, x[0], 1e-5, hidden=x)),
        (ValueError, lambda: kernels.int8_rmsnorm(x, x[0], 1e-5, residual=x, hidden=x[:2])),
        (RuntimeError, lambda: kernels.int8_rmsnorm(x, x[0], -1.0)),
        (TypeError, lambda: kernels.int8_dequantize(x, qs)),
        (TypeError, lambda: kernels.int8_dequantize(q, qs, dtype=torch.float64)),
        (ValueError, lambda: kernels.int8_dequantize(q, qs[:2])),
        (ValueError, lambda: kernels.int8_dequantize(q, qs, out=x[:2])),
        (TypeError, lambda: kernels.int8_linear(x, qs, w, ws)),
        (TypeError, lambda: kernels.int8_linear(q, qs.half(), w, ws)),
        (ValueError, lambda: kernels.int8_linear(q, qs[:3], w, ws)),
        (ValueError, lambda: kernels.int8_linear(q, qs, w, ws[:3])),
        (ValueError, lambda: kernels.int8_linear(q[:, :128].contiguous(), qs, w, ws)),
        (ValueError, lambda: kernels.int8_linear(q[:, :128], qs, w[:, :128].contiguous(), ws)),
        (ValueError, lambda: kernels.int8_linear(q, qs, w.cpu(), ws)),
        (ValueError, lambda: kernels.int8_linear(q, qs, w, ws, bias=b.float())),
        (ValueError, lambda: kernels.int8_linear(q, qs, w, ws, bias=b[:5])),
        (ValueError, lambda: kernels.int8_linear(q, qs, w, ws, residual=r[:2])),
        (ValueError, lambda: kernels.int8_linear(q, qs, w, ws, out=r[:2])),
        (TypeError, lambda: kernels.int8_linear(q, qs, w, ws, dtype=torch.int32)),
        (RuntimeError, lambda: kernels.int8_linear(q[:, :40].contiguous(), qs,
                                                   w[:, :40].contiguous(), ws)),
        (RuntimeError, lambda: kernels.int8_linear(q, qs, w, ws, path=7)),
    ]
    for i, (err, call) in enumerate(bad):
        with pytest.raises(err):
            call()
            pytest.fail(f"call {i} was not refused")
    # codes that do not start on a 16-byte boundary
    flat = torch.zeros(4 * 256 + 8, dtype=torch.int8, device="cuda")
    with pytest.raises(RuntimeError, match="16-byte"):
        kernels.int8_linear(flat[8:].view(4, 256), qs, w, ws)
    torch.cuda.synchronize()
