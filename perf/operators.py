"""Cases of the 8-bit (W8A8) operators: the per-row quantizer (of a tensor or of a SwiGLU product),
the RMS norm that quantizes its output, and the integer matrix product with a scale per token and
per output channel.  ``run`` computes them in plain torch operations, or through
``rocketllm_b200.kernels`` where ``own`` is true.

8-bit outputs are returned as the values they stand for (code times scale, in bf16).
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_EPS = 1e-5
# below this magnitude a row's scale would be subnormal: the row is stored as zeros
_TINY = 2.0 ** -119


def listed():
    return [
        # one decoded token's attention output on its way to o_proj (hidden size 4096): latency
        {"name": "quant_1x4096", "op": "quant", "m": 1, "k": 4096, "dtype": "bf16"},
        # a prompt of odd length at the width of a 1.1B model's MLP, in fp16
        {"name": "quant_1001x5632_fp16", "op": "quant", "m": 1001, "k": 5632, "dtype": "fp16"},
        # the MLP product of a decode batch: gate and up are halves of one projection's output
        {"name": "swiglu_16x14336", "op": "swiglu", "m": 16, "k": 14336, "dtype": "bf16"},
        # the MLP product of a 2048-token prompt of a 70B model
        {"name": "swiglu_2048x28672", "op": "swiglu", "m": 2048, "k": 28672, "dtype": "bf16"},
        # the norm between two halves of a layer, one decoded token: latency
        {"name": "norm_1x4096", "op": "norm", "m": 1, "k": 4096, "dtype": "bf16", "residual": True},
        # the first norm of a model (no residual yet), odd prompt, fp32 stream
        {"name": "norm_515x2048_fp32", "op": "norm", "m": 515, "k": 2048, "dtype": "fp32",
         "residual": False},
        # the norm of a long prompt (or many) of a 70B model
        {"name": "norm_8192x8192", "op": "norm", "m": 8192, "k": 8192, "dtype": "bf16",
         "residual": True},
        # q|k|v of one decoded token: the weight's bytes and the launch are all there is
        {"name": "linear_1x4096x6144", "op": "linear", "m": 1, "k": 4096, "n": 6144,
         "dtype": "bf16", "bias": False, "residual": False},
        # down_proj of a decode batch with the residual stream added
        {"name": "linear_16x14336x4096_res", "op": "linear", "m": 16, "k": 14336, "n": 4096,
         "dtype": "bf16", "bias": False, "residual": True},
        # a short prompt of odd length through a projection with a bias, in fp16
        {"name": "linear_333x2048x5632_bias", "op": "linear", "m": 333, "k": 2048, "n": 5632,
         "dtype": "fp16", "bias": True, "residual": False},
        # gate|up of a 2048-token prompt of an 8B model
        {"name": "linear_2048x4096x28672", "op": "linear", "m": 2048, "k": 4096, "n": 28672,
         "dtype": "bf16", "bias": False, "residual": False},
        # down_proj of a batch of long prompts of an 8B model, residual added
        {"name": "linear_8192x14336x4096_res", "op": "linear", "m": 8192, "k": 14336, "n": 4096,
         "dtype": "bf16", "bias": False, "residual": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quant", "swiglu", "norm", "linear", "linear"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "linear":
        # the integer product reads rows in 16-byte units: K is a multiple of 16, N is any number
        k = 16 * _log_int(rng, 16, 14336 // 16)
        n = _log_int(rng, 64, 28672)
        m = _log_int(rng, 1, 8192)
        limit = 8192 * 14336 * 4096
        m = max(1, min(m, limit // (k * n), (1 << 25) // n))
        return {"op": op, "m": m, "k": k, "n": n, "dtype": dtype, "bias": rng.random() < 0.3,
                "residual": rng.random() < 0.5}
    k = _log_int(rng, 65, 53248)
    m = max(1, min(_log_int(rng, 1, 8192), (1 << 25) // k))
    case = {"op": op, "m": m, "k": k, "dtype": dtype}
    if op == "norm":
        case["residual"] = rng.random() < 0.7
    return case


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    m, k, dt = case["m"], case["k"], _DTYPES[case["dtype"]]
    s = {"op": case["op"], "dtype": dt}
    if case["op"] == "quant":
        s["x"] = (_normal(g, m, k) * 0.7).to(dt)
    elif case["op"] == "swiglu":
        # one projection's output: gate in the left half of each row, up in the right
        gu = _normal(g, m, 2 * k).to(dt)
        s["gate"], s["up"] = gu[:, :k], gu[:, k:]
    elif case["op"] == "norm":
        s["x"] = _normal(g, m, k).to(dt)
        # a few channels of the stream carry most of its energy, as in trained models
        boost = 1 + 20 * (torch.rand(k, generator=g, device="cuda") < 0.002).float()
        s["res"] = (3 * _normal(g, m, k) * boost).to(dt) if case["residual"] else None
        s["w"] = (1 + 0.2 * _normal(g, k)).to(dt)
    else:
        n = case["n"]
        s["q"] = (_normal(g, m, k) * 31).round().clamp(-127, 127).to(torch.int8)
        s["qs"] = torch.rand(m, generator=g, device="cuda") * 0.03 + 0.01
        s["w"] = (_normal(g, n, k) * 31).round().clamp(-127, 127).to(torch.int8)
        s["ws"] = (torch.rand(n, generator=g, device="cuda") + 0.5) / (31 * math.sqrt(k))
        s["bias"] = (0.1 * _normal(g, n)).to(dt) if case["bias"] else None
        s["res"] = _normal(g, m, n).to(dt) if case["residual"] else None
    return s


def _plain_rows(y):
    """(values, scale) of fp32 rows quantized to 8 bits: one scale a row, ties to even."""
    a = y.abs().amax(-1, keepdim=True)
    live = a >= _TINY
    one = torch.ones_like(a)
    q = torch.round(y * torch.where(live, 127 / torch.where(live, a, one), 0 * one))
    scale = torch.where(live, a / 127, 0 * one)
    return (q * scale).to(torch.bfloat16), scale[:, 0]


def _plain(s):
    if s["op"] == "quant":
        return _plain_rows(s["x"].float())
    if s["op"] == "swiglu":
        gate = s["gate"].float()
        return _plain_rows(gate / (1 + torch.exp(-gate)) * s["up"].float())
    if s["op"] == "norm":
        h = s["x"]
        if s["res"] is not None:
            h = (s["x"].float() + s["res"].float()).to(s["dtype"])
        hf = h.float()
        y = hf * torch.rsqrt((hf * hf).mean(-1, keepdim=True) + _EPS) * s["w"].float()
        out = _plain_rows(y)
        return out if s["res"] is None else out + (h,)
    y = torch.matmul(s["q"].float(), s["w"].float().t())
    y = y * s["qs"][:, None] * s["ws"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["res"] is not None:
        y = y + s["res"].float()
    return y.to(s["dtype"])


def _own(s):
    from rocketllm_b200 import kernels
    if s["op"] == "linear":
        return kernels.int8_linear(s["q"], s["qs"], s["w"], s["ws"], bias=s["bias"],
                                   residual=s["res"], dtype=s["dtype"])
    hidden = ()
    if s["op"] == "quant":
        codes, scale = kernels.int8_quantize(s["x"])
    elif s["op"] == "swiglu":
        codes, scale = kernels.int8_quantize(s["up"], gate=s["gate"])
    else:
        codes, scale, *hidden = kernels.int8_rmsnorm(s["x"], s["w"], _EPS, residual=s["res"])
    return (kernels.int8_dequantize(codes, scale, dtype=torch.bfloat16), scale, *hidden)


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    m, k, e = case["m"], case["k"], _BYTES[case["dtype"]]
    if case["op"] == "linear":
        n = case["n"]
        b = m * k + n * k + 4 * (m + n) + m * n * e * (2 if case["residual"] else 1)
        return {"bytes": b + (n * e if case["bias"] else 0), "flops": 2 * m * n * k}
    out = 2 * m * k + 4 * m
    if case["op"] == "quant":
        return {"bytes": m * k * e + out, "flops": 3 * m * k}
    if case["op"] == "swiglu":
        return {"bytes": 2 * m * k * e + out, "flops": 8 * m * k}
    rows = 3 if case["residual"] else 1
    return {"bytes": (rows * m * k + k) * e + out, "flops": 8 * m * k}


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "linear":
        y = torch.einsum("mk,nk->mn", s["q"].double(), s["w"].double())
        y *= torch.outer(s["qs"].double(), s["ws"].double())
        for more in (s["bias"], s["res"]):
            if more is not None:
                y += more.double()
        return y
    hidden = []
    if s["op"] == "quant":
        y = s["x"].double()
    elif s["op"] == "swiglu":
        y = s["up"].double() * s["gate"].double() * torch.sigmoid(s["gate"].double())
    else:
        h = s["x"].double()
        if s["res"] is not None:
            h = h + s["res"].double()
            # the stored stream is the sum rounded to the inputs' type (two such values' sum,
            # rounded once from 64 bits); the norm is that of the stored stream
            h = h.to(s["dtype"]).double()
            hidden = [h]
        y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + _EPS) * s["w"].double()
    top = y.abs().max(-1, keepdim=True).values
    step = torch.where(top < _TINY, torch.ones_like(top), top / 127)
    codes = torch.round(y / step)
    step = torch.where(top < _TINY, torch.zeros_like(top), step)
    return tuple([codes * step, step[:, 0]] + hidden)
