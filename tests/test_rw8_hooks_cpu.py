"""What happens around the 8-bit Llama layers on CPU, the kernels replaced by their formulas: calls
that someone waits for are made."""
import pytest
import torch

from rocketllm_b200 import kernels
from rocketllm_b200.quant import RW8Linear, convert_modules_rw8, fuse_rw8_layers
from test_rw8_cpu import llama


def quantize(x, gate=None, out=None):
    y = x.float() if gate is None else torch.nn.functional.silu(gate.float()) * x.float()
    a = y.abs().amax(-1, keepdim=True).clamp_min(1e-30)
    return torch.round(y * (127 / a)).to(torch.int8), (a / 127)[..., 0]


def linear(codes, scale, weight, weight_scale, bias=None, residual=None, dtype=torch.bfloat16,
           out=None, path=None):
    y = codes.float() @ weight.float().t() * scale.reshape(*codes.shape[:-1], 1) * \
        weight_scale.reshape(-1)
    for more in (bias, residual):
        y = y if more is None else y + more.float()
    return y.to(dtype)


@pytest.fixture
def model(monkeypatch):
    """An RW8 Llama, and how often each 8-bit kernel was called."""
    calls = {"norm": 0, "gated": 0}

    def norm(x, weight, eps, residual=None, out=None, hidden=None):
        calls["norm"] += 1
        h = x if residual is None else x + residual
        y = h.float() * torch.rsqrt(h.float().square().mean(-1, keepdim=True) + eps) * weight.float()
        return quantize(y) if residual is None else (*quantize(y), h)

    def counted(x, gate=None, out=None):
        calls["gated"] += gate is not None
        return quantize(x, gate)

    monkeypatch.setattr(kernels, "int8_quantize", counted)
    monkeypatch.setattr(kernels, "int8_rmsnorm", norm)
    monkeypatch.setattr(kernels, "int8_linear", linear)
    dense = llama()
    weights = {n: quantize(m.weight.detach() * 5) for n, m in dense.named_modules()
               if isinstance(m, torch.nn.Linear)}
    for name in convert_modules_rw8(dense):
        m = dense.get_submodule(name)
        m.weight.data, m.weight_scale.data = weights[name][0], weights[name][1][:, None]
    return dense.eval(), calls


def run(model):
    with torch.no_grad():
        return model(torch.arange(12).view(2, 6)).logits


WATCHED = ["input_layernorm", "post_attention_layernorm", "mlp", "mlp.act_fn", "mlp.gate_proj",
           "mlp.up_proj", "mlp.down_proj", "self_attn.q_proj", "self_attn.k_proj",
           "self_attn.v_proj"]


@pytest.mark.parametrize("pre", [False, True])
@pytest.mark.parametrize("name", WATCHED)
def test_hooks_see_the_calls_of_the_modules(model, name, pre):
    """A hook on a module that the 8-bit forward passes by, or hands 8-bit rows, is called with
    tensors and may change them; once it is gone the layer is back on 8-bit rows."""
    model, calls = model
    modules = run(model)
    assert fuse_rw8_layers(model) == 2 and calls["norm"] == 0
    fused = run(model)
    assert calls == {"norm": 4, "gated": 2}
    seen = []
    watched = model.model.layers[1].get_submodule(name)

    def hook(module, args, out=None):
        seen.append(all(torch.is_tensor(t) for t in args) and (pre or torch.is_tensor(out)))

    handle = (watched.register_forward_pre_hook(hook) if pre else
              watched.register_forward_hook(hook))
    run(model)
    assert seen == [True] and calls == {"norm": 6, "gated": 3}   # the other layer's
    other = model.model.layers[0].get_submodule(name).register_forward_pre_hook(lambda m, a: None)
    assert torch.equal(run(model), modules)
    handle.remove()
    other.remove()
    assert torch.equal(run(model), fused)


def test_hooks_on_every_module_and_on_attention(model):
    model, calls = model
    fuse_rw8_layers(model)
    names = {m: n for n, m in model.named_modules()}
    seen = []
    handle = torch.nn.modules.module.register_module_forward_pre_hook(
        lambda m, a: seen.append(names[m]))
    try:
        run(model)
    finally:
        handle.remove()
    assert all(f"model.layers.{i}.{n}" in seen for i in range(2) for n in WATCHED)
    assert calls["norm"] == 0
    got = []
    layer = model.model.layers[0]
    layer.self_attn.register_forward_pre_hook(
        lambda m, a, k: got.append(k["hidden_states"]), with_kwargs=True)
    run(model)
    assert torch.is_tensor(got[0]) and calls["norm"] == 2


def test_forwards_and_adapters_put_in_after_fusing_are_called(model):
    model, calls = model
    fuse_rw8_layers(model)
    norm = model.model.layers[0].input_layernorm
    inner, seen = norm.forward, []
    norm.forward = lambda x: seen.append(1) or inner(x)      # as a dispatcher wraps a module
    run(model)
    assert seen == [1] and calls["norm"] == 2

    class Adapter(torch.nn.Module):
        def __init__(self, base):
            super().__init__()
            self.base = base

        def forward(self, x):
            return self.base(x) + x[..., :1]

    mlp = model.model.layers[1].mlp
    assert isinstance(mlp.up_proj, RW8Linear)
    mlp.up_proj = Adapter(mlp.up_proj)
    run(model)
    assert calls["norm"] == 2


def test_other_modules_in_the_place_of_those_passed_by_are_called(model):
    """Another activation or norm, put in before or after the layers were fused."""
    model, calls = model
    first, second = model.model.layers

    class Doubled(type(first.input_layernorm)):
        def forward(self, x):
            return 2 * super().forward(x)

    first.mlp.act_fn = torch.nn.GELU()
    assert fuse_rw8_layers(model) == 1
    second.mlp.act_fn = torch.nn.GELU()
    got = run(model)
    assert calls == {"norm": 0, "gated": 0}
    second.__dict__.pop("forward")
    assert torch.equal(run(model), got)        # the modules' own
    first.mlp.act_fn, second.mlp.act_fn = torch.nn.SiLU(), torch.nn.SiLU()
    first.input_layernorm.__class__ = Doubled
    assert fuse_rw8_layers(model) == 1         # not the first
    second.post_attention_layernorm.__class__ = Doubled
    run(model)
    assert calls == {"norm": 0, "gated": 0}


def test_layers_with_a_forward_of_their_own_keep_it(model):
    """A wrapped layer is left as it is; one that is wrapped after it was fused stays wrapped."""
    model, calls = model
    first, second = model.model.layers
    inner, seen = first.forward, []

    def wrapped(*a, **k):
        seen.append(1)
        return inner(*a, **k)

    first.forward = wrapped
    assert fuse_rw8_layers(model) == 1 and first.forward is wrapped
    run(model)
    assert seen == [1] and calls["norm"] == 2
    fused = second.forward
    second.forward = lambda *a, **k: fused(*a, **k)
    outer = second.forward
    assert fuse_rw8_layers(model) == 0 and second.forward is outer
    run(model)
    assert seen == [1, 1] and calls["norm"] == 4
    del first.forward, second.forward
    assert fuse_rw8_layers(model) == 2 and fuse_rw8_layers(model) == 2


def test_the_engine_leaves_layers_alone_when_asked(model, tmp_path):
    import json

    from rocketllm_b200.engine import RocketModel
    from rocketllm_b200.quant.hf import RW8Config
    from rocketllm_b200.shards import build_skeleton
    model, calls = model
    ids = torch.arange(12).view(2, 6)
    with torch.no_grad():
        want = run(model)
        plain = RocketModel(model, device="cpu", dtype=torch.float32, rw8_layers=False)
        assert torch.equal(plain(ids).logits, want) and calls["norm"] == 0
        RocketModel(model, device="cpu", dtype=torch.float32)(ids)
        assert calls["norm"] == 4
    cfg = model.config.to_dict()
    cfg["quantization_config"] = RW8Config().to_dict()
    (tmp_path / "config.json").write_text(json.dumps(cfg))
    for fused in (True, False):
        layers = build_skeleton(str(tmp_path), rw8_layers=fused).model.layers
        assert all(("forward" in layer.__dict__) == fused for layer in layers)
