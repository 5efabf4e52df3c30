"""The RW8 (8-bit) plugin surface on CPU: registry detection and sizing, module replacement through
the transformers quantizer, loading a pre-quantized checkpoint by name, and which layers take the
8-bit forward.  No kernel runs here."""
import json

import pytest
import torch

from rocketllm_b200.quant import (RW8Backend, RW8Linear, convert_modules_rw8, decision_table,
                                  detect_backend, fuse_rw8_layers)
from rocketllm_b200.quant.hf import RW8Config, rw8_linears


def llama(**kw):
    from transformers import LlamaConfig, LlamaForCausalLM
    cfg = dict(hidden_size=64, intermediate_size=160, num_hidden_layers=2, num_attention_heads=4,
               num_key_value_heads=2, vocab_size=96, max_position_embeddings=64,
               tie_word_embeddings=False)
    cfg.update(kw)
    torch.manual_seed(0)
    return LlamaForCausalLM(LlamaConfig(**cfg))


def test_backend_groups_and_sizes():
    backend = detect_backend({"quant_method": "rw8", "bits": 8}, compute_dtype=torch.bfloat16)
    assert isinstance(backend, RW8Backend)
    name = "model.layers.0.mlp.down_proj"
    shard = {f"{name}.weight": torch.zeros(64, 160, dtype=torch.int8),
             f"{name}.weight_scale": torch.ones(64, 1), f"{name}.bias": torch.zeros(64).bfloat16()}
    weights = backend.plan(shard)
    assert [w.name for w in weights] == [f"{name}.weight", f"{name}.bias"]
    w = weights[0]
    assert w.payload.dtype == torch.int8 and w.bits == 8 and w.logical_shape == (64, 160)
    assert w.packed_bytes == 64 * 160 + 64 * 4 and w.expanded_bytes == 64 * 160 * 2
    assert w.needs_scratch is False
    # codes and scales are placed as stored, whatever the compute dtype
    for key, value in shard.items():
        want = torch.bfloat16 if key.endswith("bias") else value.dtype
        assert backend.target_dtype(key, value) == want
    assert {r["format"]: r for r in decision_table()}["rw8"]["path"] == "fused_packed"


def test_conversion_covers_the_linears_and_leaves_a_tied_head():
    names = convert_modules_rw8(llama())
    assert len(names) == 2 * 7 + 1 and "lm_head" in names
    tied = llama(tie_word_embeddings=True)
    assert "lm_head" not in convert_modules_rw8(tied)
    assert not isinstance(tied.lm_head, RW8Linear)
    some = [n for n, _ in rw8_linears(llama(), ["lm_head", "model.layers.1"])]
    assert len(some) == 7 and all(n.startswith("model.layers.0.") for n in some)
    # a width that is not a multiple of 16 stays dense
    narrow = llama(intermediate_size=100)
    assert not [n for n in convert_modules_rw8(narrow) if n.endswith("down_proj")]
    assert fuse_rw8_layers(narrow) == 0


def test_config_and_module_refusals():
    with pytest.raises(ValueError, match="8-bit"):
        RW8Config(bits=4)
    with pytest.raises(ValueError, match="% 16"):
        RW8Linear(100, 64)
    with pytest.raises(ValueError, match="% 16"):
        RW8Linear(131072, 64)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        RW8Linear(64, 32)(torch.zeros(1, 64, dtype=torch.bfloat16))


def test_only_rw8_llamas_take_the_8_bit_layers():
    dense = llama()
    forward = dense.model.layers[0].forward
    assert fuse_rw8_layers(dense) == 0 and dense.model.layers[0].forward == forward
    convert_modules_rw8(dense, ["model.layers.1.mlp"])
    assert fuse_rw8_layers(dense) == 1
    model = llama()
    convert_modules_rw8(model)
    assert fuse_rw8_layers(model) == 2
    assert fuse_rw8_layers(model) == 2   # again: the same layers
    assert fuse_rw8_layers(torch.nn.Linear(2, 2)) == 0
    other = llama(hidden_act="gelu")
    convert_modules_rw8(other)
    assert fuse_rw8_layers(other) == 0


def test_checkpoint_loads_verbatim(tmp_path):
    """A pre-quantized checkpoint (codes and scales made here, as the converter lays them out)
    loads through ``from_pretrained`` with every tensor as stored."""
    from safetensors.torch import save_file
    from transformers import AutoModelForCausalLM
    model = llama()
    sd = {}
    for name, module in rw8_linears(model):
        w = module.weight.detach()
        scale = w.abs().amax(1, keepdim=True) / 127
        sd[f"{name}.weight"] = torch.round(w / scale).to(torch.int8)
        sd[f"{name}.weight_scale"] = scale
    for name, p in model.state_dict().items():
        sd.setdefault(name, p.detach())
    save_file({k: v.contiguous() for k, v in sd.items()}, str(tmp_path / "model.safetensors"),
              metadata={"format": "pt"})
    cfg = model.config.to_dict()
    cfg["quantization_config"] = RW8Config().to_dict()
    (tmp_path / "config.json").write_text(json.dumps(cfg))
    got = AutoModelForCausalLM.from_pretrained(str(tmp_path), dtype=torch.bfloat16)
    q = got.model.layers[1].mlp.down_proj
    assert isinstance(q, RW8Linear) and q.weight.dtype == torch.int8
    assert q.weight_scale.dtype == torch.float32 and not q.weight.requires_grad
    assert torch.equal(q.weight, sd["model.layers.1.mlp.down_proj.weight"])
    assert torch.equal(q.weight_scale, sd["model.layers.1.mlp.down_proj.weight_scale"])
    assert isinstance(got.lm_head, RW8Linear)
    assert got.model.norm.weight.dtype == torch.bfloat16
    assert fuse_rw8_layers(got) == 2
