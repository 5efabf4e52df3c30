"""Decoder layers of an RW8 Llama in their 8-bit form: what lies between two projections is one
kernel that ends in 8-bit rows.

Through the transformers modules a layer's norm writes a bf16 row that q, k and v each quantize
again, and the residual adds and the MLP's product are kernels of their own.  The layer forward here
keeps the attention module and computes

    int8_rmsnorm                   input_layernorm, quantized once for q, k and v
    self_attn                      the model's own; o_proj quantizes the attention output
    int8_rmsnorm(residual)         residual add + post_attention_layernorm, once for gate and up
    gate_proj, up_proj             8-bit products
    int8_quantize(up, gate=gate)   act_fn(gate) * up
    down_proj(residual)            the product with the residual added in its epilogue

Parameters are read at every call, so a streamed layer (whose parameters are views into the engine's
slots) takes the same path.

The norms and the MLP are not called as modules here, and the projections that read 8-bit rows get
:class:`Int8Rows`.  So a layer in which something waits for those calls -- a forward hook on one of
them (or on every module), a forward of its own, another module in its place -- runs the module's own
forward for as long as that is so.
"""
import types

from torch import nn
from torch.nn.modules import module as _nn

from .. import kernels
from .modules import Int8Rows, RW8Linear


def _passed_by(layer):
    """The types of the modules whose calls the 8-bit forward replaces."""
    mods = layer._modules
    m = mods.get("mlp")
    return [type(mods.get("input_layernorm")), type(mods.get("post_attention_layernorm")), type(m),
            type(m._modules.get("act_fn") if m is not None else None)]


def _covered(layer):
    from transformers.activations import ACT2FN
    from transformers.models.llama.modeling_llama import LlamaMLP, LlamaRMSNorm
    a, m = getattr(layer, "self_attn", None), getattr(layer, "mlp", None)
    return (all(isinstance(getattr(a, n, None), RW8Linear)
                for n in ("q_proj", "k_proj", "v_proj", "o_proj")) and
            all(isinstance(getattr(m, n, None), RW8Linear)
                for n in ("gate_proj", "up_proj", "down_proj")) and
            _passed_by(layer)[:3] == [LlamaRMSNorm, LlamaRMSNorm, LlamaMLP] and
            type(m.act_fn) in (nn.SiLU, type(ACT2FN["silu"])))


def fuse_rw8_layers(model):
    """Give every decoder layer of an RW8 Llama-architecture ``model`` the 8-bit forward above.
    Other models, and layers with other modules or with a forward of their own already (a dispatched
    or offloaded model's), are left as they are.  Returns how many layers have it."""
    cfg = getattr(model, "config", None)
    if getattr(cfg, "model_type", None) != "llama" or \
            getattr(cfg, "hidden_act", None) not in ("silu", "swish"):
        return 0
    layers = getattr(getattr(model, "model", None), "layers", ())
    n = 0
    for layer in layers:
        own = layer.__dict__.get("forward")
        if own is None and _covered(layer):
            layer._rw8_passed_by = _passed_by(layer)
            layer.forward = types.MethodType(rw8_layer_forward, layer)
            n += 1
        elif getattr(own, "__func__", None) is rw8_layer_forward:
            n += 1
    return n


def _norm(module, x, residual=None):
    w, eps = module.weight, float(module.variance_epsilon)
    if w.dtype == x.dtype:
        return kernels.int8_rmsnorm(x, w, eps, residual=residual)
    # a weight of another type (fp32 norms in a 16-bit model) is not rounded to the stream's: the
    # stream is rounded where int8_rmsnorm rounds it, the norm is taken in fp32
    h = x if residual is None else x + residual
    codes, scale = kernels.int8_rmsnorm(h.float(), w.float(), eps)
    return (codes, scale) if residual is None else (codes, scale, h)


_ROWS = (("self_attn", "q_proj"), ("self_attn", "k_proj"), ("self_attn", "v_proj"),
         ("mlp", "gate_proj"), ("mlp", "up_proj"), ("mlp", "down_proj"))


def _watched(module):
    d = module.__dict__
    return d["_forward_pre_hooks"] or d["_forward_hooks"] or "forward" in d


def _takes_rows(layer):
    """Whether the modules that the 8-bit forward passes by, or hands 8-bit rows, are as
    :func:`fuse_rw8_layers` found them and nothing watches their calls.  (Asked at every call, so in
    plain dictionary lookups: 3 us a layer.)"""
    if _nn._global_forward_pre_hooks or _nn._global_forward_hooks or \
            _passed_by(layer) != layer._rw8_passed_by:
        return False
    mods = layer._modules
    a, m = mods["self_attn"], mods["mlp"]
    for parent, name in _ROWS:
        p = mods[parent]._modules.get(name)
        if not isinstance(p, RW8Linear) or _watched(p):
            return False
    return not (a._forward_pre_hooks or _watched(m) or _watched(m._modules["act_fn"]) or
                _watched(mods["input_layernorm"]) or _watched(mods["post_attention_layernorm"]))


def rw8_layer_forward(self, hidden_states, attention_mask=None, position_ids=None,
                      past_key_values=None, use_cache=False, position_embeddings=None, **kwargs):
    """A Llama decoder layer (transformers ``models/llama/modeling_llama.py``) on 8-bit rows."""
    if not _takes_rows(self):
        return type(self).forward(self, hidden_states, attention_mask=attention_mask,
                                  position_ids=position_ids, past_key_values=past_key_values,
                                  use_cache=use_cache, position_embeddings=position_embeddings,
                                  **kwargs)
    dtype = hidden_states.dtype
    codes, scale = _norm(self.input_layernorm, hidden_states)
    attn, _ = self.self_attn(hidden_states=Int8Rows(codes, scale, dtype),
                             attention_mask=attention_mask, position_ids=position_ids,
                             past_key_values=past_key_values, use_cache=use_cache,
                             position_embeddings=position_embeddings, **kwargs)
    codes, scale, hidden = _norm(self.post_attention_layernorm, attn, residual=hidden_states)
    rows = Int8Rows(codes, scale, dtype)
    m = self.mlp
    codes, scale = kernels.int8_quantize(m.up_proj(rows), gate=m.gate_proj(rows))
    return m.down_proj(Int8Rows(codes, scale, dtype), residual=hidden)
