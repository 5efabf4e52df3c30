"""transformers integration: the ``rw4`` quantization config, its quantizer and experts function.

RocketLLM builds every model on the meta device and, when the checkpoint declares a
``quantization_config``, calls ``AutoHfQuantizer.from_config(...).preprocess_model(...)``
(``rocketllm/base.py:680-690``) -- the hook through which a format swaps ``nn.Linear`` for its own
module before any weight is read.  Registering ``rw4`` here makes that path (and plain
``AutoModelForCausalLM.from_pretrained``) build ``RW4Linear`` modules whose parameters are the
checkpoint's packed tensors, placed verbatim (``param_needs_quantization`` is False, so the engine's
coalesced placement copies them as stored, ``rocketllm/quant/registry.py:486-501``).

Stacked-expert modules (``MixtralExperts`` style: ``gate_up_proj [E, 2I, H]``, ``down_proj
[E, H, I]``) get RW4 triples for both weights and the model's experts implementation is pointed at
``rw4`` in transformers' ``ALL_EXPERTS_FUNCTIONS`` (``integrations/moe.py:432-515``).

``rw8`` is registered in the same way: its ``nn.Linear`` modules become ``RW8Linear`` (routed experts
stay dense).
"""
import torch
from torch import nn
from transformers.integrations.moe import ALL_EXPERTS_FUNCTIONS
from transformers.quantizers.auto import (AUTO_QUANTIZATION_CONFIG_MAPPING, AUTO_QUANTIZER_MAPPING,
                                          register_quantization_config, register_quantizer)
from transformers.quantizers.base import HfQuantizer
from transformers.utils.quantization_config import QuantizationConfigMixin

from .modules import RW4Linear, RW8Linear, rw4_experts_forward, rw4_experts_params

QUANT_METHOD = "rw4"
QUANT_METHOD_RW8 = "rw8"


class RW4Config(QuantizationConfigMixin):
    """``{"quant_method": "rw4", "bits": 4, "group_size": 64, "modules_to_not_convert": [...]}``."""

    def __init__(self, bits=4, group_size=64, modules_to_not_convert=None, **kwargs):
        if bits != 4 or group_size != 64:
            raise ValueError(f"rw4 is 4-bit with group 64, got bits={bits} group={group_size}")
        self.quant_method = QUANT_METHOD
        self.bits = bits
        self.group_size = group_size
        self.modules_to_not_convert = list(modules_to_not_convert or [])

    def to_dict(self):
        return {"quant_method": QUANT_METHOD, "bits": self.bits, "group_size": self.group_size,
                "modules_to_not_convert": list(self.modules_to_not_convert)}


def _is_stacked_experts(module):
    gu = getattr(module, "gate_up_proj", None)
    dn = getattr(module, "down_proj", None)
    return (isinstance(gu, nn.Parameter) and isinstance(dn, nn.Parameter) and gu.dim() == 3
            and dn.dim() == 3)


def convert_modules(model, modules_to_not_convert=()):
    """Replace every ``nn.Linear`` (and stacked-experts weight) not excluded by name with its RW4
    counterpart, on whatever device the skeleton lives (normally meta).  Returns the converted
    names."""
    converted = []
    skip = tuple(modules_to_not_convert)
    for name, module in list(model.named_modules()):
        if any(name == s or name.endswith("." + s) or name.startswith(s + ".") for s in skip):
            continue
        if isinstance(module, nn.Linear):
            parent_name, _, leaf = name.rpartition(".")
            parent = model.get_submodule(parent_name) if parent_name else model
            setattr(parent, leaf, RW4Linear.from_linear(module))
            converted.append(name)
        elif _is_stacked_experts(module):
            rw4_experts_params(module)
            converted.append(name)
    if any(getattr(m, "rw4", False) for m in model.modules()):
        model.config._experts_implementation = QUANT_METHOD
    return converted


class RW8Config(QuantizationConfigMixin):
    """``{"quant_method": "rw8", "bits": 8, "modules_to_not_convert": [...]}``."""

    def __init__(self, bits=8, modules_to_not_convert=None, **kwargs):
        if bits != 8:
            raise ValueError(f"rw8 is 8-bit, got bits={bits}")
        self.quant_method = QUANT_METHOD_RW8
        self.bits = bits
        self.modules_to_not_convert = list(modules_to_not_convert or [])

    def to_dict(self):
        return {"quant_method": QUANT_METHOD_RW8, "bits": self.bits,
                "modules_to_not_convert": list(self.modules_to_not_convert)}


def rw8_linears(model, modules_to_not_convert=()):
    """``(name, module)`` of every ``nn.Linear`` the RW8 format stores in 8 bits: not excluded by
    name, a width the integer product takes, and not an output head whose weight is tied to the
    embedding (it stays the embedding's)."""
    skip = tuple(modules_to_not_convert)
    tied = (model.get_output_embeddings() if hasattr(model, "get_output_embeddings") and
            getattr(getattr(model, "config", None), "tie_word_embeddings", False) else None)
    for name, module in list(model.named_modules()):
        if any(name == s or name.endswith("." + s) or name.startswith(s + ".") for s in skip):
            continue
        if isinstance(module, nn.Linear) and module is not tied and \
                RW8Linear.supports(module.in_features):
            yield name, module


def convert_modules_rw8(model, modules_to_not_convert=()):
    """Replace every ``nn.Linear`` of :func:`rw8_linears` with an ``RW8Linear``, on whatever device
    the skeleton lives (normally meta).  Returns the converted names."""
    converted = []
    for name, module in rw8_linears(model, modules_to_not_convert):
        parent_name, _, leaf = name.rpartition(".")
        parent = model.get_submodule(parent_name) if parent_name else model
        setattr(parent, leaf, RW8Linear.from_linear(module))
        converted.append(name)
    return converted


class RW4HfQuantizer(HfQuantizer):
    """Pre-quantized RW4 checkpoints only; packed tensors load verbatim into RW4 modules."""

    requires_calibration = True

    def validate_environment(self, *args, **kwargs):
        return

    def update_dtype(self, dtype):
        return torch.bfloat16 if dtype is None else dtype

    def param_needs_quantization(self, model, param_name, **kwargs):
        return False

    def _process_model_before_weight_loading(self, model, **kwargs):
        convert_modules(model, self.quantization_config.modules_to_not_convert)
        return model

    def _process_model_after_weight_loading(self, model, **kwargs):
        return model

    @property
    def is_serializable(self):
        return True

    @property
    def is_trainable(self):
        return False


class RW8HfQuantizer(RW4HfQuantizer):
    """Pre-quantized RW8 checkpoints only; codes and scales load verbatim into RW8 modules."""

    def _process_model_before_weight_loading(self, model, **kwargs):
        convert_modules_rw8(model, self.quantization_config.modules_to_not_convert)
        return model


def register():
    """Register config, quantizer and experts function with transformers (idempotent)."""
    if QUANT_METHOD not in AUTO_QUANTIZATION_CONFIG_MAPPING:
        register_quantization_config(QUANT_METHOD)(RW4Config)
    if QUANT_METHOD not in AUTO_QUANTIZER_MAPPING:
        register_quantizer(QUANT_METHOD)(RW4HfQuantizer)
    if QUANT_METHOD_RW8 not in AUTO_QUANTIZATION_CONFIG_MAPPING:
        register_quantization_config(QUANT_METHOD_RW8)(RW8Config)
    if QUANT_METHOD_RW8 not in AUTO_QUANTIZER_MAPPING:
        register_quantizer(QUANT_METHOD_RW8)(RW8HfQuantizer)
    ALL_EXPERTS_FUNCTIONS._global_mapping[QUANT_METHOD] = rw4_experts_forward


register()
