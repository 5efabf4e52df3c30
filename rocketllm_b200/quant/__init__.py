"""RW4 quantization plugin surface: registry + backend, transformers quantizer, modules, converter.

Importing this package registers the ``rw4`` and ``rw8`` backends (``register_backend``), their
transformers quantization configs and quantizers, and the ``rw4`` experts implementation.
"""
from .registry import (COMPANION_SUFFIXES, PackedWeight, QuantBackend, TensorSpec, decision_table,
                       detect_backend, quant_method_of, register_backend, registered_backends)
from .rw4 import RW4Backend
from .rw8 import RW8Backend
from .modules import Int8Rows, RW4Linear, RW8Linear, rw4_experts_forward, rw4_experts_params
from .hf import (RW4Config, RW4HfQuantizer, RW8Config, RW8HfQuantizer, convert_modules,
                 convert_modules_rw8)
from .rw8_layers import fuse_rw8_layers

__all__ = ["COMPANION_SUFFIXES", "PackedWeight", "QuantBackend", "TensorSpec", "decision_table",
           "detect_backend", "quant_method_of", "register_backend", "registered_backends",
           "RW4Backend", "RW4Linear", "rw4_experts_forward", "rw4_experts_params", "RW4Config",
           "RW4HfQuantizer", "convert_modules", "RW8Backend", "Int8Rows", "RW8Linear", "RW8Config",
           "RW8HfQuantizer", "convert_modules_rw8", "fuse_rw8_layers"]
