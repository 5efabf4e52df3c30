"""The RW8 quant backend: 8-bit weights with one scale per output channel, multiplied by activations
that are quantized per token as they are produced (W8A8).

A logical weight ``X.weight`` is stored as two checkpoint tensors (the companion-suffix convention
of ``rocketllm/quant/registry.py:33``):

    X.weight         int8  [N, K]
    X.weight_scale   fp32  [N, 1]     value = code * scale

the tensors of a channel-wise ``int-quantized`` compressed-tensors checkpoint (whose config still has
to say ``quant_method: "rw8"``: nothing else selects this backend), which the reference
expands to a bf16 scratch copy on every fetch (``rocketllm/quant/safetensors_quant.py:244-293``).
Here ``needs_scratch`` is False: the library multiplies the codes as they are.
"""
import torch

from .registry import QuantBackend, register_backend


@register_backend
class RW8Backend(QuantBackend):
    format = "rw8"
    quant_methods = ("rw8",)
    PAYLOAD_SUFFIXES = ()

    @classmethod
    def example_config(cls):
        return {"quant_method": "rw8", "bits": 8}

    def bits(self, weight):
        return 8 if weight.payload.dtype == torch.int8 else super().bits(weight)

    def logical_shape(self, weight):
        p = weight.payload
        return tuple(p.shape) if p.dtype == torch.int8 else None

    def needs_scratch(self, weight):
        """Never: the library computes on the 8-bit weight (no dequant-to-scratch)."""
        return False

    def decision(self):
        from .. import _lib
        try:
            _lib.lib()
            available, reason = True, "librw4.so loaded: 8-bit tcgen05 products on packed weights"
        except RuntimeError as exc:
            available, reason = False, str(exc)
        return {"format": self.format, "capability": "rw8 sm_100a kernels (librw4.so)",
                "available": available, "path": "fused_packed" if available else "unavailable",
                "reason": reason}
