"""8-bit serving operators on the B200: activations, weights and the key/value
cache as int8 codes with fp32 scales.

* ``rms_norm_quant``  residual addition + (adaptive) RMSNorm -> 8-bit codes
* ``quantize`` / ``dequantize``  rows to 8-bit codes (plain, or of the GeGLU
  product) and back
* ``pack_weight`` / ``linear``   int8 x int8 matrix product with a scale for
  each token and output channel
* ``KVCache8``, ``kv_append``, ``kv_values``, ``kv_attention``  a cache in 8
  bits with a scale for each block of 16 tokens and head, and attention over it

Importing registers the ``pi05_w8a8::*`` custom ops (bodies in C++,
``csrc/torch_ops8.cpp``).  Inference only: no op has a gradient.  An input (scales,
gain, shift, gate and bias as well) that requires one is refused outside
``torch.no_grad()``, one with a forward-mode tangent everywhere.
"""

from .extension import (
    Int8Weight,
    KVCache8,
    dequantize,
    kv_append,
    kv_attention,
    kv_values,
    linear,
    pack_weight,
    quantize,
    rms_norm_quant,
)

__all__ = [
    "Int8Weight",
    "KVCache8",
    "dequantize",
    "kv_append",
    "kv_attention",
    "kv_values",
    "linear",
    "pack_weight",
    "quantize",
    "rms_norm_quant",
]
