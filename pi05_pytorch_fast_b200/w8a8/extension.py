"""``pi05_w8a8::*`` PyTorch custom ops: schemas, fake implementations and the
Python functions around them.  The bodies are C++ (``_w4a4_ops.so``, built from
``csrc/torch_ops8.cpp``) on the kernels of ``libw4a4_sm100.so``.  There is no
CPU path: CPU tensors raise, missing libraries raise.

Ops run on the current stream of their tensors' device; what they allocate
comes from torch's caching allocator on that stream, and nothing synchronises.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _native as nat
from ..w4a4 import extension as _w4a4

CACHE_BLOCK = nat.KV8_BLOCK  # cache tokens that share a scale


def _code_stride(h: int) -> int:
    """Row stride of codes: a multiple of 128 bytes, or of 16 for short rows."""
    return (h + 15) // 16 * 16 if h <= 128 else (h + 127) // 128 * 128


def _fake_codes(x: torch.Tensor) -> torch.Tensor:
    ld = _code_stride(x.shape[-1])
    if ld == x.shape[-1]:
        return torch.empty(x.shape, dtype=torch.int8, device=x.device)
    stride, step = [1], ld
    for n in reversed(x.shape[:-1]):
        stride.insert(0, step)
        step *= n
    return torch.empty_strided(x.shape, stride, dtype=torch.int8, device=x.device)


def _fake_scale(x: torch.Tensor) -> torch.Tensor:
    return torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)


def _fake_rms_norm_quant(x, gain, eps, delta=None, gate=None, shift=None):
    total = torch.empty(x.shape if delta is not None else (0,), dtype=x.dtype, device=x.device)
    return _fake_codes(x), _fake_scale(x), total


def _fake_kv_values(k, v, ks, vs, lengths, dtype):
    return torch.empty(k.shape, dtype=dtype, device=k.device), torch.empty(k.shape, dtype=dtype, device=k.device)


# name, schema arguments / returns, fake implementation
_OPS = (
    ("rms_norm_quant",
     "(Tensor x, Tensor gain, float eps, Tensor? delta=None, Tensor? gate=None, Tensor? shift=None)"
     " -> (Tensor, Tensor, Tensor)", _fake_rms_norm_quant),
    ("quantize", "(Tensor x, Tensor? up=None) -> (Tensor, Tensor)",
     lambda x, up=None: (_fake_codes(x), _fake_scale(x))),
    ("dequantize", "(Tensor codes, Tensor scale, ScalarType dtype) -> Tensor",
     lambda codes, scale, dtype: torch.empty(codes.shape, dtype=dtype, device=codes.device)),
    ("linear",
     "(Tensor codes, Tensor scale, Tensor weight, Tensor weight_scale, Tensor? bias, ScalarType dtype) -> Tensor",
     lambda codes, scale, weight, weight_scale, bias, dtype: torch.empty(
         *codes.shape[:-1], weight.shape[0], dtype=dtype, device=codes.device)),
    ("kv_append",
     "(Tensor(a!) keys, Tensor(b!) values, Tensor(c!) key_scale, Tensor(d!) value_scale, Tensor k, Tensor v,"
     " Tensor start, Tensor? valid=None) -> Tensor",
     lambda keys, values, key_scale, value_scale, k, v, start, valid=None: torch.empty_like(start)),
    ("kv_values",
     "(Tensor keys, Tensor values, Tensor key_scale, Tensor value_scale, Tensor lengths, ScalarType dtype)"
     " -> (Tensor, Tensor)", _fake_kv_values),
    ("kv_attention",
     "(Tensor q, Tensor keys, Tensor values, Tensor key_scale, Tensor value_scale, Tensor lengths, bool causal,"
     " float scale) -> Tensor",
     lambda q, keys, values, key_scale, value_scale, lengths, causal, scale: torch.empty(
         q.shape, dtype=q.dtype, device=q.device)),
)

# kept alive for the life of the process
_library = torch.library.Library("pi05_w8a8", "DEF")
for _name, _schema, _fake in _OPS:
    _library.define(_name + _schema)
    torch.library.register_fake("pi05_w8a8::" + _name, _fake, lib=_library)
_ops = {name: getattr(torch.ops.pi05_w8a8, name).default for name, _, _ in _OPS}


def _call(name: str, *args):
    if not _w4a4._ops_loaded and not _w4a4._load_ops():
        _w4a4._not_built()
    return _ops[name](*args)


class Int8Weight(NamedTuple):
    """A Linear weight in 8 bits: codes int8 [N, K] (rows that begin at
    multiples of 16 bytes) and one scale fp32 [N] for each output channel."""

    codes: torch.Tensor
    scale: torch.Tensor


class KVCache8(NamedTuple):
    """Keys and values int8 [batch, capacity, heads, width] (width 64, 128 or
    256) and their scales fp32 [batch, heads, capacity / 16].  How many
    tokens of each sequence are filled is the caller's: an int32 tensor
    [batch] on the device, given to and returned by ``kv_append``."""

    keys: torch.Tensor
    values: torch.Tensor
    key_scale: torch.Tensor
    value_scale: torch.Tensor

    @classmethod
    def allocate(cls, batch: int, capacity: int, heads: int, width: int, device, *, clear: bool = True) -> "KVCache8":
        """An empty cache; the capacity is rounded up to a multiple of 16.
        ``clear=False`` leaves its memory as it is, which no result of the
        operators depends on: they use no slot from the length on, and no scale
        of a block that has none below it."""
        capacity = (capacity + CACHE_BLOCK - 1) // CACHE_BLOCK * CACHE_BLOCK
        make = torch.zeros if clear else torch.empty
        codes = make((2, batch, capacity, heads, width), dtype=torch.int8, device=device)
        scale = make((2, batch, heads, capacity // CACHE_BLOCK), dtype=torch.float32, device=device)
        return cls(codes[0], codes[1], scale[0], scale[1])


def rms_norm_quant(x: torch.Tensor, gain: torch.Tensor, eps: float = 1e-6, *, delta: torch.Tensor | None = None,
                   gate: torch.Tensor | None = None, shift: torch.Tensor | None = None):
    """Residual addition, RMSNorm and 8-bit codes in one pass over x [..., h]:
    total = x + gate * delta; y = total * rsqrt(mean(total^2) + eps) * gain +
    shift; scale = amax|y| * fl(1 / 127) per row; codes = rint(y / scale).

    x and delta (the sublayer's output) fp16, bf16 or fp32 of one shape; gain
    and shift fp32, gate of x's dtype, each [h], or [batch, h] for x [batch,
    ..., h] (Gemma's norm: gain = 1 + weight; pi0.5's adaptive norm: gain = 1 +
    scale, shift and gate of the time condition).  The norm is taken of the
    fp32 sum; ``total`` is its rounding to x's dtype.

    Returns (codes int8 like x, scale fp32 [...], total); without delta, total
    is x itself."""
    codes, scale, total = _call("rms_norm_quant", x, gain, eps, delta, gate, shift)
    return codes, scale, x if delta is None else total


def quantize(x: torch.Tensor, up: torch.Tensor | None = None):
    """8-bit codes of the rows of x [..., h] (fp16, bf16, fp32), or with ``up``
    of gelu_tanh(x) * up (the input of a GeGLU's down projection; x and up may
    be the halves of one product).  Returns (codes int8 like x, scale fp32
    [...]): scale = amax * fl(1 / 127), codes = rint(value / scale) in fp32."""
    return _call("quantize", x, up)


def dequantize(codes: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """codes [..., h] times their row's scale, rounded once to dtype."""
    return _call("dequantize", codes, scale, dtype)


def pack_weight(weight: torch.Tensor) -> Int8Weight:
    """A Linear weight [N, K] (fp16, bf16, fp32; on the GPU) as int8 codes with
    one scale for each output channel, laid out for ``linear``."""
    if weight.dim() != 2:
        raise RuntimeError(f"pack_weight expects a weight [N, K], got {tuple(weight.shape)}")
    return Int8Weight(*quantize(weight.detach()))


def linear(codes: torch.Tensor, scale: torch.Tensor, weight: Int8Weight, *, bias: torch.Tensor | None = None,
           dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """y = (codes @ weight.codes^T) * scale * weight.scale + bias: int8 x int8
    products with exact int32 sums, scaled in fp32 and rounded once to dtype
    (fp16, bf16, fp32; bias of the same dtype).  codes [..., K] and scale [...]
    as ``quantize`` / ``rms_norm_quant`` give them.  Returns y [..., N]."""
    return _call("linear", codes, scale, weight.codes, weight.scale, bias, dtype)


def kv_append(cache: KVCache8, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor, *,
              valid: torch.Tensor | None = None) -> torch.Tensor:
    """Writes new keys and values [batch, tokens, heads, width] (fp16 or bf16,
    any strides of batch, token and head) into the cache from slot start[b] on,
    those with ``valid`` [batch, tokens] (bool) False left out, the others
    without gaps.  Returns the new lengths int32 [batch].

    Each block of 16 slots and head has one scale, amax / 127 of its tokens.  A
    block that already holds earlier tokens keeps its scale unless the new ones
    need a larger one; the earlier codes are then rounded again to it.  Tokens
    past the capacity are dropped and a start outside the cache writes nothing;
    both are reported by ``_native.device_error`` (ERR_CACHE_FULL)."""
    return _call("kv_append", cache.keys, cache.values, cache.key_scale, cache.value_scale, k, v, start, valid)


def kv_values(cache: KVCache8, lengths: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
    """The keys and values that the cache stands for, [batch, capacity, heads,
    width] of dtype, zero from lengths[b] on."""
    return _call("kv_values", cache.keys, cache.values, cache.key_scale, cache.value_scale, lengths, dtype)


def kv_attention(q: torch.Tensor, cache: KVCache8, lengths: torch.Tensor, *, causal: bool = False,
                 softmax_scale: float | None = None) -> torch.Tensor:
    """softmax(q k^T * softmax_scale) v over the first lengths[b] tokens of the
    cache, for q [batch, tokens, q_heads, width] (fp16 or bf16; q_heads a
    multiple of the cache's heads, consecutive query heads sharing one).
    ``causal``: the queries are the cache's last tokens, and each sees the
    tokens up to its own.  softmax_scale defaults to width ** -0.5.  A query
    that sees no token gives zeros.  Returns a tensor like q."""
    scale = q.shape[-1] ** -0.5 if softmax_scale is None else softmax_scale
    return _call("kv_attention", q, cache.keys, cache.values, cache.key_scale, cache.value_scale, lengths, causal, scale)
