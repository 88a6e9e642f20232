"""Operators of an INT8 decoder layer on torch CUDA tensors (include/spkv2_transformer.h).

The graph runtime (spinnv2_b200.runtime) leaves an image's features on the device; these calls are what a
decoder that reads them needs next to it:

  rms_norm_i8         residual addition, root-mean-square norm, int8 codes and a scale for each token
  quantize_rows_i8    int8 codes and a scale for each row (activations, or a weight's output channels)
  dequantize_rows_i8  the values that codes stand for
  linear_i8           int8 product with a scale for each token and channel, bias and activation
  cross_attention     attention to an encoder's keys and values of another length

Each call launches on `stream` (a cudaStream_t as an int, or an object with `cuda_stream`; default: torch's
current stream of the tensors' device) and returns at once.  Outputs are allocated unless they are given.
A tensor used on another stream than its own has to live until that stream is done with it
(Tensor.record_stream), as in any torch call.  The calls are for inference: what they answer carries no
gradient, also where an argument requires one.  Codes that a call allocates start their rows on 16-byte boundaries, whatever the width, which is what
linear_i8 reads fastest.  A wrong type raises TypeError, a wrong shape, device or stride ValueError, and a
code of the library Spkv2Error.  The checks run in the compiled binding (binding/torch_ops.cpp): a call
takes about a microsecond more than the launch.
"""

from __future__ import annotations

import ctypes

import torch

from .runtime import Spkv2Error, load_library

try:
    from ._lib import _torch_ops as _ops
except ImportError as e:
    raise ImportError("spinnv2_b200/_lib/_torch_ops.so is not built for this torch; run __graft_entry__.build()") from e


def _bind() -> None:
    lib = load_library()
    names = ("spkv2_cuda_rms_norm_i8", "spkv2_cuda_quantize_rows_i8", "spkv2_cuda_dequantize_rows_i8",
             "spkv2_cuda_linear_i8", "spkv2_cuda_cross_attention", "spkv2_cuda_status_string")
    _ops.bind(*(ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in names), Spkv2Error)


_bind()

_ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "silu": 2}


def rms_norm_i8(x, weight, residual=None, *, eps: float = 1e-6, out=None, scale_out=None, sum_out=None, stream=None):
    """(codes, scale, sum) of s = x + residual, y = s * weight / sqrt(mean(s^2) + eps), over the last dimension.

    codes [..., width] int8 and scale [...] float32 stand for y: scale = max|y| / 127, codes =
    round_half_even(y / scale).  sum is s in x's type; it is x itself where no residual is given, and with a
    residual it is written to sum_out (which may be x or residual: in place) or a new tensor.  A row that
    holds an infinity or a NaN has scale NaN and codes 0.
    """
    return _ops.rms_norm_i8(x, weight, residual, eps, out, scale_out, sum_out, stream)


def quantize_rows_i8(x, *, out=None, scale_out=None, stream=None):
    """(codes, scale) of x over its last dimension: scale = max|x| / 127, codes = round_half_even(x / scale).

    On activations [..., width] it gives what linear_i8 takes as (codes, scale); on a weight [channels,
    width] it gives linear_i8's weight and weight_scale.
    """
    return _ops.quantize_rows_i8(x, out, scale_out, stream)


def dequantize_rows_i8(codes, scale, dtype=torch.bfloat16, *, out=None, stream=None):
    """codes * scale, row by row, in `dtype` (or out's)."""
    return _ops.dequantize_rows_i8(codes, scale, dtype, out, stream)


def linear_i8(codes, scale, weight, weight_scale, *, bias=None, activation=None, dtype=torch.bfloat16, out=None,
              stream=None):
    """act(float(codes @ weight.T) * scale[..., None] * weight_scale + bias), in `dtype` (or out's).

    codes [..., k] and weight [n, k] are int8, scale [...], weight_scale [n] and bias [n] float32; the
    product is exact in 32 bits (k <= 131071).  activation: None, "relu" (which keeps a NaN) or "silu".
    """
    act = _ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation: expected None, 'relu' or 'silu', got {activation!r}")
    return _ops.linear_i8(codes, scale, weight, weight_scale, bias, act, dtype, out, stream)


def cross_attention(q, k, v, *, lengths=None, key_mask=None, scale: float | None = None, out=None, stream=None):
    """softmax(scale * q k^T) v over the keys that count; q [batch, queries, heads, width], k and v [batch,
    keys, kv_heads, width] of q's type, heads a multiple of kv_heads, width at most 256.

    Key j of entry b counts if j < lengths[b] (int32 [batch]) and key_mask[b, j] (bool or uint8 [batch,
    keys]), where they are given.  What lies in keys and values that do not count has no influence, and a
    query without keys is answered with zeros.  scale: 1 / sqrt(width) by default.  In 16-bit types each
    probability is rounded to the type before it meets its value.
    """
    return _ops.cross_attention(q, k, v, lengths, key_mask, scale, out, stream)


def check(device=None) -> None:
    """Waits for the device's work and raises Spkv2Error if a kernel of these calls gave up a bounded wait
    since the last check (its outputs are then incomplete)."""
    with torch.cuda.device(device):
        code = ctypes.c_int(0)
        rc = load_library().spkv2_cuda_transformer_status(ctypes.byref(code))
    if rc != 0:
        raise Spkv2Error(f"wait (code {code.value})", rc, load_library().spkv2_cuda_status_string(rc).decode())
