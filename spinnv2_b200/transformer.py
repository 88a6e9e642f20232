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
Codes that a call allocates start their rows on 16-byte boundaries, whatever the width, which is what
linear_i8 reads fastest.  A wrong type raises TypeError, a wrong shape, device or stride ValueError, and a
code of the library Spkv2Error.
"""

from __future__ import annotations

import ctypes
import math
import struct

import torch

from .runtime import Spkv2Error, load_library

_DTYPES = {torch.float32: 1, torch.float16: 3, torch.bfloat16: 16}
_ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "silu": 2}

# The argument structs of spkv2_transformer.h, in native alignment.
_NORM = struct.Struct("@6P6qfi")
_CODES = struct.Struct("@3P4qii")
_LINEAR = struct.Struct("@6P6qii")
_CROSS = struct.Struct("@6P16q4ifi")

_FUNCTIONS: dict = {}


def _function(name: str):
    fn = _FUNCTIONS.get(name)
    if fn is None:
        fn = getattr(load_library(), name)
        fn.restype, fn.argtypes = ctypes.c_int, [ctypes.c_char_p, ctypes.c_void_p]
        _FUNCTIONS[name] = fn
    return fn


def _call(name: str, args: bytes, device: torch.device, stream) -> None:
    index = device.index
    if stream is None:
        stream = torch._C._cuda_getCurrentRawStream(index)
    elif not isinstance(stream, int):
        stream = stream.cuda_stream
    fn = _FUNCTIONS.get(name) or _function(name)
    if torch._C._cuda_getDevice() == index:
        code = fn(args, stream)
    else:
        with torch.cuda.device(index):
            code = fn(args, stream)
    if code != 0:
        text = load_library().spkv2_cuda_status_string(code)
        raise Spkv2Error(name.removeprefix("spkv2_cuda_"), code, text.decode() if text else "")


def _empty(shape, dtype, device, stream) -> torch.Tensor:
    """A new output, in the memory pool of the stream that writes it."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    ptr = stream if isinstance(stream, int) else stream.cuda_stream
    with torch.cuda.stream(torch.cuda.ExternalStream(ptr, device=device)):
        return torch.empty(shape, dtype=dtype, device=device)


def _empty_codes(shape, device, stream) -> torch.Tensor:
    pitch = (shape[-1] + 15) // 16 * 16
    return _empty((*shape[:-1], pitch), torch.int8, device, stream)[..., : shape[-1]]


def _rows(t: torch.Tensor, name: str) -> tuple[int, int, int]:
    """(rows, width, stride between rows) of [..., width], whose leading dims must be one list of rows."""
    if t.dim() == 2:
        rows, width = t.shape
        stride = t.stride(0)
    else:
        if t.dim() < 1:
            raise ValueError(f"{name}: expected [..., width], got a scalar")
        width = t.shape[-1]
        rows, stride = 1, 0
        for size, st in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
            if size == 1:
                continue
            if rows == 1:
                stride = st
            elif st != stride * rows:
                raise ValueError(f"{name}: leading dimensions are not evenly strided; call contiguous()")
            rows *= size
    if width > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    return rows, width, (stride if rows > 1 else width)


def _device(t: torch.Tensor, name: str) -> torch.device:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor, got one on {t.device}")
    return t.device


def _check(t, name: str, shape, dtype, device) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch tensor, got {type(t).__name__}")
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name}: expected a tensor on {device}, got one on {t.device}")
    if t.shape != shape:
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")


def _check_vector(t, name: str, size: int, dtype, device) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch tensor, got {type(t).__name__}")
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name}: expected a tensor on {device}, got one on {t.device}")
    if t.numel() != size or not t.is_contiguous():
        raise ValueError(f"{name}: expected {size} contiguous values, got {tuple(t.shape)}")


def _code(t: torch.Tensor, name: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{name}: expected float32, float16 or bfloat16, got {t.dtype}")
    return code


def rms_norm_i8(x, weight, residual=None, *, eps: float = 1e-6, out=None, scale_out=None, sum_out=None, stream=None):
    """(codes, scale, sum) of s = x + residual, y = s * weight / sqrt(mean(s^2) + eps), over the last dimension.

    codes [..., width] int8 and scale [...] float32 stand for y: scale = max|y| / 127, codes =
    round_half_even(y / scale).  sum is s in x's type; it is x itself where no residual is given, and with a
    residual it is written to sum_out (which may be x or residual: in place) or a new tensor.  A row that
    holds an infinity or a NaN has scale NaN and codes 0.
    """
    device = _device(x, "x")
    dtype = _code(x, "x")
    rows, width, x_stride = _rows(x, "x")
    _check_vector(weight, "weight", width, x.dtype, device)
    r_ptr = r_stride = s_ptr = s_stride = 0
    if residual is not None:
        _check(residual, "residual", x.shape, x.dtype, device)
        r_ptr, r_stride = residual.data_ptr(), _rows(residual, "residual")[2]
        if sum_out is None:
            sum_out = _empty(x.shape, x.dtype, device, stream)
    if sum_out is not None:
        _check(sum_out, "sum_out", x.shape, x.dtype, device)
        s_ptr, s_stride = sum_out.data_ptr(), _rows(sum_out, "sum_out")[2]
    if out is None:
        out = _empty_codes(x.shape, device, stream)
    else:
        _check(out, "out", x.shape, torch.int8, device)
    if scale_out is None:
        scale_out = _empty(x.shape[:-1], torch.float32, device, stream)
    else:
        _check_vector(scale_out, "scale_out", rows, torch.float32, device)
    _call("spkv2_cuda_rms_norm_i8",
          _NORM.pack(x.data_ptr(), r_ptr, weight.data_ptr(), s_ptr, out.data_ptr(), scale_out.data_ptr(), rows, width,
                     x_stride, r_stride, s_stride, _rows(out, "out")[2], eps, dtype), device, stream)
    return out, scale_out, (x if sum_out is None else sum_out)


def quantize_rows_i8(x, *, out=None, scale_out=None, stream=None):
    """(codes, scale) of x over its last dimension: scale = max|x| / 127, codes = round_half_even(x / scale).

    On activations [..., width] it gives what linear_i8 takes as (codes, scale); on a weight [channels,
    width] it gives linear_i8's weight and weight_scale.
    """
    device = _device(x, "x")
    dtype = _code(x, "x")
    rows, width, x_stride = _rows(x, "x")
    if out is None:
        out = _empty_codes(x.shape, device, stream)
    else:
        _check(out, "out", x.shape, torch.int8, device)
    if scale_out is None:
        scale_out = _empty(x.shape[:-1], torch.float32, device, stream)
    else:
        _check_vector(scale_out, "scale_out", rows, torch.float32, device)
    _call("spkv2_cuda_quantize_rows_i8",
          _CODES.pack(x.data_ptr(), out.data_ptr(), scale_out.data_ptr(), rows, width, x_stride, _rows(out, "out")[2],
                      dtype, 0), device, stream)
    return out, scale_out


def dequantize_rows_i8(codes, scale, dtype=torch.bfloat16, *, out=None, stream=None):
    """codes * scale, row by row, in `dtype` (or out's)."""
    device = _device(codes, "codes")
    if codes.dtype != torch.int8:
        raise TypeError(f"codes: expected torch.int8, got {codes.dtype}")
    rows, width, c_stride = _rows(codes, "codes")
    _check_vector(scale, "scale", rows, torch.float32, device)
    if out is None:
        out = _empty(codes.shape, dtype, device, stream)
    else:
        _check(out, "out", codes.shape, out.dtype, device)
    _call("spkv2_cuda_dequantize_rows_i8",
          _CODES.pack(codes.data_ptr(), scale.data_ptr(), out.data_ptr(), rows, width, c_stride, _rows(out, "out")[2],
                      _code(out, "out"), 0), device, stream)
    return out


def linear_i8(codes, scale, weight, weight_scale, *, bias=None, activation=None, dtype=torch.bfloat16, out=None,
              stream=None):
    """act(float(codes @ weight.T) * scale[..., None] * weight_scale + bias), in `dtype` (or out's).

    codes [..., k] and weight [n, k] are int8, scale [...], weight_scale [n] and bias [n] float32; the
    product is exact in 32 bits (k <= 131071).  activation: None, "relu" or "silu".
    """
    device = _device(codes, "codes")
    if codes.dtype != torch.int8:
        raise TypeError(f"codes: expected torch.int8, got {codes.dtype}")
    m, k, a_stride = _rows(codes, "codes")
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError("weight: expected a tensor [n, k]")
    n = weight.shape[0]
    _check(weight, "weight", (n, k), torch.int8, device)
    _check_vector(scale, "scale", m, torch.float32, device)
    _check_vector(weight_scale, "weight_scale", n, torch.float32, device)
    if bias is not None:
        _check_vector(bias, "bias", n, torch.float32, device)
    act = _ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation: expected None, 'relu' or 'silu', got {activation!r}")
    shape = (*codes.shape[:-1], n)
    if out is None:
        out = _empty(shape, dtype, device, stream)
    else:
        _check(out, "out", shape, out.dtype, device)
    _call("spkv2_cuda_linear_i8",
          _LINEAR.pack(codes.data_ptr(), scale.data_ptr(), weight.data_ptr(), weight_scale.data_ptr(),
                       0 if bias is None else bias.data_ptr(), out.data_ptr(), m, n, k, a_stride,
                       _rows(weight, "weight")[2], _rows(out, "out")[2], _code(out, "out"), act), device, stream)
    return out


def _heads(t: torch.Tensor, name: str) -> tuple[int, int, int]:
    """Strides of batch, token and head of [batch, tokens, heads, width]."""
    st = t.stride()
    if t.shape[3] > 1 and st[3] != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    return st[:3]


def cross_attention(q, k, v, *, lengths=None, key_mask=None, scale: float | None = None, out=None, stream=None):
    """softmax(scale * q k^T) v over the keys that count; q [batch, queries, heads, width], k and v [batch,
    keys, kv_heads, width] of q's type, heads a multiple of kv_heads, width at most 256.

    Key j of entry b counts if j < lengths[b] (int32 [batch]) and key_mask[b, j] (bool or uint8 [batch,
    keys]), where they are given.  What lies in keys and values that do not count has no influence, and a
    query without keys is answered with zeros.  scale: 1 / sqrt(width) by default.
    """
    device = _device(q, "q")
    dtype = _code(q, "q")
    if q.dim() != 4:
        raise ValueError(f"q: expected [batch, queries, heads, width], got {tuple(q.shape)}")
    batch, queries, heads, width = q.shape
    if not isinstance(k, torch.Tensor) or k.dim() != 4:
        raise ValueError("k: expected a tensor [batch, keys, kv_heads, width]")
    keys, kv_heads = k.shape[1], k.shape[2]
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"heads: {heads} query heads are not a multiple of {kv_heads} key heads")
    shape = (batch, keys, kv_heads, width)
    _check(k, "k", shape, q.dtype, device)
    _check(v, "v", shape, q.dtype, device)
    l_ptr = m_ptr = m_stride = 0
    if lengths is not None:
        _check_vector(lengths, "lengths", batch, torch.int32, device)
        l_ptr = lengths.data_ptr()
    if key_mask is not None:
        if isinstance(key_mask, torch.Tensor) and key_mask.dtype == torch.uint8:
            _check(key_mask, "key_mask", (batch, keys), torch.uint8, device)
        else:
            _check(key_mask, "key_mask", (batch, keys), torch.bool, device)
        if keys > 1 and key_mask.stride(1) != 1:
            raise ValueError("key_mask: the last dimension must be contiguous")
        m_ptr, m_stride = key_mask.data_ptr(), key_mask.stride(0)
    if scale is None:
        scale = 1.0 / math.sqrt(max(width, 1))
    if out is None:
        out = _empty(q.shape, q.dtype, device, stream)
    else:
        _check(out, "out", q.shape, q.dtype, device)
        if 0 in out.stride() and any(st == 0 and n > 1 for st, n in zip(out.stride(), out.shape)):
            raise ValueError("out: its elements must not overlap")
    _call("spkv2_cuda_cross_attention",
          _CROSS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), l_ptr, m_ptr, batch, queries, keys,
                      *_heads(q, "q"), *_heads(k, "k"), *_heads(v, "v"), *_heads(out, "out"), m_stride, heads, kv_heads,
                      width, dtype, scale, 0), device, stream)
    return out
