"""The 8-bit linear layer: weights held in 8-bit integers with a scale per output channel, tokens rounded to 8 bits one by one.

No counterpart in the reference, whose layers run transformers' dense modules (src/flashdeberta/model.py:259-272); this is
the 8-bit form of what ``ops.linear_gelu`` does in bf16.  Forward only.
"""
from __future__ import annotations

import struct
from typing import Optional, Tuple

import torch

from . import _lib, ops
from .norms import TYPES

MAX_IN_FEATURES = 131071  # products of two 8-bit integers that a 32-bit sum holds
MAX_COLS = 1 << 30        # of a row that quantize_int8 takes


def _pitch(cols: int) -> int:
    """Bytes between rows: 16-byte pieces, and whole lines of memory where a row is longer than one (a tile's 128 bytes of a row would
    lie on two otherwise)."""
    return (cols + 127) // 128 * 128 if cols > 128 else (cols + 15) // 16 * 16


def int8_rows(t: torch.Tensor) -> torch.Tensor:
    """An int8 matrix (..., cols) in the layout the kernels read: rows that start on 16 bytes.  The tensor itself where it has
    it; else a copy, which a program that keeps a weight makes once."""
    if t.dtype != torch.int8 or t.dim() < 1:
        raise TypeError("int8_rows takes an int8 tensor of rows")
    if _rows(t) is not None:
        return t
    out = torch.empty(*t.shape[:-1], _pitch(t.shape[-1]), dtype=torch.int8, device=t.device)[..., :t.shape[-1]]
    out.copy_(t)
    return out


def _rows(t: torch.Tensor):
    """(address, pitch) of a matrix whose rows start on 16 bytes, else None."""
    shape, strides, at = t.shape, t.stride(), t.data_ptr()
    cols = shape[-1]
    if at % 16 != 0 or (strides[-1] != 1 and cols > 1):
        return None
    pitch = inner = None
    for n, s in zip(shape[-2::-1], strides[-2::-1]):  # the leading dimensions as one
        if n == 1:
            continue
        if pitch is None:
            pitch = s
        elif s != inner:
            return None
        inner = n * s
    if pitch is None:  # one row: any will do
        return at, _pitch(cols)
    # (an expanded dimension has a stride of zero: no pitch, and nothing that further dimensions could go on from)
    return (at, pitch) if pitch % 16 == 0 and pitch >= cols else None


def quantize_int8(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows as 8-bit integers with a scale each: ``scale = amax / 127``, ``q = round(x * (127 / amax))``, ties to even, in float32.  x:
    (..., cols) bfloat16, float16 or float32; returns int8 of x's shape (rows start on 16 bytes) and float32 of shape ``x.shape[:-1]``.
    The same call scales the tokens of an activation and the output channels of a weight.  Rows of zeros (or below 2^-100) have scale
    zero; rows with an infinity or NaN have integers zero and a scale that makes NaN of whatever is multiplied by it.
    No gradient is recorded; rows have at most 2^30 elements."""
    if not x.is_cuda:
        raise RuntimeError("flashdeberta_b200 runs on CUDA devices only; there is no CPU path")
    if x.dtype not in TYPES:
        raise TypeError(f"quantize_int8 takes bfloat16, float16 or float32, not {x.dtype}")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_COLS:
        raise ValueError(f"quantize_int8 takes rows of 1 to {MAX_COLS} elements")
    if ops.intercepted(x):
        raise RuntimeError("quantize_int8 goes by the memory of plain tensors: call it outside tracing, or linear_int8, which rounds within")
    ops.refuse_tangents("quantize_int8", (x,))
    cols = x.shape[-1]
    x = x if x.is_contiguous() else x.contiguous()
    q = torch.empty(*x.shape[:-1], _pitch(cols), dtype=torch.int8, device=x.device)[..., :cols]
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    if scale.numel() == 0:
        return q, scale
    with ops.on_device(x.device):
        _lib.check(_lib.load().fdb_quantize_int8(x.data_ptr(), TYPES[x.dtype], scale.numel(), cols, q.data_ptr(), _pitch(cols),
                                                 scale.data_ptr(), ops.raw_stream(x.device)))
    ops._launches += 1
    return q, scale


@torch.library.custom_op("flashdeberta_b200::linear_int8", mutates_args=())
def linear_int8_op(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor],
                   x_scale: Optional[torch.Tensor], gelu: bool, out_dtype: torch.dtype) -> torch.Tensor:
    return _call(x, weight, weight_scale, bias, x_scale, gelu, out_dtype)


@linear_int8_op.register_fake
def _(x, weight, weight_scale, bias, x_scale, gelu, out_dtype):
    return x.new_empty((*x.shape[:-1], weight.shape[0]), dtype=out_dtype)


_PARAMS, _PARAMS_TAIL = struct.Struct("@IiPqPPqPPPq6iPQP"), struct.Struct("@PQP")  # fdb_linear_int8_params, its last three fields


def _call(x, weight, weight_scale, bias, x_scale, gelu, out_dtype):
    shape, n, device = x.shape, weight.shape[0], x.device
    out = x.new_empty((*shape[:-1], n), dtype=out_dtype)
    if out.numel() == 0:
        return out
    if not weight_scale.is_contiguous():
        weight_scale = weight_scale.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    w = _rows(weight)
    if w is None:
        weight = int8_rows(weight)
        w = _rows(weight)
    rows, k = out.numel() // n, shape[-1]
    lib = _lib.load()
    if x_scale is None:
        x = x if x.is_contiguous() else x.contiguous()
        x_at, x_pitch, kind, scale_at = x.data_ptr(), 0, TYPES[x.dtype], 0
    else:
        x_scale = x_scale if x_scale.is_contiguous() else x_scale.contiguous()
        x = int8_rows(x)
        (x_at, x_pitch), kind, scale_at = _rows(x), _lib.FDB_INT8, x_scale.data_ptr()
    status = ops._status_word(device).data_ptr()
    p = _PARAMS.pack(
        _PARAMS.size, kind, x_at, x_pitch, scale_at, w[0], w[1], weight_scale.data_ptr(), 0 if bias is None else bias.data_ptr(),
        out.data_ptr(), rows, k, n, 0 if bias is None else TYPES[bias.dtype], TYPES[out_dtype], gelu, 0, 0, 0, status)
    need = lib.fdb_linear_int8_workspace_bytes(p)
    if need:  # the tokens as integers
        ws = x.new_empty(need + 255, dtype=torch.uint8)
        p = p[:-_PARAMS_TAIL.size] + _PARAMS_TAIL.pack((ws.data_ptr() + 255) & ~255, need, status)
    ops.call_on(device, lib.fdb_linear_int8, p)
    ops._launches += 1 + int(need > 0)
    return out


def linear_int8(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                x_scale: Optional[torch.Tensor] = None, gelu: bool = False, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``act(x_scale * weight_scale * (x @ weight.T) + bias)`` in 8-bit integers (``fdb_linear_int8``), act the identity or the erf GELU.

    weight: int8 (out_features, in_features) and weight_scale: float32 (out_features), as ``quantize_int8`` of a linear layer's weight
    gives them.  x: (..., in_features), bfloat16, float16 or float32, rounded to 8 bits token by token within the call as
    ``quantize_int8`` does; or int8 with its ``x_scale``, float32 of shape ``x.shape[:-1]``.  bias: of the output's type or float32.
    The sum is exact (in_features up to 131071), the rest float32, rounded once to ``out_dtype`` (x's type, or bfloat16 for int8).
    int8 rows that do not start on 16 bytes are copied first (``int8_rows`` does that once for a weight).  Forward only."""
    if not x.is_cuda:
        raise RuntimeError("flashdeberta_b200 runs on CUDA devices only; there is no CPU path")
    if ops.wants_grad(x, weight_scale, bias, x_scale):
        raise RuntimeError("the 8-bit linear layer is forward-only; call under torch.no_grad() or detach the inputs")
    ops.refuse_tangents("the 8-bit linear layer", (x, weight_scale, bias, x_scale))
    if weight.dtype != torch.int8 or weight.dim() != 2 or weight_scale.dtype != torch.float32 or weight_scale.shape != weight.shape[:1]:
        raise ValueError("weight must be int8 (out_features, in_features) with float32 weight_scale (out_features,)")
    if x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x of shape {tuple(x.shape)} does not fit a weight of shape {tuple(weight.shape)}")
    if not 1 <= weight.shape[1] <= MAX_IN_FEATURES or weight.shape[0] < 1:
        raise ValueError(f"linear_int8 takes 1 to {MAX_IN_FEATURES} in_features and at least one out_feature")
    if (x_scale is None) != (x.dtype in TYPES) or (x_scale is not None and x.dtype != torch.int8):
        raise TypeError("x must be bfloat16, float16 or float32, or int8 with x_scale")
    if x_scale is not None and (x_scale.dtype != torch.float32 or x_scale.shape != x.shape[:-1]):
        raise ValueError(f"x_scale must be float32 of shape {tuple(x.shape[:-1])}")
    if out_dtype is None:
        out_dtype = x.dtype if x_scale is None else torch.bfloat16
    if out_dtype not in TYPES:
        raise TypeError(f"out_dtype must be bfloat16, float16 or float32, not {out_dtype}")
    if bias is not None and (bias.shape != weight.shape[:1] or bias.dtype not in (out_dtype, torch.float32)):
        raise ValueError(f"bias must be ({weight.shape[0]},), {out_dtype} or float32")
    for name, t in (("weight", weight), ("weight_scale", weight_scale), ("bias", bias), ("x_scale", x_scale)):
        if t is not None and t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    call = linear_int8_op if ops.intercepted(x, weight, weight_scale, bias, x_scale) else _call
    return call(x, weight, weight_scale, bias, x_scale, bool(gelu), out_dtype)
