"""Residual norms: what lies between two blocks of a layer, in one pass, with its backward.

``ops.residual_norm`` covers the tails of transformers' DebertaV2SelfOutput / DebertaV2Output, which the reference's layer classes
keep (src/flashdeberta/model.py:259-272), and the other residual streams that encoders are built with: a norm after the block as
well, a gate per channel, per sequence or per element, a weighted residual, LayerNorm or RMSNorm.  Unlike ``ops.add_layernorm`` it
trains, takes every width up to 8192 and bf16, fp16 and fp32 rows.
"""
from __future__ import annotations

import struct
from typing import Optional, Tuple

import torch

from . import _lib, ops

TYPES = {torch.bfloat16: _lib.FDB_BF16, torch.float16: _lib.FDB_FP16, torch.float32: _lib.FDB_FP32}
MAX_HIDDEN = 8192


def _gate_rows(gate: torch.Tensor, shape) -> Optional[int]:
    """Rows of ``shape`` that share a row of the gate, or None where the gate's rows do not each cover one run of rows."""
    own = gate.shape
    if own[-1] != shape[-1]:
        return None
    own, lead = (1,) * (len(shape) - len(own)) + tuple(own[:-1]), shape[:-1]
    i = 0
    while i < len(lead) and own[i] == lead[i]:
        i += 1
    rows = 1
    for n, mine in zip(lead[i:], own[i:]):
        if mine != 1:
            return None
        rows *= n
    return rows


def _refusal(x, residual, weight, bias, post_weight, post_bias, gate, rms) -> Exception:
    """What is wrong with a call that ``_gate_of`` does not take."""
    shape, dtype = x.shape, x.dtype
    if not x.is_cuda:
        return RuntimeError("flashdeberta_b200 runs on CUDA devices only; there is no CPU path")
    if dtype not in TYPES:
        return TypeError(f"residual_norm takes bfloat16, float16 or float32 rows, not {dtype}")
    if len(shape) < 1 or not 1 <= shape[-1] <= MAX_HIDDEN:
        return ValueError(f"residual_norm takes rows of 1 to {MAX_HIDDEN} elements")
    if residual is not None and (residual.shape != shape or residual.dtype != dtype):
        return ValueError("residual must match x in shape and dtype")
    if rms and (bias is not None or post_bias is not None):
        return ValueError("the RMS norm takes no bias")
    if post_bias is not None and post_weight is None:
        return ValueError("post_bias needs post_weight")
    named = {"weight": weight, "bias": bias, "post_weight": post_weight, "post_bias": post_bias}
    for name, t in named.items():
        if t is not None and t.shape != shape[-1:]:
            return ValueError(f"{name} must have shape ({shape[-1]},), got {tuple(t.shape)}")
        if t is not None and (t.dtype != weight.dtype or t.dtype not in (dtype, torch.float32)):
            return TypeError(f"{name} must be {dtype} or float32, the norms' parameters all alike; got {t.dtype}")
    for name, t in {"residual": residual, **named, "gate": gate}.items():
        if t is not None and t.device != x.device:
            return ValueError(f"{name} is on {t.device}, x on {x.device}")
    if gate.dtype not in (dtype, torch.float32):
        return TypeError(f"gate must be {dtype} or float32, got {gate.dtype}")
    return ValueError(f"gate of shape {tuple(gate.shape)} does not broadcast to {tuple(shape)}")


def _gate_of(x, residual, weight, bias, post_weight, post_bias, gate, rms):
    """The gate as it is passed on (broadcast where it has to be); raises on what the operator does not take.  (Written for the calls that
    go through: on a single token the checks take as long as anything else.)"""
    shape, dtype, card, kind = x.shape, x.dtype, x.get_device(), weight.dtype
    vector = shape[-1:]
    if (card < 0 or dtype not in TYPES or len(shape) < 1 or not 1 <= shape[-1] <= MAX_HIDDEN
            or weight.shape != vector or weight.get_device() != card or (kind != dtype and kind != torch.float32)
            or (residual is not None and (residual.shape != shape or residual.dtype != dtype or residual.get_device() != card))):
        raise _refusal(x, residual, weight, bias, post_weight, post_bias, gate, rms)
    for t in (bias, post_weight, post_bias):
        if t is not None and (t.shape != vector or t.dtype != kind or t.get_device() != card):
            raise _refusal(x, residual, weight, bias, post_weight, post_bias, gate, rms)
    if (rms and (bias is not None or post_bias is not None)) or (post_bias is not None and post_weight is None):
        raise _refusal(x, residual, weight, bias, post_weight, post_bias, gate, rms)
    if gate is None:
        return None
    if (gate.dtype != dtype and gate.dtype != torch.float32) or gate.get_device() != card or gate.dim() > len(shape):
        raise _refusal(x, residual, weight, bias, post_weight, post_bias, gate, rms)
    if gate.shape != vector and (gate.dim() == 0 or _gate_rows(gate, shape) is None):  # shared in some other way: one per element then
        try:
            # (its gradient is summed where it is shared: of numbers that are not rounded before)
            return (gate.float() if gate.requires_grad and torch.is_grad_enabled() else gate).expand(shape)
        except RuntimeError:
            raise _refusal(x, residual, weight, bias, post_weight, post_bias, gate, rms) from None
    return gate


def _dense(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return t if t is None or t.is_contiguous() else t.contiguous()


def _address(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


# fdb_residual_norm_params and, behind it, what fdb_residual_norm_bwd_params adds: packed in one step (a ctypes structure of
# so many fields takes as long as the launch)
_FWD, _BWD = struct.Struct("@Ii10P2q4i2f"), struct.Struct("@Ii")
_BWD_TAIL = struct.Struct("@10PQ")


def _params(x, residual, weight, bias, post_weight, post_bias, gate, normed, stream, stats, eps, rms, residual_scale) -> bytes:
    """fdb_residual_norm_params over contiguous tensors."""
    shape, kind = x.shape, TYPES[x.dtype]
    rows = x.numel() // shape[-1]
    if gate is None:
        gate_at = gate_rows = gate_kind = 0
    else:
        gate_at, gate_rows, gate_kind = gate.data_ptr(), rows if gate.dim() == 1 else _gate_rows(gate, shape), TYPES[gate.dtype]
    return _FWD.pack(
        _FWD.size, kind, x.data_ptr(), 0 if residual is None else residual.data_ptr(), weight.data_ptr(), 0 if bias is None else bias.data_ptr(),
        0 if post_weight is None else post_weight.data_ptr(), 0 if post_bias is None else post_bias.data_ptr(), gate_at, normed.data_ptr(),
        0 if stream is None else stream.data_ptr(), 0 if stats is None else stats.data_ptr(), rows, gate_rows, shape[-1], TYPES[weight.dtype],
        gate_kind, rms, residual_scale, eps)


def _forward(x, residual, weight, bias, post_weight, post_bias, gate, eps, rms, residual_scale, keep):
    """(normed, stream, stats); the statistics where a backward will want them (``keep``), else None."""
    x, residual, weight, bias, post_weight, post_bias, gate = [
        t if t is None or t.is_contiguous() else t.contiguous() for t in (x, residual, weight, bias, post_weight, post_bias, gate)]
    normed, stream = torch.empty_like(x), torch.empty_like(x)
    stats = x.new_empty((x.numel() // x.shape[-1], 4), dtype=torch.float32) if keep else None
    if x.numel() == 0:
        return normed, stream, stats
    p = _params(x, residual, weight, bias, post_weight, post_bias, gate, normed, stream, stats, eps, rms, residual_scale)
    ops.call_on(x.device, _lib.load().fdb_residual_norm, p)
    ops._launches += 1
    return normed, stream, stats


def _backward(dnormed, dstream, x, residual, weight, bias, post_weight, post_bias, gate, stats, eps, rms, residual_scale, wanted):
    """Gradients of x, residual, weight, bias, post_weight, post_bias and gate; None where ``wanted`` is false."""
    tensors = [t if t is None or t.is_contiguous() else t.contiguous() for t in (x, residual, weight, bias, post_weight, post_bias, gate)]
    x = tensors[0]
    grads = [torch.empty_like(t) if w and t is not None else None for t, w in zip(tensors, wanted)]
    if x.numel() == 0 or (dnormed is None and dstream is None):
        return [None if g is None else g.zero_() for g in grads]
    dnormed, dstream = _dense(dnormed), _dense(dstream)
    dx = grads[0] if grads[0] is not None else torch.empty_like(x)
    lib, device = _lib.load(), x.device
    head = _BWD.pack(_BWD.size + _FWD.size + _BWD_TAIL.size, 0) + _params(*tensors, x, None, stats, eps, rms, residual_scale)
    addresses = (_address(dnormed), _address(dstream), dx.data_ptr(), *map(_address, grads[1:]))
    with ops.on_device(device):
        need = lib.fdb_residual_norm_bwd_workspace_bytes(head + _BWD_TAIL.pack(*addresses, 0, 0))
    ws = x.new_empty(need, dtype=torch.uint8)
    ops.call_on(device, lib.fdb_residual_norm_bwd, head + _BWD_TAIL.pack(*addresses, ws.data_ptr(), need))
    # (the gradient of a gate per element is no sum over rows)
    summed = any(g is not None for g in grads[2:6]) or (grads[6] is not None and (grads[6].numel() < x.numel() or x.numel() == x.shape[-1]))
    ops._launches += 1 + int(summed)
    return grads


@torch.library.custom_op("flashdeberta_b200::residual_norm", mutates_args=())
def residual_norm_op(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, bias: Optional[torch.Tensor],
                     post_weight: Optional[torch.Tensor], post_bias: Optional[torch.Tensor], gate: Optional[torch.Tensor], eps: float,
                     rms: bool, residual_scale: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(normed, stream, statistics) as one node for tracing; the statistics carry no gradient."""
    return _forward(x, residual, weight, bias, post_weight, post_bias, gate, eps, rms, residual_scale, True)


@residual_norm_op.register_fake
def _(x, residual, weight, bias, post_weight, post_bias, gate, eps, rms, residual_scale):
    rows = x.numel() // x.shape[-1]
    return x.new_empty(x.shape), x.new_empty(x.shape), x.new_empty((rows, 4), dtype=torch.float32)


@torch.library.custom_op("flashdeberta_b200::residual_norm_bwd", mutates_args=())
def residual_norm_bwd_op(dnormed: torch.Tensor, dstream: torch.Tensor, x: torch.Tensor, residual: Optional[torch.Tensor],
                         weight: torch.Tensor, bias: Optional[torch.Tensor], post_weight: Optional[torch.Tensor],
                         post_bias: Optional[torch.Tensor], gate: Optional[torch.Tensor], stats: torch.Tensor, eps: float, rms: bool,
                         residual_scale: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Every gradient of ``residual_norm_op``; an absent tensor gives an empty one."""
    grads = _backward(dnormed, dstream, x, residual, weight, bias, post_weight, post_bias, gate, stats, eps, rms, residual_scale, (True,) * 7)
    return tuple(x.new_empty(0) if g is None else g for g in grads)


@residual_norm_bwd_op.register_fake
def _(dnormed, dstream, x, residual, weight, bias, post_weight, post_bias, gate, stats, eps, rms, residual_scale):
    return tuple(x.new_empty(0) if t is None else t.new_empty(t.shape) for t in (x, residual, weight, bias, post_weight, post_bias, gate))


def _setup(ctx, inputs, output):
    *tensors, eps, rms, residual_scale = inputs
    ctx.save_for_backward(*tensors, output[2])
    ctx.norm_args = (eps, rms, residual_scale)


def _op_backward(ctx, dnormed, dstream, _):
    *tensors, stats = ctx.saved_tensors
    ops.refuse_tangents("the backward of residual_norm", (dnormed, dstream))
    x = tensors[0]
    dnormed, dstream = (torch.zeros_like(x) if g is None else g for g in (dnormed, dstream))
    grads = residual_norm_bwd_op(dnormed, dstream, *tensors, stats, *ctx.norm_args)
    return (*(None if t is None else g for t, g in zip(tensors, grads)), None, None, None)


residual_norm_op.register_autograd(_op_backward, setup_context=_setup)


class _ResidualNorm(torch.autograd.Function):
    """The training call outside tracing.  (forward takes ctx: with a setup_context of its own, torch binds the arguments to the
    signature on every call, which takes longer than the kernels of a short batch.)"""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, post_weight, post_bias, gate, eps, rms, residual_scale):
        normed, stream, stats = _forward(x, residual, weight, bias, post_weight, post_bias, gate, eps, rms, residual_scale, True)
        ctx.save_for_backward(x, residual, weight, bias, post_weight, post_bias, gate, stats)
        ctx.norm_args = (eps, rms, residual_scale)
        ctx.set_materialize_grads(False)
        return normed, stream

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dnormed, dstream):
        if ops.intercepted(dnormed, dstream) or any(g is not None and ops.batched(g) for g in (dnormed, dstream)):
            return _op_backward(ctx, dnormed, dstream, None)
        ops.refuse_tangents("the backward of residual_norm", (dnormed, dstream))
        grads = _backward(dnormed, dstream, *ctx.saved_tensors, *ctx.norm_args, ctx.needs_input_grad)
        return (*grads, None, None, None)


def residual_norm(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                  eps: float = 1e-7, *, rms: bool = False, post_weight: Optional[torch.Tensor] = None,
                  post_bias: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                  residual_scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """``stream = residual_scale * residual + gate * norm(x; post_weight, post_bias)`` and ``normed = norm(stream; weight, bias)``
    over the last dimension, one kernel forward and two backward.  Returns ``(normed, stream)``, both of x's shape and type.

    The norm is LayerNorm, or RMSNorm (no bias) with ``rms``; without ``post_weight`` the block's output x goes into the stream as it
    is.  ``gate`` broadcasts to x: (hidden,) a gate per channel, (batch, 1, hidden) one per sequence, x's shape one per element; None is
    a gate of one.  ``residual`` may be None.  Rows are bfloat16, float16 or float32; the norms' parameters are of that type or all
    float32, the gate of either.  Statistics and sums are float32, every result is rounded once (``normed`` is made of the stream
    before it is rounded).  Gradients of every input, in the inputs' types; no second derivative, and none in
    forward mode."""
    gate = _gate_of(x, residual, weight, bias, post_weight, post_bias, gate, rms)
    tensors = (x, residual, weight, bias, post_weight, post_bias, gate)
    eps, rms, residual_scale = float(eps), bool(rms), float(residual_scale)
    ops.refuse_tangents("residual_norm", tensors)
    if ops.intercepted(*tensors):
        return residual_norm_op(*tensors, eps, rms, residual_scale)[:2]
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return _ResidualNorm.apply(*tensors, eps, rms, residual_scale)
    return _forward(*tensors, eps, rms, residual_scale, False)[:2]
