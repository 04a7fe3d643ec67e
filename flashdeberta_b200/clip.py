"""The global norm of a model's gradients, and clipping by it: two launches however many tensors there are.

The reference leaves this step of training to torch (its models are trained by transformers' Trainer over
src/flashdeberta/model.py:394-920), which launches over lists of tensors per type and keeps the norms of the single tensors.
"""
from __future__ import annotations

import array
import bisect
import ctypes as C
import math
from typing import Iterable, List, Optional, Sequence, Union

import torch

from . import _lib, ops
from .norms import TYPES

Tensors = Union[torch.Tensor, Iterable[torch.Tensor]]
_NORMS = {1.0: 1, 2.0: 2, math.inf: 0}


def _dense(t: torch.Tensor) -> bool:
    """Whether the elements fill one run of memory, in any order."""
    if t.is_contiguous():
        return True
    expect = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != expect:
            return False
        expect *= size
    return True


def _span(t: torch.Tensor):
    return t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()


def _apart(writes, reads=()) -> bool:
    """Whether runs of memory (from, to) that are written keep clear of one another and of those that are read."""
    writes = sorted(writes)
    if any(a[1] > b[0] for a, b in zip(writes, writes[1:])):
        return False
    starts = [w[0] for w in writes]
    for lo, hi in reads:
        i = bisect.bisect_left(starts, hi)  # runs from here on begin behind it
        if i and writes[i - 1][1] > lo:
            return False
    return True


def _run(grads: Sequence[torch.Tensor], outs: Optional[Sequence[torch.Tensor]], max_norm: float, norm_type: float, device) -> torch.Tensor:
    """One C call: the norm, and, with ``outs``, the scaled tensors."""
    table = array.array("q")
    for i, g in enumerate(grads):
        kind = TYPES[g.dtype]
        out = g if outs is None else outs[i]
        table.extend((g.data_ptr(), out.data_ptr(), g.numel(), kind | TYPES[out.dtype] << 32))  # fdb_grad_tensor
    norm = torch.empty((), dtype=torch.float32, device=device)
    p = _lib.ClipGradsParams(C.sizeof(_lib.ClipGradsParams), len(grads), table.buffer_info()[0], _NORMS[norm_type], int(outs is not None),
                             max_norm, norm.data_ptr(), None, 0)
    lib = _lib.load()
    with ops.on_device(device):
        need = lib.fdb_clip_grads_workspace_bytes(C.byref(p))
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device=device)
        p.workspace, p.workspace_bytes = ws.data_ptr(), need
        _lib.check(lib.fdb_clip_grads(C.byref(p), ops.raw_stream(device)))
    ops._launches += 2
    return norm


def _listed(grads: Tensors, what: str) -> List[torch.Tensor]:
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    for g in grads:
        if g.layout != torch.strided:
            raise TypeError(f"{what} takes dense tensors, not {g.layout}")
        if not g.is_cuda:
            raise RuntimeError("flashdeberta_b200 runs on CUDA devices only; there is no CPU path")
        if g.dtype not in TYPES:
            raise TypeError(f"{what} takes bfloat16, float16 or float32 tensors, not {g.dtype}")
        if g.device != grads[0].device:
            raise ValueError(f"{what} takes tensors of one device, got {grads[0].device} and {g.device}")
    return grads


def _norm_type(norm_type: float) -> float:
    norm_type = float(norm_type)
    if norm_type not in _NORMS:
        raise ValueError(f"norm_type must be 1, 2 or inf, not {norm_type}")
    return norm_type


@torch.no_grad()
def grad_norm(grads: Tensors, norm_type: float = 2.0) -> torch.Tensor:
    """The norm (1, 2 or inf) over all elements of the tensors taken as one vector: a float32 scalar on their device, zero where there
    are none.  Tensors are bfloat16, float16 or float32 in any mixture, of one device."""
    norm_type, grads = _norm_type(norm_type), _listed(grads, "grad_norm")
    if not grads:
        return torch.tensor(0.0)
    return _run([g if _dense(g) else g.contiguous() for g in grads], None, 0.0, norm_type, grads[0].device)


@torch.no_grad()
def clip_grads_(grads: Tensors, max_norm: float, *, norm_type: float = 2.0, out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Scales the tensors by ``min(1, max_norm / (norm + 1e-6))``, norm as in ``grad_norm``, in place, or into ``out`` (tensors of the same
    shapes, of any of the three types: an optimizer's float32 buffers beside bfloat16 gradients), and returns the norm before.  Nothing
    is read back to the host.  Where the factor is one, tensors scaled in place are not written.  The tensors that are written must not
    overlap one another or, but for a tensor that is its own output, those that are read."""
    norm_type, grads = _norm_type(norm_type), _listed(grads, "clip_grads_")
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative or NaN, got {max_norm}")
    outs = grads if out is None else _listed(out, "clip_grads_")
    if len(outs) != len(grads) or any(o is not g and o.shape != g.shape for g, o in zip(grads, outs)):
        raise ValueError("out must hold one tensor of the same shape for each gradient")
    if not grads:
        return torch.tensor(0.0)
    if outs[0].device != grads[0].device:
        raise ValueError(f"out is on {outs[0].device}, the gradients on {grads[0].device}")
    # the kernel goes through memory: a tensor that is no run of it, or is ordered unlike its output, is taken through a copy
    reads, writes, back, read_only = [], [], [], []
    for g, o in zip(grads, outs):
        if g.numel() == 0:
            continue
        if g is o or (g.data_ptr() == o.data_ptr() and g.stride() == o.stride()):
            if g.dtype != o.dtype:
                raise ValueError("a gradient cannot be scaled in place into another type")
            if _dense(g):
                reads.append(g)
                writes.append(g)
                continue
        elif _dense(g) and _dense(o) and g.stride() == o.stride():
            reads.append(g)
            writes.append(o)
            read_only.append(g)
            continue
        reads.append(g.contiguous())
        if reads[-1] is g:
            read_only.append(g)
        writes.append(o if o.is_contiguous() else torch.empty(o.shape, dtype=o.dtype, device=o.device))
        if writes[-1] is not o:
            back.append((o, writes[-1]))
    if not _apart(map(_span, writes), map(_span, read_only)):
        raise ValueError("the tensors that are written overlap one another or a gradient that is read")
    norm = _run(reads, writes, max_norm, norm_type, grads[0].device)
    for o, scaled in back:
        o.copy_(scaled)
    return norm


@torch.no_grad()
def clip_grad_norm_(parameters: Tensors, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """``torch.nn.utils.clip_grad_norm_`` over this package's kernels: the gradients of the parameters that have one are clipped in
    place to ``max_norm``; returns their norm before.  ``error_if_nonfinite`` reads the norm back to the host first (and raises before
    anything is scaled); without it nothing is read back."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else parameters
    grads = [p.grad for p in parameters if p.grad is not None]
    if error_if_nonfinite and grads:
        norm = grad_norm(grads, norm_type)
        if not math.isfinite(norm.item()):
            raise RuntimeError(f"the norm of order {norm_type} of the gradients is not finite, so they are not clipped")
    return clip_grads_(grads, max_norm, norm_type=norm_type)
