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


_at, _count, _size, _whole, _card = (
    torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.element_size, torch.Tensor.is_contiguous, torch.Tensor.get_device)


def _run(grads: Sequence[torch.Tensor], outs: Optional[Sequence[torch.Tensor]], max_norm: float, norm_type: float) -> torch.Tensor:
    """One C call: the norm, and, with ``outs``, the scaled tensors.  All are runs of memory."""
    table = array.array("q", bytes(32 * len(grads)))  # rows of fdb_grad_tensor: two addresses, the count, both types
    at, count, kinds = list(map(_at, grads)), list(map(_count, grads)), [TYPES[g.dtype] for g in grads]
    to, into = at, kinds
    if outs is not None and outs is not grads:
        to, into = list(map(_at, outs)), [TYPES[o.dtype] for o in outs]
        own = [a == b for a, b in zip(at, to)]
        if any(i and a != b for i, a, b in zip(own, kinds, into)):
            raise ValueError("a gradient cannot be scaled in place into another type")
    if outs is not None:
        ends = [a + n * s for a, n, s in zip(to, count, map(_size, outs))]
        more = [] if outs is grads else [(a, a + n * s) for a, n, s, i in zip(at, count, map(_size, grads), own) if not i]
        # runs of memory are apart where each ends, in order, before the next begins
        if any(a > b for a, b in zip(sorted(ends + [hi for _, hi in more]), sorted(to + [lo for lo, _ in more])[1:])) and not _apart(zip(to, ends), more):
            raise ValueError("the tensors that are written overlap one another or a gradient that is read")
    table[0::4], table[1::4], table[2::4] = array.array("q", at), array.array("q", to), array.array("q", count)
    table[3::4] = array.array("q", [a | b << 32 for a, b in zip(kinds, into)])
    device, lib = grads[0].device, _lib.load()
    norm = torch.empty((), dtype=torch.float32, device=device)
    p = _lib.ClipGradsParams(C.sizeof(_lib.ClipGradsParams), len(grads), table.buffer_info()[0], _NORMS[norm_type], int(outs is not None),
                             max_norm, norm.data_ptr(), None, 0)
    with ops.on_device(device):
        need = lib.fdb_clip_grads_workspace_bytes(C.byref(p))
        ws = norm.new_empty(max(need, 16), dtype=torch.uint8)
        p.workspace, p.workspace_bytes = ws.data_ptr(), need
        _lib.check(lib.fdb_clip_grads(C.byref(p), ops.raw_stream(device)))
    ops._launches += 2
    return norm


def _listed(grads: Tensors, what: str) -> List[torch.Tensor]:
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    if any(g.layout is not torch.strided for g in grads):
        raise TypeError(f"{what} takes dense tensors")
    cards = set(map(_card, grads))
    if -1 in cards:
        raise RuntimeError("flashdeberta_b200 runs on CUDA devices only; there is no CPU path")
    if len(cards) > 1:
        raise ValueError(f"{what} takes tensors of one device, got {sorted(cards)}")
    other = {g.dtype for g in grads} - TYPES.keys()
    if other:
        raise TypeError(f"{what} takes bfloat16, float16 or float32 tensors, not {other.pop()}")
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
    return _run([g if _dense(g) else g.contiguous() for g in grads], None, 0.0, norm_type)


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
    if out is None and all(map(_whole, grads)):
        if 0 in map(_count, grads):
            grads = [g for g in grads if g.numel()] or grads[:1]
        return _run(grads, grads, max_norm, norm_type)
    # the kernel goes through memory: a tensor that is no run of it, or is ordered unlike its output, is taken through a copy
    reads, writes, back = [], [], []
    for g, o in zip(grads, outs):
        if g.numel() == 0:
            continue
        if (g.is_contiguous() and o.is_contiguous()) or (_dense(g) and _dense(o) and g.stride() == o.stride()):
            reads.append(g)
            writes.append(o)
            continue
        if g.data_ptr() == o.data_ptr() and g.dtype != o.dtype:
            raise ValueError("a gradient cannot be scaled in place into another type")
        reads.append(g.contiguous())
        writes.append(o if o.is_contiguous() else torch.empty(o.shape, dtype=o.dtype, device=o.device))
        if writes[-1] is not o:
            back.append((o, writes[-1]))
    if not reads:
        return grads[0].new_zeros((), dtype=torch.float32)
    norm = _run(reads, writes, max_norm, norm_type)
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
