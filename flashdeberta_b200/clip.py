"""The global norm of a model's gradients, and clipping by it: two launches for every thousand tensors.

The reference leaves this step of training to torch (its models are trained by transformers' Trainer over
src/flashdeberta/model.py:394-920), which launches over lists of tensors per type and keeps the norms of the single tensors.
"""
from __future__ import annotations

import bisect
import ctypes as C
import math
import operator
from typing import Iterable, List, Optional, Sequence, Union

import numpy as np
import torch

from . import _lib, ops
from .norms import TYPES

Tensors = Union[torch.Tensor, Iterable[torch.Tensor]]
_NORMS = {1.0: 1, 2.0: 2, math.inf: 0}
_TABLE = 1000  # tensors that a launch takes


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


def _layout(t: torch.Tensor):
    """(first byte, bytes of a run without gaps, [(bytes between, count)] of what the runs are repeated over)."""
    run, outer = t.element_size(), []
    for stride, size in sorted((s * t.element_size(), n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride == run and not outer:
            run *= size
        else:
            outer.append((stride, size))
    return t.data_ptr(), run, outer


def _starts(at, run, outer) -> np.ndarray:
    """Where the runs begin, in order."""
    starts = np.array([at], np.int64)
    for stride, size in outer:
        if stride == 0:  # (the same places again)
            continue
        starts = (starts[:, None] + stride * np.arange(size, dtype=np.int64)).ravel()
    return np.sort(starts)


def _folded(at, run, outer) -> bool:
    """Whether two elements of a tensor lie in the same place."""
    span = run
    for stride, size in outer:
        if stride == 0:  # (an expanded dimension)
            return True
        if stride < span:  # windows that slide, or rows that pass through one another
            return bool((np.diff(_starts(at, run, outer)) < run).any())
        span += stride * (size - 1)
    return False


def _apart_modulo(layouts) -> bool:
    """Whether the runs keep apart modulo what all strides are multiples of: slices of one matrix's columns do.  (They may be
    apart without that.)"""
    period = math.gcd(*(stride for _, _, outer in layouts for stride, _ in outer))
    if period == 0:
        return False
    runs = sorted((at % period, run) for at, run, _ in layouts)
    return all(a + n <= b for (a, n), (b, _) in zip(runs, runs[1:] + [(runs[0][0] + period, 0)]))


def _cross(a, b) -> bool:
    """Whether two tensors have an element in the same place."""
    if _apart_modulo((a, b)):
        return False
    (sa, ra), (sb, rb) = (_starts(*a), a[1]), (_starts(*b), b[1])
    near = np.searchsorted(sa, sb + rb) - 1  # the last run that begins before each of b's ends
    return bool(((near >= 0) & (sa[near] + ra > sb)).any())


def _end(at, run, outer) -> int:
    return at + run + sum(stride * (size - 1) for stride, size in outer)


def _collide(writes, reads) -> bool:
    """Whether an element that is written is also another one that is written, or one that is read."""
    placed = [(_layout(t), True) for t in writes] + [(_layout(t), False) for t in reads]
    if any(writes and _folded(*layout) for layout, writes in placed):
        return True
    placed = sorted(((layout[0], _end(*layout), layout, w) for layout, w in placed), key=lambda p: p[:2])
    group, end = [], 0
    for p in placed + [(math.inf, math.inf, None, False)]:
        if p[0] >= end:  # nothing so far reaches further: a group of tensors in one another's way
            if any(g[3] for g in group) and len(group) > 1 and not _apart_modulo([g[2] for g in group]):
                for i, a in enumerate(group):
                    for b in group[i + 1:]:
                        if (a[3] or b[3]) and b[0] < a[1] and _cross(a[2], b[2]):
                            return True
            group = []
        group.append(p)
        end = max(end, p[1])
    return False


_at, _count, _whole, _card = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.is_contiguous, torch.Tensor.get_device
_dtype, _shape = operator.attrgetter("dtype"), operator.attrgetter("shape")
_PLAIN = {torch.Tensor, torch.nn.Parameter}
_BYTES = np.zeros(1 + max(TYPES.values()), np.int64)
for _t, _kind in TYPES.items():
    _BYTES[_kind] = _t.itemsize


class _Listed:
    """Tensors of one device as the C call sees them: addresses, counts, types."""

    def __init__(self, tensors: Tensors, what: str):
        tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
        if not set(map(type, tensors)) <= _PLAIN:
            raise TypeError(f"{what} takes plain tensors (it goes by their memory: no traced, fake or distributed ones)")
        cards = set(map(_card, tensors))
        if -1 in cards:
            raise RuntimeError("flashdeberta_b200 runs on CUDA devices only; there is no CPU path")
        if len(cards) > 1:
            raise ValueError(f"{what} takes tensors of one device, got {sorted(cards)}")
        ops.refuse_tangents(what, tensors)
        self.tensors, n = tensors, len(tensors)
        try:
            self.kind = np.fromiter(map(TYPES.__getitem__, map(_dtype, tensors)), np.int64, n)
        except KeyError as e:
            raise TypeError(f"{what} takes bfloat16, float16 or float32 tensors, not {e.args[0]}") from None
        try:
            self.at = np.fromiter(map(_at, tensors), np.int64, n)
        except (RuntimeError, NotImplementedError):  # no memory to point at
            raise TypeError(f"{what} takes dense tensors") from None
        self.count = np.fromiter(map(_count, tensors), np.int64, n)

    def whole(self) -> bool:
        return all(map(_whole, self.tensors))


def _run(grads: _Listed, outs: Optional[_Listed], max_norm: float, norm_type: float) -> torch.Tensor:
    """One C call: the norm, and, with ``outs``, the scaled tensors.  All are runs of memory."""
    at, count, kind = grads.at, grads.count, grads.kind
    to, into = (at, kind) if outs is None else (outs.at, outs.kind)
    if outs is not None:
        starts, ends = to, to + count * _BYTES[into]
        if outs is not grads:
            read = (at != to) & (count > 0)  # (the others are their own outputs)
            if (kind != into)[(at == to) & (count > 0)].any():
                raise ValueError("a gradient cannot be scaled in place into another type")
            starts, ends = np.concatenate((to, at[read])), np.concatenate((ends, (at + count * _BYTES[kind])[read]))
        # runs of memory are apart where each ends, in order, before the next begins (one of no bytes begins and ends between two)
        if (np.sort(ends)[:-1] > np.sort(starts)[1:]).any():
            n = len(to)
            if not _apart(zip(starts[:n].tolist(), ends[:n].tolist()), zip(starts[n:].tolist(), ends[n:].tolist())):
                raise ValueError("the tensors that are written overlap one another or a gradient that is read")
    table = np.empty((len(at), 4), np.int64)  # rows of fdb_grad_tensor: two addresses, the count, both types
    table[:, 0], table[:, 1], table[:, 2], table[:, 3] = at, to, count, kind | into << 32
    first, lib = grads.tensors[0], _lib.load()
    device = first.device
    norm = first.new_empty((), dtype=torch.float32)
    p = _lib.ClipGradsParams(C.sizeof(_lib.ClipGradsParams), len(at), table.ctypes.data, _NORMS[norm_type], int(outs is not None),
                             max_norm, norm.data_ptr(), None, 0)
    with ops.on_device(device):
        need = lib.fdb_clip_grads_workspace_bytes(C.byref(p))
        ws = norm.new_empty(max(need, 16), dtype=torch.uint8)
        p.workspace, p.workspace_bytes = ws.data_ptr(), need
        _lib.check(lib.fdb_clip_grads(C.byref(p), ops.raw_stream(device)))
    if outs is not None:  # the write is seen by whoever compares versions (autograd, the caches of this package)
        torch.autograd.graph.increment_version(outs.tensors)
    tables = -(-len(at) // _TABLE)
    ops._launches += tables + (tables if outs is not None else 1)
    return norm


def _norm_type(norm_type: float) -> float:
    norm_type = float(norm_type)
    if norm_type not in _NORMS:
        raise ValueError(f"norm_type must be 1, 2 or inf, not {norm_type}")
    return norm_type


def grad_norm(grads: Tensors, norm_type: float = 2.0) -> torch.Tensor:
    """The norm (1, 2 or inf) over all elements of the tensors taken as one vector: a float32 scalar on their device, zero where there
    are none.  Tensors are bfloat16, float16 or float32 in any mixture, of one device.  As torch's own, it records no gradient."""
    norm_type, grads = _norm_type(norm_type), _Listed(grads, "grad_norm")
    if not grads.tensors:
        return torch.tensor(0.0)
    if not grads.whole():
        grads = _Listed([g if g.is_contiguous() or _dense(g) else g.detach().contiguous() for g in grads.tensors], "grad_norm")
    return _run(grads, None, 0.0, norm_type)


def clip_grads_(grads: Tensors, max_norm: float, *, norm_type: float = 2.0, out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Scales the tensors by ``min(1, max_norm / (norm + 1e-6))``, norm as in ``grad_norm``, in place, or into ``out`` (tensors of the same
    shapes, of any of the three types: an optimizer's float32 buffers beside bfloat16 gradients), and returns the norm before.  Nothing
    is read back to the host.  Where the factor is one, tensors scaled in place are not written (but for those with gaps in memory,
    which go through a copy).  The tensors that are written must not overlap one another or, but for a tensor that is its own
    output, those that are read."""
    norm_type, grads = _norm_type(norm_type), _Listed(grads, "clip_grads_")
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative or NaN, got {max_norm}")
    outs = grads if out is None else _Listed(out, "clip_grads_")
    if out is not None and list(map(_shape, outs.tensors)) != list(map(_shape, grads.tensors)):
        raise ValueError("out must hold one tensor of the same shape for each gradient")
    if not grads.tensors:
        return torch.tensor(0.0)
    if outs.tensors[0].device != grads.tensors[0].device:
        raise ValueError(f"out is on {outs.tensors[0].device}, the gradients on {grads.tensors[0].device}")
    if grads.whole() and (out is None or outs.whole()):
        return _run(grads, outs, max_norm, norm_type)
    return _clip_any(grads, outs, max_norm, norm_type)


def _check_any(grads: _Listed, outs: _Listed) -> None:
    """What ``_run`` checks of tensors without gaps, of tensors in any layout."""
    same, live = grads.at == outs.at, grads.count > 0
    if (same & live & (grads.kind != outs.kind)).any():
        raise ValueError("a gradient cannot be scaled in place into another type")
    writes, reads = np.flatnonzero(live), np.flatnonzero(live & ~same)

    gaps = []  # layouts of the tensors that are written and not contiguous

    def ends(listed):
        to = listed.at + listed.count * _BYTES[listed.kind]
        for i in np.flatnonzero(~np.fromiter(map(_whole, listed.tensors), bool, len(to)) & live):
            layout = _layout(listed.tensors[i])
            to[i] = _end(*layout)
            if listed is outs:
                gaps.append(layout)
        return to

    starts, to = outs.at[writes], ends(outs)[writes]
    if len(reads):
        starts, to = np.concatenate((starts, grads.at[reads])), np.concatenate((to, ends(grads)[reads]))
    order = np.argsort(starts)
    if (np.maximum.accumulate(to[order])[:-1] > starts[order][1:]).any():  # one reaches into another: they may still pass by one another
        bad = _collide([outs.tensors[i] for i in writes], [grads.tensors[i] for i in reads])
    else:
        bad = any(_folded(*layout) for layout in gaps)
    if bad:
        raise ValueError("the tensors that are written overlap one another or a gradient that is read")


@torch.no_grad()
def _clip_any(grads: _Listed, outs: _Listed, max_norm, norm_type):
    """The kernel goes through memory: a tensor that is no run of it, or is ordered unlike its output, is taken through a copy."""
    _check_any(grads, outs)
    grads, outs = grads.tensors, outs.tensors
    reads, writes, back = [], [], []
    for g, o in zip(grads, outs):
        if g.numel() == 0:
            continue
        if (g.is_contiguous() and o.is_contiguous()) or (_dense(g) and _dense(o) and g.stride() == o.stride()):
            reads.append(g)
            writes.append(o)
            continue
        reads.append(g.contiguous())
        writes.append(o if o.is_contiguous() else torch.empty(o.shape, dtype=o.dtype, device=o.device))
        if writes[-1] is not o:
            back.append((o, writes[-1]))
    if not reads:
        return grads[0].new_zeros((), dtype=torch.float32)
    into = _Listed(writes, "clip_grads_")
    norm = _run(into if all(map(operator.is_, reads, writes)) else _Listed(reads, "clip_grads_"), into, max_norm, norm_type)
    for o, scaled in back:
        o.copy_(scaled)
    return norm


def clip_grad_norm_(parameters: Tensors, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """``torch.nn.utils.clip_grad_norm_`` over this package's kernels: the gradients of the parameters that have one are clipped in
    place to ``max_norm``; returns their norm before.  Narrower than torch's: plain bfloat16, float16 or float32 tensors of one device,
    and norms 1, 2 and inf; anything else raises.  ``error_if_nonfinite`` reads the norm back to the host first (and raises before
    anything is scaled); without it nothing is read back."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else parameters
    grads = [p.grad for p in parameters if p.grad is not None]
    if error_if_nonfinite and grads:
        norm = grad_norm(grads, norm_type)
        if not math.isfinite(norm.item()):
            raise RuntimeError(f"the norm of order {norm_type} of the gradients is not finite, so they are not clipped")
    return clip_grads_(grads, max_norm, norm_type=norm_type)
