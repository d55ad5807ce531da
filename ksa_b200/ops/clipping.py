"""Global gradient norm over many tensors, and clipping by it (``csrc/grad_norm.cu``).

``norm = scale * sqrt(sum of all squares)`` and ``factor = scale * min(1, max_norm / (norm + 1e-6))``: what
``torch.nn.utils.clip_grad_norm_`` computes, for gradients that are still to be multiplied by ``scale`` (one over the number
of accumulated micro-batches or of ranks).  Both stay on the device.

The gradients of one call may have different types (fp32, bf16, fp16), sizes, strides and alignments, and there may be none.  The sums
have a fixed order: the same gradients give the same bits.  Not differentiable.
"""
from __future__ import annotations

import ctypes
import math
from typing import Iterable, List, Optional, Sequence, Tuple, Union

import torch

from . import _lib
from . import reference as ref
from ._lib import native as _native
from .calls import observed as _observed

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _dense(t: torch.Tensor) -> bool:
    """Whether the values fill one range of memory (in any order of the dimensions)."""
    return t.is_contiguous() or torch.ops.aten.is_non_overlapping_and_dense(t)


def _check(grads: Iterable[torch.Tensor], scale: float) -> List[torch.Tensor]:
    grads = list(grads)
    for g in grads:
        if not isinstance(g, torch.Tensor) or g.layout != torch.strided:
            raise TypeError("the gradients must be dense tensors")
        if g.dtype not in _TYPES:
            raise TypeError(f"gradients are fp32, bf16 or fp16, got {g.dtype}")
        if g.device != grads[0].device:
            raise ValueError(f"the gradients lie on several devices: {grads[0].device} and {g.device}")
    if not (math.isfinite(scale) and scale > 0):
        raise ValueError(f"the scale must be a positive number, got {scale}")
    return grads


def _check_most(max_norm: float) -> float:
    if not max_norm >= 0:
        raise ValueError(f"the largest norm must not be negative, got {max_norm}")
    return float(max_norm)


def _collide(src: Sequence[torch.Tensor], dst: Sequence[torch.Tensor]) -> bool:
    """Whether memory that is written is written or read for another tensor too."""
    spans = []
    for s, d in zip(src, dst):
        if s.numel() == 0:
            continue
        size, a, b = s.numel() * s.element_size(), s.data_ptr(), d.data_ptr()
        spans.append((b, b + size, True))
        if a != b:
            spans.append((a, a + size, False))
    spans.sort()
    any_end = written_end = 0
    for lo, hi, written in spans:
        if lo < (any_end if written else written_end):
            return True
        any_end = max(any_end, hi)
        if written:
            written_end = max(written_end, hi)
    return False


def _layout(t: torch.Tensor) -> List[Tuple[int, int]]:
    """(stride in bytes, size) of the dimensions that have more than one element, the widest first."""
    return sorted(((st * t.element_size(), n) for n, st in zip(t.shape, t.stride()) if n > 1), reverse=True)


def _end(t: torch.Tensor) -> int:
    return t.data_ptr() + sum((n - 1) * st for st, n in _layout(t)) + t.element_size()


def _folded(t: torch.Tensor) -> bool:
    """Whether elements of ``t`` may share memory with one another: a dimension steps over less than those below it take."""
    reach = t.element_size()
    for st, n in reversed(_layout(t)):
        if st < reach:
            return True
        reach += (n - 1) * st
    return False


_MOST_STEPS = 10000         # of the search below; layouts that take more count as meeting


def _meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether an element of ``a`` has memory in common with one of ``b``, by the difference of their places: a sum of strides, each as often as
    the indices of the two may differ, which has to come within an element of the distance between the tensors."""
    often = {}
    for t, sign in ((a, 1), (b, -1)):
        for st, n in _layout(t):
            lo, hi = often.get(st, (0, 0))
            often[st] = (lo, hi + n - 1) if sign > 0 else (lo - n + 1, hi)
    dims = sorted(often.items(), reverse=True)
    low, high = [0], [0]                                # what the strides from here on can add up to
    for st, (lo, hi) in reversed(dims):
        low.insert(0, low[0] + lo * st)
        high.insert(0, high[0] + hi * st)
    apart = b.data_ptr() - a.data_ptr()
    first, last = apart - a.element_size() + 1, apart + b.element_size() - 1
    steps = 0

    def search(i: int, at: int) -> bool:
        nonlocal steps
        steps += 1
        if steps > _MOST_STEPS:
            return True
        if i == len(dims):
            return first <= at <= last
        st, (lo, hi) = dims[i]
        lo, hi = max(lo, -((at + high[i + 1] - first) // st)), min(hi, (last - at - low[i + 1]) // st)
        return any(search(i + 1, at + k * st) for k in range(lo, hi + 1))
    return search(0, 0)


def _share(targets: Sequence[torch.Tensor]) -> bool:
    """Whether two of the targets, or two elements of one, have memory in common; those that fill theirs are compared by :func:`_collide`."""
    targets = [(t, _dense(t)) for t in targets if t.numel() > 0]
    if all(dense for _, dense in targets):
        return False
    if any(not dense and _folded(t) for t, dense in targets):
        return True
    targets = sorted(((t.data_ptr(), _end(t), dense, t) for t, dense in targets), key=lambda x: x[:2])
    for i, (_, end, dense, t) in enumerate(targets):
        for lo, _, other_dense, other in targets[i + 1:]:
            if lo >= end:
                break
            if not (dense and other_dense) and _meet(t, other):
                return True
    return False


def _launch(src: Sequence[torch.Tensor], dst: Optional[Sequence[torch.Tensor]], scale: float, most: float) -> Tuple[torch.Tensor, torch.Tensor]:
    device = src[0].device
    n = len(src)
    with torch.cuda.device(device):
        parts = torch.empty(_lib.grad_norm_parts(n), dtype=torch.float64, device=device)
        norm, factor = torch.empty((), dtype=torch.float32, device=device), torch.empty((), dtype=torch.float32, device=device)
        at = (ctypes.c_void_p * n)(*[t.data_ptr() for t in src])
        to = None if dst is None else (ctypes.c_void_p * n)(*[t.data_ptr() for t in dst])
        meta = (ctypes.c_longlong * n)(*[4 * t.numel() + _TYPES[t.dtype] for t in src])
        _lib.call("ksa_grad_norm", at, to, meta, n, float(scale), float(most), parts, norm, factor)
    return norm, factor


def grad_norm(grads: Iterable[torch.Tensor], scale: float = 1.0,
              max_norm: Optional[float] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """The global 2-norm of ``grads`` times ``scale``, an fp32 scalar on their device; with ``max_norm`` also the factor that
    clips: ``scale * min(1, max_norm / (norm + 1e-6))``."""
    grads = grads if isinstance(grads, (list, tuple)) else list(grads)
    if not _observed():
        made = _native.grad_norm(grads, None, 0 if max_norm is None else 1, scale, math.inf if max_norm is None else max_norm)
        if made is not None:
            return made
    grads = _check(grads, scale)
    most = math.inf if max_norm is None else _check_most(max_norm)
    with torch.no_grad():
        if not grads or not grads[0].is_cuda:
            norm, factor = ref.grad_norm(grads, scale, most)
        else:
            norm, factor = _launch([g if _dense(g) else g.contiguous() for g in grads], None, scale, most)
    return norm if max_norm is None else (norm, factor)


def clip_grad_norm_(grads: Iterable[torch.Tensor], max_norm: float, scale: float = 1.0,
                    out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Multiply every gradient by ``scale * min(1, max_norm / (norm + 1e-6))`` and return ``norm``, the global 2-norm times
    ``scale``.  In place, or into the tensors ``out`` (of the gradients' shapes and types); gradients that share memory with
    one another are refused (those that only interleave, as the columns of one matrix do, are fine).  A norm that is no number makes all of them so, an infinite one makes them zero where they are finite."""
    grads = grads if isinstance(grads, (list, tuple)) else list(grads)
    if not _observed():
        made = _native.grad_norm(grads, out, 2, scale, max_norm)
        if made is not None:
            return made
    grads = _check(grads, scale)
    most = _check_most(max_norm)
    to = grads if out is None else list(out)
    if len(to) != len(grads) or any(o.shape != g.shape or o.dtype != g.dtype or o.device != g.device for o, g in zip(to, grads)):
        raise ValueError("the clipped gradients go into tensors of the same number, shapes, types and device")
    with torch.no_grad():
        if _share(to):
            raise ValueError("gradients that are clipped must not share memory")
        # values that do not fill their memory, or in another order than their target's: through a copy
        src = [g if _dense(g) and g.stride() == o.stride() else g.contiguous() for g, o in zip(grads, to)]
        dst = [o if s.stride() == o.stride() and _dense(o) else torch.empty_like(s) for s, o in zip(src, to)]
        if _collide(src, dst):
            raise ValueError("gradients that are clipped must not share memory")
        if not grads or not grads[0].is_cuda:
            norm, factor = ref.grad_norm(grads, scale, most)
            for d, s in zip(dst, src):
                d.copy_(s.float() * factor)
        else:
            norm = _launch(src, dst, scale, most)[0]
        for o, d in zip(to, dst):
            if d is not o:
                o.copy_(d)
        torch.autograd.graph.increment_version([t for t in to if not t.is_inference()])
    return norm
