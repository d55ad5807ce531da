"""Log probabilities of given tokens under the output head, forward and backward, without logits in memory (``csrc/log_probs.cu``)."""
from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from . import reference as ref
from ._lib import native as _native
from .calls import observed as _observed
from .token_losses import _Forward

_ROW_PAD = 256              # rows of the gathered arrays: a multiple of this (kLpRowPad in csrc/log_probs.cu)
_STAT_COLS = 128            # columns that share a log-sum (kLpStatCols)
SLAB_BYTES = 4 << 30        # the backward pass holds the logits' gradient (bf16) of so many bytes at a time, or of 256 columns;
                            # where that is all of it, the forward pass keeps the logits in as many bytes


KEEP_WIDTH = 768            # least width at which it does: the product of narrower rows costs no more than keeping it (3000 rows of 256 against 151936
                            # tokens 1017 us, kept 1141; of 512 the same; of 1024 3297 and 2839, 300 rows of 1024 478 and 406)
PLANE_BYTES = 512 << 20     # and cuts the vocabulary of the rows' gradient into as many parts (at most 64) as have fp32 results of so many bytes


def _pitch(n: int) -> int:
    """Elements from row to row of what the kernels make for themselves (``lp_pitch``)."""
    return -(-n // 64) * 64


def _planes(padded: int, D: int) -> int:
    return max(1, min(64, PLANE_BYTES // (4 * padded * D)))


def _slab(padded: int, V: int) -> int:
    """Columns of the vocabulary that the backward pass takes at a time."""
    return min(_pitch(V), max(256, SLAB_BYTES // (2 * padded) // 256 * 256))


class _LinearLogProbsFn(torch.autograd.Function):
    """``h`` ``[T, D]`` with contiguous rows, ``w`` ``[V, D]``, ``labels`` ``[T]``."""

    @staticmethod
    def forward(ctx, h, w, labels, ignore_index, temperature):
        (T, D), V, dev = h.shape, w.shape[0], h.device
        with torch.cuda.device(dev):
            y = torch.empty(T, dtype=torch.float32, device=dev)
            padded = -(-T // _ROW_PAD) * _ROW_PAD
            dense = torch.empty((padded, _pitch(D)), dtype=h.dtype, device=dev)
            rows, row_label, place = torch.empty((3, T), dtype=torch.int32, device=dev).unbind()
            count = torch.empty(1, dtype=torch.int32, device=dev)
            lse2 = torch.empty(2 * T, dtype=torch.float32, device=dev)
            codes = tops = None
            if any(ctx.needs_input_grad[:2]) and D >= KEEP_WIDTH and _slab(padded, V) >= V:
                codes = torch.empty((padded, _slab(padded, V)), dtype=torch.int16, device=dev)
                tops = torch.empty(-(-T // 4) * 4 * -(-V // _STAT_COLS), dtype=torch.float32, device=dev)
            work = torch.empty(_lib.log_probs_work(T, V), dtype=torch.float32, device=dev)
            weight = _pitched(w)
            _lib.call("ksa_log_probs", h, weight, labels, dense, rows, row_label, place, count, lse2, work, y, codes, tops, T, V, D, h.stride(0),
                      weight.stride(0), ignore_index, float(temperature))
        ctx.save_for_backward(dense, w, rows, row_label, place, count, lse2, codes, tops)
        ctx.temperature = temperature
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        dense, w, rows, row_label, place, count, lse2, codes, tops = ctx.saved_tensors
        T, (V, D), dev = rows.shape[0], w.shape, w.device
        need_h, need_w = ctx.needs_input_grad[:2]
        dh = dw = dh32 = None
        planes = 1
        with torch.cuda.device(dev):
            dy = dy.to(torch.float32).contiguous()
            weight = _pitched(w)
            dx = torch.empty((dense.shape[0], codes.shape[1] if codes is not None else _slab(dense.shape[0], V)), dtype=w.dtype, device=dev)
            if need_h:
                dh = torch.empty((T, D), dtype=w.dtype, device=dev)
                planes = _planes(dense.shape[0], D) if dx.shape[1] >= V else 1
                dh32 = torch.empty(planes * dense.shape[0] * D + 1, dtype=torch.float32, device=dev)      # (the word behind them: how many were used)

            def run(out, add):
                _lib.call("ksa_log_probs_bwd", dense, weight, rows, row_label, place, count, lse2, codes, tops, dy, dx, dh32, dh, out, T, V, D,
                          weight.stride(0), out.stride(0) if out is not None else D, int(out is not None and out.dtype == torch.float32),
                          int(add), dx.shape[1], planes, float(ctx.temperature))

            if not need_w:
                run(None, False)
            else:
                from . import _weight_grad

                def compute(out, add):
                    if out is None:
                        out = torch.empty((V, D), dtype=w.dtype, device=dev)
                    run(out, add)
                    return out
                dw = _weight_grad(w, compute)
        return dh, dw, None, None, None


def _pitched(w: torch.Tensor) -> torch.Tensor:
    """``w`` with contiguous rows that begin on 16 bytes."""
    fits = w.stride(1) == 1 and w.stride(0) % 8 == 0 and w.stride(0) >= w.shape[1] and w.data_ptr() % 16 == 0
    return w if fits else w.clone(memory_format=torch.contiguous_format)


def linear_log_probs(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, ignore_index: int = -100,
                     temperature: float = 1.0) -> torch.Tensor:
    """``log_softmax(hidden @ weight.T / temperature)`` at ``labels``: fp32 of the labels' shape, 0 where the label is ``ignore_index`` or no
    row of ``weight``.

    ``hidden`` is ``[..., D]``, ``weight`` the output head ``[V, D]`` (both bf16 on a GPU, ``D`` a multiple of 8), ``labels`` ``[...]``.  Rows
    without a label cost next to nothing and take part in nothing, whatever they hold; their gradient is 0.  Without a
    gradient the logits are never in memory.  With one the forward pass keeps them in 16 bits where the width is at least 768 and that takes at most
    ``SLAB_BYTES`` (4 GB: 14080 rows of 151936 tokens); else the backward pass computes them again, at most 4 GB of their gradient at a time.
    The logits' gradient enters its products in bf16, of up to 128 labelled rows in two parts of bf16 each.
    With ``main_grad`` on the weight its gradient goes there."""
    if not _observed():
        y = _native.linear_log_probs(hidden, weight, labels, ignore_index, temperature, _ROW_PAD, _STAT_COLS, SLAB_BYTES, PLANE_BYTES, KEEP_WIDTH)
        if y is not None:
            return y
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"rows {tuple(hidden.shape)} and an output head {tuple(weight.shape)}")
    if labels.shape != hidden.shape[:-1] or labels.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"labels are whole numbers of shape {tuple(hidden.shape[:-1])}, got {labels.dtype} {tuple(labels.shape)}")
    if not (math.isfinite(temperature) and temperature > 0):
        raise ValueError(f"the temperature must be a positive number, got {temperature}")
    if weight.shape[0] < 1:
        raise ValueError("an output head without rows")
    if not hidden.device == weight.device == labels.device:
        raise ValueError(f"tensors on {hidden.device}, {weight.device} and {labels.device}")
    if not hidden.is_cuda:
        return ref.linear_log_probs(hidden, weight, labels, ignore_index, temperature)
    if hidden.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise TypeError(f"the sm_100a kernels take bf16 activations/weights, got {hidden.dtype}, {weight.dtype}")
    if weight.shape[1] % 8 != 0 or weight.shape[1] == 0:
        raise ValueError(f"the width {weight.shape[1]} must be a multiple of 8")
    if labels.numel() == 0:
        return (hidden.sum(-1) * 0).float().reshape(labels.shape) + 0 * weight[:0].sum().float()
    h2 = hidden.reshape(-1, hidden.shape[-1])
    if h2.stride(1) != 1:
        h2 = h2.contiguous()
    flat = labels.reshape(-1).to(torch.int64).contiguous()
    if _observed() or (torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad)):
        y = _LinearLogProbsFn.apply(h2, weight, flat, ignore_index, temperature)
    else:
        y = _LinearLogProbsFn.forward(_Forward(), h2, weight, flat, ignore_index, temperature)
    return y.view(labels.shape)
