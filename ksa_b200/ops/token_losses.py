"""Losses of a post-training step over the log probabilities of answer tokens: the clipped policy loss with a KL term and the
preference loss of pairs (``csrc/token_losses.cu``).

Tokens come as rows ``[sequences, length]``, or packed: one dimension (or ``[1, tokens]``) with the sequences' offsets
``cu_seqlens`` ``[sequences + 1]`` (int32 or int64, on the tokens' device, from 0 on and never falling; a sequence may be empty).  One dimension
without offsets is one sequence.  ``mask`` (bool or uint8, a value for every token) says which tokens count; what the others hold, NaN included, is
never read into a sum, and neither is what lies behind the last offset: their gradient is zero.  Log probabilities and advantages are fp32, bf16 or
fp16, each for itself.  Gradients flow to ``log_probs`` alone.
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from . import reference as ref
from ._lib import native as _native
from .calls import observed as _observed

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class _Sequences(NamedTuple):
    n: int                              # tokens, those behind the last sequence included
    count: int
    length: int                         # of every sequence, where there are no offsets
    cu: Optional[torch.Tensor]

    def args(self):
        return self.cu, int(self.cu is not None and self.cu.dtype == torch.int64)


def _sequences(log_probs: torch.Tensor, cu_seqlens: Optional[torch.Tensor]) -> _Sequences:
    n = log_probs.numel()
    if cu_seqlens is None:
        if log_probs.dim() == 1:
            return _Sequences(n, 1, n, None)
        if log_probs.dim() != 2:
            raise ValueError(f"log probabilities are [sequences, length] or packed, got shape {tuple(log_probs.shape)}")
        return _Sequences(n, log_probs.shape[0], log_probs.shape[1], None)
    if log_probs.dim() != 1 and not (log_probs.dim() == 2 and log_probs.shape[0] == 1):
        raise ValueError(f"packed log probabilities have one dimension, got shape {tuple(log_probs.shape)}")
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1 or cu_seqlens.dtype not in (torch.int32, torch.int64):
        raise ValueError("the sequences' offsets are int32 or int64 [sequences + 1]")
    return _Sequences(n, cu_seqlens.numel() - 1, 0, cu_seqlens.contiguous())


def _check(log_probs: torch.Tensor, mask: Optional[torch.Tensor], cu_seqlens: Optional[torch.Tensor], constants) -> None:
    """``constants``: (name, tensor or None) of what has a value for every token and no gradient."""
    for name, t in (("log_probs", log_probs), *constants):
        if t is None:
            continue
        if t.dtype not in _TYPES:
            raise TypeError(f"{name} is fp32, bf16 or fp16, got {t.dtype}")
        if name != "log_probs" and t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"no gradient flows to {name}: detach it")
        if name not in ("log_probs", "advantages") and t.shape != log_probs.shape:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, log_probs {tuple(log_probs.shape)}")
    if mask is not None and (mask.dtype not in (torch.bool, torch.uint8) or mask.shape != log_probs.shape):
        raise ValueError(f"the mask is bool or uint8 of shape {tuple(log_probs.shape)}, got {mask.dtype} {tuple(mask.shape)}")
    for t in (mask, cu_seqlens, *(t for _, t in constants)):
        if t is not None and t.device != log_probs.device:
            raise ValueError(f"tensors on {log_probs.device} and {t.device}")


def _type_bits(*tensors) -> int:
    return sum(_TYPES[t.dtype] << 4 * i for i, t in enumerate(tensors) if t is not None)


def _flat(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if t is None else t if t.is_contiguous() else t.contiguous()


class _PolicyLossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, old, adv, ref_y, mask, seq, by_sequence_adv, clip_low, clip_high, kl_coef, by_sequence):
        dev = y.device
        with torch.cuda.device(dev):
            grad = torch.empty(seq.n, dtype=torch.float32, device=dev) if ctx.needs_input_grad[0] else None
            partial = torch.empty(4 * _lib.token_loss_units(seq.n, seq.count), dtype=torch.float64, device=dev)
            inv = torch.empty(max(seq.count, 1), dtype=torch.float32, device=dev)
            loss, stats = torch.empty((), dtype=torch.float32, device=dev), torch.empty(3, dtype=torch.float32, device=dev)
            bounds = (ctypes.c_double * 4)(math.log1p(clip_high), math.log1p(-clip_low) if clip_low < 1 else -math.inf, 1 + clip_high, 1 - clip_low)
            y_, old, adv, ref_y, mask = (_flat(t) for t in (y, old, adv, ref_y, mask))
            _lib.call("ksa_policy_loss", y_, old, ref_y, adv, mask, *seq.args(), grad, partial, inv, loss, stats,
                      _type_bits(y_, old, ref_y, adv), seq.n, seq.count, seq.length, int(by_sequence_adv), int(by_sequence), bounds,
                      float(kl_coef))
        ctx.save_for_backward(grad, inv, seq.cu)
        ctx.cfg = (seq._replace(cu=None), by_sequence, y.dtype, y.shape)
        ctx.mark_non_differentiable(stats)
        return loss, stats

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _):
        grad, inv, cu = ctx.saved_tensors
        seq, by_sequence, dtype, shape = ctx.cfg
        with torch.cuda.device(inv.device):
            dy = torch.empty(shape, dtype=dtype, device=inv.device)
            _lib.call("ksa_policy_loss_bwd", grad, inv, dloss, dy, _TYPES[dtype], *seq._replace(cu=cu).args(), seq.n, seq.count, seq.length,
                      int(by_sequence))
        return (dy,) + (None,) * 10


class _Forward:
    """The context of a forward pass that nobody will differentiate."""
    needs_input_grad = (False,) * 16

    def save_for_backward(self, *tensors):
        pass

    def mark_non_differentiable(self, *tensors):
        pass


def _run(fn, y, *args):
    if y.requires_grad and torch.is_grad_enabled() or _observed():
        return fn.apply(y, *args)
    return fn.forward(_Forward(), y, *args)


def policy_loss(log_probs: torch.Tensor, old_log_probs: torch.Tensor, advantages: torch.Tensor, ref_log_probs: Optional[torch.Tensor] = None,
                mask: Optional[torch.Tensor] = None, cu_seqlens: Optional[torch.Tensor] = None, *, clip_low: float = 0.2, clip_high: float = 0.2,
                kl_coef: float = 0.0, reduction: str = "token") -> Tuple[torch.Tensor, torch.Tensor]:
    """The clipped policy loss with a KL term: ``(loss, stats)``.

    With ``r = exp(log_probs - old_log_probs)`` a token's loss is ``-min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef K``,
    ``K = exp(x) - 1 - x`` for ``x = ref_log_probs - log_probs`` (0 without a reference); where ``A`` is 0 so is the first part, however large ``r``.
    ``advantages``: of the shape of ``log_probs``, a value for every token; else ``[sequences]`` or ``[sequences, 1]``, one for every sequence.  (Packed in
    one dimension, as many values as tokens are one for every token, also where there are as many sequences; ``[sequences, 1]`` says otherwise.)
    ``reduction``: "token", the mean over the valid tokens, or "sequence", the mean over the sequences that have one of each sequence's mean;
    without any valid token the loss is 0.  ``stats`` (fp32 ``[3]``, no gradient): the same means of the clipped
    part, of ``K`` and of being cut off, that is ``A > 0`` with ``r > 1 + clip_high`` or ``A < 0`` with ``r < 1 - clip_low``; such a token has no
    gradient but that of ``K``.  With a ``kl_coef`` of 0 the reference counts in the statistics alone."""
    if not _observed() and reduction in ("token", "sequence"):
        made = _native.policy_loss(log_probs, old_log_probs, advantages, ref_log_probs, mask, cu_seqlens, clip_low, clip_high, kl_coef,
                                   reduction == "sequence")
        if made is not None:
            return made
    _check(log_probs, mask, cu_seqlens, (("old_log_probs", old_log_probs), ("advantages", advantages), ("ref_log_probs", ref_log_probs)))
    seq = _sequences(log_probs, cu_seqlens)
    by_token = advantages.shape == log_probs.shape
    if not by_token and tuple(advantages.shape) not in ((seq.count,), (seq.count, 1)):
        raise ValueError(f"advantages are {tuple(log_probs.shape)} or [{seq.count}], got {tuple(advantages.shape)}")
    if reduction not in ("token", "sequence"):
        raise ValueError(f"unknown reduction {reduction!r}")
    if not (0 <= clip_low <= 1 and clip_high >= 0) or not math.isfinite(kl_coef):
        raise ValueError(f"clip_low {clip_low} (0 to 1), clip_high {clip_high} (0 or more), kl_coef {kl_coef}")
    if not log_probs.is_cuda:
        flat = lambda t: None if t is None else t.reshape(-1)  # noqa: E731
        of = ref.sequence_of(seq.n, seq.count, seq.cu, log_probs.device)
        return ref.policy_loss(flat(log_probs), flat(old_log_probs), flat(advantages), flat(ref_log_probs), flat(mask), of, seq.count, clip_low,
                               clip_high, kl_coef, reduction == "sequence", not by_token)
    return _run(_PolicyLossFn, log_probs, old_log_probs, advantages, ref_log_probs, mask, seq, not by_token, clip_low, clip_high, kl_coef,
                reduction == "sequence")


class _PreferenceLossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, ref_y, mask, seq, beta, smoothing):
        dev = y.device
        with torch.cuda.device(dev):
            partial = torch.empty(_lib.token_loss_units(seq.n, seq.count), dtype=torch.float64, device=dev)
            coef = torch.empty(seq.count, dtype=torch.float32, device=dev)
            loss, rewards = torch.empty((), dtype=torch.float32, device=dev), torch.empty((seq.count // 2, 2), dtype=torch.float32, device=dev)
            y_, ref_y, mask = (_flat(t) for t in (y, ref_y, mask))
            _lib.call("ksa_preference_loss", y_, ref_y, mask, *seq.args(), partial, coef, rewards, loss, _type_bits(y_, ref_y), seq.n, seq.count,
                      seq.length, float(beta), float(smoothing))
        ctx.save_for_backward(coef, mask, seq.cu)
        ctx.cfg = (seq._replace(cu=None), y.dtype, y.shape)
        ctx.mark_non_differentiable(rewards)
        return loss, rewards

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _):
        coef, mask, cu = ctx.saved_tensors
        seq, dtype, shape = ctx.cfg
        with torch.cuda.device(coef.device):
            dy = torch.empty(shape, dtype=dtype, device=coef.device)
            _lib.call("ksa_preference_loss_bwd", mask, coef, dloss, dy, _TYPES[dtype], *seq._replace(cu=cu).args(), seq.n, seq.count, seq.length)
        return (dy,) + (None,) * 5


def preference_loss(log_probs: torch.Tensor, ref_log_probs: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                    cu_seqlens: Optional[torch.Tensor] = None, *, beta: float = 0.1,
                    label_smoothing: float = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """The preference loss of pairs of answers: ``(loss, rewards)``.

    Sequences ``2 i`` and ``2 i + 1`` are the preferred and the rejected answer of pair ``i``.  ``D_s`` is the sum of ``log_probs - ref_log_probs``
    (``log_probs`` alone without a reference) over the valid tokens of sequence ``s``, ``z_i = beta (D_2i - D_2i+1)``; the loss is the mean over
    the pairs of ``(1 - label_smoothing) log(1 + exp(-z)) + label_smoothing log(1 + exp(z))``, 0 without any pair.  ``rewards`` (fp32
    ``[pairs, 2]``, no gradient): ``beta D``.  An answer without valid tokens has ``D = 0``."""
    if not _observed():
        made = _native.preference_loss(log_probs, ref_log_probs, mask, cu_seqlens, beta, label_smoothing)
        if made is not None:
            return made
    _check(log_probs, mask, cu_seqlens, (("ref_log_probs", ref_log_probs),))
    seq = _sequences(log_probs, cu_seqlens)
    if seq.count % 2 != 0:
        raise ValueError(f"{seq.count} sequences are not pairs")
    if not math.isfinite(beta) or not 0 <= label_smoothing <= 1:
        raise ValueError(f"beta {beta}, label_smoothing {label_smoothing} (0 to 1)")
    if not log_probs.is_cuda:
        flat = lambda t: None if t is None else t.reshape(-1)  # noqa: E731
        of = ref.sequence_of(seq.n, seq.count, seq.cu, log_probs.device)
        return ref.preference_loss(flat(log_probs), flat(ref_log_probs), flat(mask), of, seq.count, beta, label_smoothing)
    return _run(_PreferenceLossFn, log_probs, ref_log_probs, mask, seq, beta, label_smoothing)

