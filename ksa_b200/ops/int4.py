"""Serving in four bits: a KV cache that is quantised as it is written, decode attention over it, and projections whose
weights are held in four bits.  For inference only: nothing here is differentiated.

Format (:func:`ksa_b200.ops.reference.int4_quantize`).  A group of values (32 along the head dimension of a cache row; 32, 64
or 128 along ``K`` of a weight row) with least value ``lo`` and greatest ``hi`` has, in bf16, a scale
``S = bf16((hi - lo) / 15 * 16)`` (0 where that is below 2^-100) and an offset ``O = bf16(lo - S)``.  A code
``c = rint((x - O) / S * 16) - 16``, cut to 0 .. 15, stands for ``bf16(S * (1 + c / 16) + O)``: those bf16 values are what reading
returns and what attention and products compute with, to the bit.  The error is at most half a step, ``(hi - lo) / 30``, and the
roundings of ``S``, ``O`` and the result to bf16.  Eight codes make a little-endian 32-bit word, its nibbles from the lowest being
values 0, 2, 4, 6, 1, 3, 5, 7.  A group that holds an infinity or a NaN stands for NaN; finite magnitudes over 2^126 count as 2^126, and those
below 2^-126 as zero.
"""
from __future__ import annotations

import contextlib
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from . import reference as ref
from ._lib import native as _native

CACHE_GROUP = 32          # values of a cache row that share a scale
CACHE_DIM = 2048          # largest head dimension
CACHE_SLOTS = 16          # the capacity of a cache is a multiple of this
FEW_ROWS = 32             # rows that the kernels of ``int4_linear`` take
FUSED_ROWS = 16           # and that of ``int4_linear_swiglu``
NORM_ROWS = 4             # rows that ``int4_norm_linear`` takes in one launch,
NORM_VALUES = 32768       # and values, which every CTA keeps in shared memory


class Int4Cache(NamedTuple):
    """Keys and values of one layer: codes ``[B, Hkv, cap, D / 2]`` uint8, scales ``[B, Hkv, cap, D / 32, 2]`` bf16 (scale,
    offset), all contiguous; ``cap`` is a multiple of 16 and ``D`` of 32.  A slice along ``B`` is a cache as well (:meth:`rows`)."""
    k: torch.Tensor
    k_scale: torch.Tensor
    v: torch.Tensor
    v_scale: torch.Tensor

    def rows(self, sequences: slice) -> "Int4Cache":
        return Int4Cache(*(t[sequences] for t in self))

    @property
    def capacity(self) -> int:
        return self.k.shape[2]

    def bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self)


class Int4Weight(NamedTuple):
    """A weight ``[N, K]``: codes ``[N, K / 2]`` uint8, scales ``[K / group, pitch, 2]`` bf16 (scale, offset) of row ``n`` at
    ``[:, n]``, ``pitch`` being ``N`` rounded up to a multiple of 4; both contiguous."""
    codes: torch.Tensor
    scale: torch.Tensor

    @property
    def shape(self) -> Tuple[int, int]:
        return self.codes.shape[0], 2 * self.codes.shape[1]

    @property
    def group(self) -> int:
        return 2 * self.codes.shape[1] // self.scale.shape[0]


def _require(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _require_inference(*ts: torch.Tensor) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in ts):
        raise RuntimeError("operators in four bits are not differentiable: call them under torch.no_grad() or on detached tensors")


def _on(x: torch.Tensor):
    """Kernels are launched on the current stream of the device that holds the data, whichever device is current."""
    return contextlib.nullcontext() if x.device.index == torch.cuda.current_device() else torch.cuda.device(x.device)


def _check_cache(c: Int4Cache) -> Tuple[int, int, int, int]:
    _require(c.k.dim() == 4 and c.k_scale.dim() == 5, "an int4 cache has codes of 4 dimensions and scales of 5")
    B, H, cap, half = c.k.shape
    D = 2 * half
    _require(D % CACHE_GROUP == 0 and 0 < D <= CACHE_DIM and cap % CACHE_SLOTS == 0 and cap > 0 and H > 0,
             f"an int4 cache takes head dims in multiples of {CACHE_GROUP} up to {CACHE_DIM} and capacities in multiples of {CACHE_SLOTS}, got {D} and {cap}")
    for codes, scale in ((c.k, c.k_scale), (c.v, c.v_scale)):
        _require(codes.shape == c.k.shape and tuple(scale.shape) == (B, H, cap, D // CACHE_GROUP, 2),
                 "the parts of an int4 cache do not fit together")
        if codes.dtype != torch.uint8 or scale.dtype != torch.bfloat16:
            raise TypeError(f"an int4 cache has uint8 codes and bf16 scales, got {codes.dtype} and {scale.dtype}")
        _require(codes.is_contiguous() and scale.is_contiguous(), "the parts of an int4 cache must be contiguous")
        _require(codes.device == scale.device == c.k.device, "the parts of an int4 cache are on different devices")
        _require(codes.data_ptr() % 16 == 0 and scale.data_ptr() % 16 == 0, "the parts of an int4 cache must be 16-byte aligned")
    return B, H, cap, D


def _int32(x: torch.Tensor, shape, device, what: str) -> torch.Tensor:
    _require(tuple(x.shape) == tuple(shape), f"{what} has shape {tuple(x.shape)}, expected {tuple(shape)}")
    _require(x.device == device, f"{what} is on {x.device}, the cache on {device}")
    if x.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{what} must be int32 or int64, got {x.dtype}")
    if x.dtype == torch.int64:         # far outside the cache stays outside
        x = x.clamp(-(1 << 31), (1 << 31) - 1)
    return x.to(torch.int32).contiguous()


# =============================================================================== cache
def int4_cache(batch: int, kv_heads: int, capacity: int, head_dim: int, device=None) -> Int4Cache:
    """An empty cache (every slot stands for zeros) of at least ``capacity`` slots."""
    _require(0 < head_dim <= CACHE_DIM and head_dim % CACHE_GROUP == 0, f"head_dim {head_dim} is no multiple of {CACHE_GROUP} up to {CACHE_DIM}")
    _require(batch >= 0 and kv_heads > 0 and capacity > 0, "an int4 cache needs heads and slots")
    cap = -(-capacity // CACHE_SLOTS) * CACHE_SLOTS
    codes = lambda: torch.zeros(batch, kv_heads, cap, head_dim // 2, dtype=torch.uint8, device=device)
    scale = lambda: torch.zeros(batch, kv_heads, cap, head_dim // CACHE_GROUP, 2, dtype=torch.bfloat16, device=device)
    return Int4Cache(codes(), scale(), codes(), scale())


def int4_cache_write(cache: Int4Cache, k_new: torch.Tensor, v_new: torch.Tensor, slots: torch.Tensor,
                     distinct: bool = False) -> None:
    """``k_new`` / ``v_new`` ``[B, T, Hkv, D]`` (views of packed rows allowed) go, quantised, into slots ``slots[b, t]``.  Rows whose
    slot is negative or past the capacity are not written; of several rows of a sequence with one slot the last stays.
    ``distinct=True`` vouches that no slot occurs twice in a sequence (saves looking for it in calls of more than 64 rows)."""
    if _native.int4_cache_write(*cache, k_new, v_new, slots, distinct):
        return
    B, H, cap, D = _check_cache(cache)
    _require(k_new.dim() == 4 and k_new.shape == v_new.shape and k_new.shape[0] == B and tuple(k_new.shape[2:]) == (H, D),
             f"keys {tuple(k_new.shape)} and values {tuple(v_new.shape)} do not fit a cache of {B} x {H} heads of {D}")
    _require(k_new.device == v_new.device == cache.k.device, "rows and cache are on different devices")
    _require_inference(k_new, v_new)
    T = k_new.shape[1]
    slots = _int32(slots, (B, T), cache.k.device, "slots")
    if not k_new.is_cuda:
        for rows, codes, scale in ((k_new, cache.k, cache.k_scale), (v_new, cache.v, cache.v_scale)):
            c, s = ref.int4_quantize(rows, CACHE_GROUP)
            for b in range(B):
                for t, slot in enumerate(slots[b].tolist()):
                    if 0 <= slot < cap:
                        codes[b, :, slot], scale[b, :, slot] = c[b, t], s[b, t]
        return
    if k_new.dtype != torch.bfloat16 or v_new.dtype != torch.bfloat16:
        raise TypeError(f"the sm_100a kernels take bf16 rows, got {k_new.dtype} and {v_new.dtype}")
    if not (k_new.stride() == v_new.stride() and k_new.stride(3) == 1 and all(s % 8 == 0 for s in k_new.stride()[:3])
            and k_new.data_ptr() % 16 == 0 and v_new.data_ptr() % 16 == 0):
        k_new, v_new = k_new.clone(memory_format=torch.contiguous_format), v_new.clone(memory_format=torch.contiguous_format)
    with _on(k_new):
        table = not distinct and _lib.load().ksa_int4_cache_write_table(B, T, H, D, cap)
        last = torch.empty((B, cap), dtype=torch.int32, device=k_new.device) if table else None
        _lib.call("ksa_int4_cache_write", k_new, v_new, cache.k, cache.k_scale, cache.v, cache.v_scale, slots, last, B, T, H, D, cap,
                  k_new.stride(0), k_new.stride(1), k_new.stride(2), int(distinct))


def int4_qk_norm_rope_decode(qkv: torch.Tensor, q_w: Optional[torch.Tensor], k_w: Optional[torch.Tensor], pos: torch.Tensor, Hq: int, theta: float,
                             eps: float, interleaved: bool, cache: Int4Cache, slots: torch.Tensor) -> torch.Tensor:
    """``ops.qk_norm_rope_decode`` of rows ``[q | k | v]`` whose keys and values go, quantised, into ``cache``: those of row ``i < len(slots)``
    (sequence ``i``) into slot ``slots[i]``, as :func:`int4_cache_write` would write them; at head dim 128 in the same launch."""
    B, H, cap, D = _check_cache(cache)
    _require(qkv.dim() == 2 and qkv.shape[1] == (Hq + 2 * H) * D, f"rows {tuple(qkv.shape)} are not {Hq} query and twice {H} key heads of {D}")
    _require(qkv.device == cache.k.device, "rows and cache are on different devices")
    _require_inference(qkv)
    n = slots.numel()
    _require(n <= min(B, qkv.shape[0]), f"{n} slots for {qkv.shape[0]} rows and a cache of {B}")
    slots = _int32(slots.reshape(-1), (n,), cache.k.device, "slots")
    _require(pos.shape == qkv.shape[:1] and pos.device == qkv.device, f"positions {tuple(pos.shape)} for {qkv.shape[0]} rows")
    for w in (q_w, k_w):
        _require(w is None or (w.shape == (D,) and w.device == qkv.device), f"norm weights are {D} values beside the rows")
    if not qkv.is_cuda:
        return _rotate_then_write(qkv, q_w, k_w, pos, Hq, theta, eps, interleaved, cache, slots)
    for w in (q_w, k_w):
        _require(w is None or (w.dtype == qkv.dtype and w.is_contiguous() and w.data_ptr() % 4 == 0), f"norm weights are {D} contiguous bf16 values")
    pos = pos.to(torch.int32).contiguous()
    if qkv.stride(1) != 1 or qkv.stride(0) % 2 != 0 or qkv.data_ptr() % 4 != 0:            # pairs of values are read as words
        qkv = qkv.clone(memory_format=torch.contiguous_format)
    with _on(qkv):
        if D != 128 or qkv.dtype != torch.bfloat16:
            return _rotate_then_write(qkv, q_w, k_w, pos, Hq, theta, eps, interleaved, cache, slots)
        out = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device)
        _lib.call("ksa_qknorm_rope_decode_int4", qkv, out, q_w, k_w, pos, qkv.stride(0), out.stride(0), qkv.shape[0], Hq, H, D, float(theta), float(eps),
                  int(interleaved), cache.k, cache.k_scale, cache.v, cache.v_scale, slots, n, cap)
    return out


def _rotate_then_write(qkv, q_w, k_w, pos, Hq, theta, eps, interleaved, cache, slots):
    from . import qk_norm_rope_decode
    H, D, n = cache.k.shape[1], 2 * cache.k.shape[3], slots.numel()
    out = qk_norm_rope_decode(qkv, q_w, k_w, pos, Hq, H, D, theta, eps, interleaved)
    heads = out[:n, Hq * D:].view(n, 1, 2 * H, D)
    int4_cache_write(cache.rows(slice(0, n)), heads[:, :, :H], heads[:, :, H:], slots.view(n, 1))
    return out


def int4_cache_read(cache: Int4Cache, start: torch.Tensor, rows: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """The values of slots ``start[b] .. start[b] + rows`` of every sequence: ``(k, v)``, each ``[B, Hkv, rows, D]`` bf16; zeros for
    slots outside the cache."""
    made = _native.int4_cache_read(*cache, start, rows)
    if made is not None:
        return made
    B, H, cap, D = _check_cache(cache)
    _require(rows >= 0, f"{rows} rows")
    start = _int32(start, (B,), cache.k.device, "start")
    if not cache.k.is_cuda:
        at = start.long()[:, None] + torch.arange(rows)
        inside = ((at >= 0) & (at < cap))[:, None, :, None]
        b, at = torch.arange(B)[:, None], at.clamp(0, cap - 1)
        return tuple(torch.where(inside, ref.int4_values(c[b, :, at], s[b, :, at]).transpose(1, 2), torch.zeros((), dtype=torch.bfloat16))
                     for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    out = torch.empty((2, B, H, rows, D), dtype=torch.bfloat16, device=cache.k.device)
    with _on(cache.k):
        _lib.call("ksa_int4_cache_read", cache.k, cache.k_scale, cache.v, cache.v_scale, start, out[0], out[1], B, H, D, cap, rows)
    return out[0], out[1]


def int4_cache_move(cache: Int4Cache, src: torch.Tensor, dst: torch.Tensor, enable: torch.Tensor, rows: int) -> None:
    """Slots ``src[b] .. src[b] + rows`` go to ``dst[b] .. dst[b] + rows`` in the sequences with ``enable[b] != 0`` (all ``[B]``), as they
    are; slots outside the cache are left out.  The two ranges of a sequence must not overlap.  Head dims in multiples of 64."""
    B, H, cap, D = _check_cache(cache)
    _require(rows >= 0 and D % 64 == 0, f"{rows} rows of heads of {D} (a multiple of 64 is moved)")
    src, dst, enable = (_int32(x, (B,), cache.k.device, n) for x, n in ((src, "src"), (dst, "dst"), (enable, "enable")))
    if not cache.k.is_cuda:
        for b, (s, d, on) in enumerate(zip(src.tolist(), dst.tolist(), enable.tolist())):
            lo, hi = max(0, -s, -d), min(rows, cap - s, cap - d)
            if on and hi > lo:
                for t in cache:
                    t[b, :, d + lo:d + hi] = t[b, :, s + lo:s + hi].clone()
        return
    with _on(cache.k):
        _lib.call("ksa_int4_cache_move", cache.k, cache.k_scale, cache.v, cache.v_scale, src, dst, enable, B, H, D, cap, rows)


def int4_decode_attention(q: torch.Tensor, cache: Int4Cache, start: torch.Tensor, length: torch.Tensor,
                          scale: Optional[float] = None) -> torch.Tensor:
    """``q`` ``[B, Tq, Hq, D]``: query ``(b, t)`` attends slots ``start[b, t] .. start[b, t] + length[b, t]`` of sequence ``b``, cut to the
    cache, with no mask inside; zeros where no slot is left.  ``Hq`` is a multiple of the cache's heads; ``D`` is 64 or 128
    on a GPU; ``scale`` defaults to ``D ** -0.5``.  Slots outside a query's slice do not touch its result, whatever they hold.  A score below
    what fp32 holds is minus infinity, and NaN comes out where all of a slice are."""
    if q.dim() == 4 and q.shape[3] > 0:
        made = _native.int4_decode_attention(q, *cache, start, length, q.shape[3] ** -0.5 if scale is None else scale)
        if made is not None:
            return made
    B, Hkv, cap, D = _check_cache(cache)
    _require(q.dim() == 4 and q.shape[0] == B and q.shape[3] == D and q.shape[2] > 0 and q.shape[2] % Hkv == 0,
             f"queries {tuple(q.shape)} do not fit a cache of {B} x {Hkv} heads of {D}")
    _require(q.device == cache.k.device, "queries and cache are on different devices")
    _require_inference(q)
    Tq, Hq = q.shape[1], q.shape[2]
    start, length = _int32(start, (B, Tq), q.device, "start"), _int32(length, (B, Tq), q.device, "length")
    scale = D ** -0.5 if scale is None else float(scale)
    if not q.is_cuda:
        return ref.int4_decode_attention(q, cache.k, cache.k_scale, cache.v, cache.v_scale, start, length, scale)
    if q.dtype != torch.bfloat16:
        raise TypeError(f"the sm_100a kernels take bf16 queries, got {q.dtype}")
    _require(D in (64, 128), f"head_dim {D} unsupported (64 or 128)")
    if q.stride(3) != 1 or any(s % 8 for s in q.stride()[:3]) or q.data_ptr() % 16 != 0:
        q = q.clone(memory_format=torch.contiguous_format)
    out = torch.empty((B, Tq, Hq, D), dtype=q.dtype, device=q.device)
    with _on(q):
        n = _lib.load().ksa_int4_attn_workspace(B, Tq, Hq, Hkv, D, cap)
        workspace = torch.empty(n, dtype=torch.float32, device=q.device) if n > 0 else None
        _lib.call("ksa_int4_decode_attn", q, cache.k, cache.k_scale, cache.v, cache.v_scale, start, length, workspace, out, B, Tq, Hq, Hkv, D,
                  cap, q.stride(0), q.stride(1), q.stride(2), scale)
    return out


# =============================================================================== weights
def _check_weight(w: Int4Weight) -> Tuple[int, int, int, int]:
    codes, scale = w
    _require(codes.dim() == 2 and scale.dim() == 3 and scale.shape[2] == 2 and scale.shape[0] > 0,
             "an int4 weight has codes [N, K / 2] and scales [K / group, pitch, 2]")
    if codes.dtype != torch.uint8 or scale.dtype != torch.bfloat16:
        raise TypeError(f"an int4 weight has uint8 codes and bf16 scales, got {codes.dtype} and {scale.dtype}")
    (N, K), pitch = w.shape, scale.shape[1]
    _require(w.group in (32, 64, 128) and w.group * scale.shape[0] == K and pitch == -(-N // 4) * 4,
             f"scales {tuple(scale.shape)} do not fit codes {tuple(codes.shape)}")
    _require(codes.is_contiguous() and scale.is_contiguous() and codes.data_ptr() % 16 == 0 and scale.data_ptr() % 16 == 0,
             "the parts of an int4 weight must be contiguous and 16-byte aligned")
    _require(codes.device == scale.device, "the parts of an int4 weight are on different devices")
    return N, K, w.group, pitch


def int4_quantize_weight(weight: torch.Tensor, group: int = 64) -> Int4Weight:
    """``weight`` ``[N, K]`` (``K`` a multiple of ``group``: 32, 64 or 128) in four bits."""
    _require(weight.dim() == 2 and group in (32, 64, 128) and weight.shape[1] > 0 and weight.shape[1] % group == 0,
             f"a weight {tuple(weight.shape)} has no groups of {group} (32, 64 or 128) along its rows")
    weight = weight.detach()
    N, K = weight.shape
    pitch = -(-N // 4) * 4
    scale = torch.zeros((K // group, pitch, 2), dtype=torch.bfloat16, device=weight.device)
    if not weight.is_cuda:
        codes, s = ref.int4_quantize(weight, group)
        scale[:, :N] = s.transpose(0, 1)
        return Int4Weight(codes, scale)
    if weight.dtype != torch.bfloat16:
        raise TypeError(f"the sm_100a kernels take bf16 weights, got {weight.dtype}")
    if weight.stride(1) != 1 or weight.stride(0) % 8 != 0 or weight.data_ptr() % 16 != 0:
        weight = weight.clone(memory_format=torch.contiguous_format)
    codes = torch.empty((N, K // 2), dtype=torch.uint8, device=weight.device)
    with _on(weight):
        _lib.call("ksa_int4_weight", weight, codes, scale, N, K, group, weight.stride(0), pitch)
    return Int4Weight(codes, scale)


def int4_dequantize_weight(weight: Int4Weight) -> torch.Tensor:
    """The bf16 values ``[N, K]`` that ``weight`` stands for."""
    N, K, group, pitch = _check_weight(weight)
    if not weight.codes.is_cuda:
        return ref.int4_values(weight.codes, weight.scale[:, :N].transpose(0, 1))
    out = torch.empty((N, K), dtype=torch.bfloat16, device=weight.codes.device)
    _weight_values(weight, out)
    return out


def _weight_values(weight: Int4Weight, out: torch.Tensor) -> None:
    N, K = weight.shape
    with _on(out):
        _lib.call("ksa_int4_weight_values", weight.codes, weight.scale, out, N, K, weight.group, weight.scale.shape[1])


def int4_linear(x: torch.Tensor, weight: Int4Weight) -> torch.Tensor:
    """``x @ W.T`` for ``x`` ``[..., K]`` and ``W = int4_dequantize_weight(weight)``.  At most 32 rows (a decode step) read the codes
    once, some more in blocks of 32; many rows multiply with the bf16 values, written out for the call."""
    return _linear(x, weight, False)


def int4_linear_swiglu(x: torch.Tensor, w13: Int4Weight) -> torch.Tensor:
    """``swiglu(int4_linear(x, w13))`` with ``w13 = [gate rows | up rows]``; up to 16 rows in one launch."""
    return _linear(x, w13, True)


def int4_norm_linear(x: torch.Tensor, delta: Optional[torch.Tensor], norm_w: torch.Tensor, eps: float, weight: Int4Weight,
                     glu: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """``ops.norm_linear`` with a weight in four bits: ``res = x + delta`` (the first rows of ``x`` where ``delta`` has fewer), and the product
    of ``rms_norm(res, norm_w)`` (``glu``: of gate and up rows, with its activation).  Returns ``(res, y)``; for up to 4 rows in one launch."""
    from . import add_rms_norm, rms_norm
    N, K, group, pitch = _check_weight(weight)
    _require(x.dim() == 2 and x.shape[1] == K and norm_w.shape == (K,), f"rows {tuple(x.shape)} and norm {tuple(norm_w.shape)} do not fit a weight [{N}, {K}]")
    _require(delta is None or (delta.dim() == 2 and delta.shape[1] == K and delta.shape[0] <= x.shape[0]), "the added rows do not fit the rows")
    _require(not glu or N % 2 == 0, f"{N} rows are not as many gate as up rows")
    _require(all(t is None or t.device == weight.codes.device for t in (x, delta, norm_w)), "rows, norm and weight are on different devices")
    _require_inference(x, norm_w.detach(), *(() if delta is None else (delta,)))
    if not x.is_cuda:
        res, h = (x, rms_norm(x, norm_w.detach(), eps)) if delta is None else add_rms_norm(x, delta, norm_w.detach(), eps)
        return res, _linear(h, weight, glu)
    M, norm_w = x.shape[0], norm_w.detach()
    if not norm_w.is_contiguous() or norm_w.data_ptr() % 16 != 0:
        norm_w = norm_w.clone(memory_format=torch.contiguous_format)
    rows, delta = _aligned_rows(x), None if delta is None else _aligned_rows(delta)
    n = 0 if delta is None else delta.shape[0]
    if 0 < M <= NORM_ROWS and M * K <= NORM_VALUES and N > 0 and all(t is None or t.dtype == torch.bfloat16 for t in (x, delta, norm_w)):
        res = x if delta is None else torch.empty((M, K), dtype=x.dtype, device=x.device)
        y = torch.empty((M, N // 2 if glu else N), dtype=x.dtype, device=x.device)
        with _on(x):
            _lib.call("ksa_int4_norm_linear", rows, delta, norm_w, None if delta is None else res, weight.codes, weight.scale, y, M, N, K, group, pitch,
                      rows.stride(0), K if delta is None else delta.stride(0), K, y.shape[1], float(eps), n, int(glu))
        return res, y
    step = min(NORM_ROWS, NORM_VALUES // K)
    if step < M <= NORM_ROWS and step > 0:
        parts = [int4_norm_linear(rows[r:r + step], None if r >= n else delta[r:r + step], norm_w, eps, weight, glu) for r in range(0, M, step)]
        return x if delta is None else torch.cat([res for res, _ in parts]), torch.cat([y for _, y in parts])
    with _on(x):
        if K > 8192:               # wider than the norm's own kernel takes
            res = x if delta is None else torch.cat([(rows[:n].float() + delta.float()).to(x.dtype), rows[n:]])
            return res, _linear(ref.rms_norm(res, norm_w, eps), weight, glu)
        res, h = (x, rms_norm(rows, norm_w, eps)) if delta is None else add_rms_norm(rows, delta, norm_w, eps)
        return res, _linear(h, weight, glu)


def _aligned_rows(x: torch.Tensor) -> torch.Tensor:
    """``x`` ``[M, K]`` with rows that kernels can read: on 16 bytes, beside or behind one another."""
    return x if x.stride(1) == 1 and x.stride(0) % 8 == 0 and x.data_ptr() % 16 == 0 else x.clone(memory_format=torch.contiguous_format)


def _block_rows(N: int, K: int) -> int:
    """Rows up to which blocks of ``FEW_ROWS`` read the codes, once each.  More rows multiply with the bf16 values, written out for the call, at
    a cost that hardly depends on them.  Measured, values against blocks: a weight of ``[1280, 1280]`` 6.5 us against 9.3 for 32 rows,
    ``[2560, 4096]`` 13.7 against 10.3, ``[2560, 9728]`` 25.3 against 13.5, for 33 rows 13.7 against 15.0 and 25.5 against 21.0; what nearly fills
    the L2 cache, gate and up rows of ``[19456, 2560]``, 52 against 34 for 33 rows, 56 against 42 for 64, 58 against 61 for 96; values that outgrow it,
    ``[151936, 2560]``, 379 against 311 for 128 rows."""
    return FUSED_ROWS if N * K <= 4 << 20 else 32 if 2 * N * K <= 64 << 20 else 64 if 2 * N * K <= 126 << 20 else 128


def _linear(x: torch.Tensor, weight: Int4Weight, glu: bool) -> torch.Tensor:
    made = _native.int4_linear(x, *weight, glu)
    if made is not None:
        return made
    N, K, group, pitch = _check_weight(weight)
    _require(x.dim() >= 1 and x.shape[-1] == K, f"rows {tuple(x.shape)} do not fit a weight [{N}, {K}]")
    _require(not glu or N % 2 == 0, f"{N} rows are not as many gate as up rows")
    _require(x.device == weight.codes.device, "rows and weight are on different devices")
    _require_inference(x)
    if not x.is_cuda:
        y = ref.linear(x, int4_dequantize_weight(weight).to(x.dtype))
        return ref.swiglu(y) if glu else y
    if x.dtype != torch.bfloat16:
        raise TypeError(f"the sm_100a kernels take bf16 activations, got {x.dtype}")
    M, out_shape = x.numel() // K, (*x.shape[:-1], N // 2 if glu else N)
    if M == 0 or N == 0:
        return torch.empty(out_shape, dtype=x.dtype, device=x.device)
    if glu and FUSED_ROWS < M <= _block_rows(N, K):
        from . import swiglu
        y = _linear(x.reshape(M, K), weight, False)
        with _on(x):
            return (swiglu(y) if N % 16 == 0 else ref.swiglu(y)).view(out_shape)
    rows = _aligned_rows(x.reshape(M, K))
    if rows.stride(0) < K:
        rows = rows.clone(memory_format=torch.contiguous_format)
    if M > _block_rows(N, K):
        from . import linear, swiglu
        values = torch.empty((-(-N // 8) * 8, K), dtype=torch.bfloat16, device=x.device)       # the products take columns in eights
        values[N:].zero_()
        _weight_values(weight, values)
        with _on(x):
            y = linear(rows, values)
            if glu:
                gate, up = y[:, :N // 2], y[:, N // 2:N]
                y = swiglu(y) if N % 16 == 0 else ref.swiglu(torch.cat([gate, up], -1))
        return (y if glu or N % 8 == 0 else y[:, :N].contiguous()).view(out_shape)
    out = torch.empty((M, out_shape[-1]), dtype=x.dtype, device=x.device)
    with _on(x):
        for r in range(0, M, FEW_ROWS):
            part = rows[r:r + FEW_ROWS]
            _lib.call("ksa_int4_linear", part, weight.codes, weight.scale, out[r:], part.shape[0], N, K, group, pitch, rows.stride(0), out.shape[1],
                      int(glu))
    return out.view(out_shape)


__all__ = ["Int4Cache", "Int4Weight", "int4_cache", "int4_cache_write", "int4_qk_norm_rope_decode", "int4_cache_read", "int4_cache_move", "int4_decode_attention",
           "int4_quantize_weight", "int4_dequantize_weight", "int4_linear", "int4_linear_swiglu", "int4_norm_linear"]
