"""Performance cases of serving in four bits: a KV cache that is quantised as it is written, decode attention that reads it,
and projections whose weights are held in four bits.

A case has one of three kinds:

===========  =========================================================================================================
``cache``    ``T`` new rows of every sequence go into the cache (quantised) and the same slots are read back
``attend``   decode attention over a slice ``[start, start + length)`` of the cache for every sequence and query token
``linear``   ``x @ W.T`` of a few rows ``x`` with ``W`` in four bits
===========  =========================================================================================================

Format.  A group (32 values along the head dimension; ``group`` values along K for weights) with least value ``lo`` and
greatest ``hi`` has a scale ``S = bf16((hi - lo) / 15 * 16)`` (0 below 2^-100) and an offset ``O = bf16(lo - S)``; a code
``c = rint((x - O) / S * 16) - 16``, cut to 0 .. 15, stands for ``bf16(S * (1 + c / 16) + O)``.  Eight codes make a 32-bit
word, nibbles 0 .. 7 from the lowest being values 0, 2, 4, 6, 1, 3, 5, 7.  Cache: codes ``[B, H, cap, D / 2]`` uint8, scales
``[B, H, cap, D / 32, 2]`` bf16 (S, O).  Weights: codes ``[N, K / 2]``, scales ``[K / group, N rounded up to 4, 2]``.

Widths are those of the presets "ksa-4b" (32 query and 8 key heads of 128, width 2560, feed-forward 9728, vocabulary 151936),
"qwen3-1.9b-ksa" (16 and 8 heads) and "qwen3-ksa-tiny" (heads of 64).
"""
from __future__ import annotations

import math

import torch

own = False

GROUP = 32                    # values of a cache row that share a scale
LEAST = 2.0 ** -100


def listed():
    return [
        # one user decoding: a layer's new key and value row
        {"name": "cache_step_1", "kind": "cache", "B": 1, "T": 1, "H": 8, "D": 128, "cap": 2048},
        # a server's batch decoding together, each sequence at its own slot
        {"name": "cache_step_64", "kind": "cache", "B": 64, "T": 1, "H": 8, "D": 128, "cap": 1168},
        # ragged prompts of a small model: heads of 64
        {"name": "cache_prompt_3x1501", "kind": "cache", "B": 3, "T": 1501, "H": 2, "D": 64, "cap": 1600},
        # a long prompt goes into a full-attention layer's cache
        {"name": "cache_prompt_32767", "kind": "cache", "B": 1, "T": 32767, "H": 8, "D": 128, "cap": 32768},
        # a summary layer's slice of one user: current chunk, ring of eight chunks, some summaries
        {"name": "attend_ksa_1", "kind": "attend", "B": 1, "Tq": 1, "Hq": 32, "H": 8, "D": 128, "cap": 1424, "fill": 1181},
        # a chunk boundary: the text token and the summary token of four sequences, two of which do not close a chunk
        {"name": "attend_boundary_4", "kind": "attend", "B": 4, "Tq": 2, "Hq": 16, "H": 8, "D": 128, "cap": 1296, "fill": 1201},
        # ragged batch on a full-attention layer
        {"name": "attend_full_24", "kind": "attend", "B": 24, "Tq": 1, "Hq": 16, "H": 8, "D": 128, "cap": 8192, "fill": 8000},
        # one user at the longest context
        {"name": "attend_full_128k", "kind": "attend", "B": 1, "Tq": 1, "Hq": 32, "H": 8, "D": 128, "cap": 131072, "fill": 131071},
        # a batch of long contexts
        {"name": "attend_full_16x32k", "kind": "attend", "B": 16, "Tq": 1, "Hq": 32, "H": 8, "D": 128, "cap": 32768, "fill": 32768},
        # the projections of a decode step: queries, keys and values of one row
        {"name": "linear_qkv_1", "kind": "linear", "M": 1, "N": 6144, "K": 2560, "group": 64},
        # the second feed-forward product of a few rows
        {"name": "linear_down_5", "kind": "linear", "M": 5, "N": 2560, "K": 9728, "group": 64},
        # the output head of a batch
        {"name": "linear_head_16", "kind": "linear", "M": 16, "N": 151936, "K": 2560, "group": 128},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 8, 128), (16, 8, 128), (16, 16, 128), (32, 2, 128), (4, 2, 64), (16, 2, 64)]


def draw(rng):
    kind = rng.choice(["cache", "attend", "attend", "linear", "linear"])
    if kind == "linear":
        group = rng.choice([32, 64, 128])
        K = group * max(1, _log(rng, 256, 10240) // group)
        N = _log(rng, 200, min(160000, 151936 * 2560 // K))
        return {"kind": kind, "M": _log(rng, 1, 16), "N": N, "K": K, "group": group}
    Hq, H, D = rng.choice(HEADS)
    if kind == "cache":
        T = rng.choice([1, 1, 2, _log(rng, 3, 32767)])
        B = _log(rng, 1, max(1, min(128, 32767 * 8 * 128 // (T * H * D))))
        return {"kind": kind, "B": B, "T": T, "H": H, "D": D, "cap": (T + rng.randint(0, 900) + 15) // 16 * 16}
    Tq = rng.choice([1, 1, 1, 2])
    fill = _log(rng, 100, 131072)
    B = _log(rng, 1, max(1, min(96, 16 * 32768 * 8 * 128 // (fill * H * D * Tq * max(1, Hq // H // 8)))))
    return {"kind": kind, "B": B, "Tq": Tq, "Hq": Hq, "H": H, "D": D, "cap": (fill + rng.randint(0, 200) + 15) // 16 * 16, "fill": fill}


# ------------------------------------------------------------------------------------------------- the format, plainly
def _quantize(x, group):
    """bf16 values ``[..., n]`` -> codes ``[..., n]`` (fp32 whole numbers) and scale, offset ``[..., n / group]`` bf16."""
    x = x.float().unflatten(-1, (-1, group))
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s = ((hi - lo) / torch.full_like(lo, 15) * 16).bfloat16().float()         # (by a number, it is a product with 1 / 15 on a GPU)
    s = torch.where(s < LEAST, torch.zeros_like(s), s)
    o = (lo - s).bfloat16().float()
    c = torch.where(s > 0, ((x - o) / s * 16).round() - 16, torch.zeros_like(x)).clamp(0, 15)
    return c.flatten(-2), s[..., 0].bfloat16(), o[..., 0].bfloat16()


def _pack(c):
    """Whole numbers 0 .. 15 ``[..., n]`` -> bytes ``[..., n / 2]``."""
    c = c.to(torch.uint8).unflatten(-1, (-1, 8))
    return (c[..., [0, 4, 1, 5]] | (c[..., [2, 6, 3, 7]] << 4)).flatten(-2)


def _unpack(b):
    b = b.unflatten(-1, (-1, 4))
    return torch.cat([b & 15, b >> 4], -1)[..., [0, 2, 4, 6, 1, 3, 5, 7]].flatten(-2)


def _values(codes, s, o):
    """What bytes ``[..., n / 2]`` stand for, with scales and offsets ``[..., groups]``, as fp32 (bf16 values)."""
    u = (1 + _unpack(codes).float() / 16).unflatten(-1, (s.shape[-1], -1))
    return (u * s.float()[..., None] + o.float()[..., None]).bfloat16().float().flatten(-2)


def _weight(codes, scale):
    """fp32 ``[N, K]`` of a weight's codes and scales."""
    s = scale[:, :codes.shape[0]].transpose(0, 1)
    return _values(codes, s[..., 0], s[..., 1])


# ------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(g, *shape):
    """Keys or values: channels of unlike spread, a few of them far from zero, as trained projections give them."""
    d = shape[-1]
    spread = torch.exp(0.4 * torch.randn(d, generator=g, device="cuda"))
    shift = torch.randn(d, generator=g, device="cuda") * (torch.rand(d, generator=g, device="cuda") < 0.1) * 3
    x = torch.randn(*shape, generator=g, device="cuda", dtype=torch.bfloat16)
    return x.mul_(spread.bfloat16()).add_(shift.bfloat16())


def _filled(g, *shape):
    c, s, o = _quantize(_rows(g, *shape), GROUP)
    return _pack(c), torch.stack([s, o], -1)


def prepare(case, seed):
    g = _gen(seed)
    st = {"case": case}
    if case["kind"] == "linear":
        M, N, K, group = case["M"], case["N"], case["K"], case["group"]
        w = torch.randn(N, K, generator=g, device="cuda", dtype=torch.bfloat16).mul_(0.02)
        c, s, o = _quantize(w, group)
        st["codes"] = _pack(c)
        st["scale"] = torch.zeros(K // group, (N + 3) // 4 * 4, 2, dtype=torch.bfloat16, device="cuda")
        st["scale"][:, :N, 0], st["scale"][:, :N, 1] = s.t(), o.t()
        st["x"] = torch.randn(M, K, generator=g, device="cuda", dtype=torch.bfloat16)
        return st
    B, H, D, cap = case["B"], case["H"], case["D"], case["cap"]
    if case["kind"] == "cache":
        T = case["T"]
        for n in ("k", "v"):
            st[n] = torch.zeros(B, H, cap, D // 2, dtype=torch.uint8, device="cuda")
            st[n + "_scale"] = torch.zeros(B, H, cap, D // GROUP, 2, dtype=torch.bfloat16, device="cuda")
        # rows of a projection: all keys, then all values of a row
        st["rows"] = torch.cat([_rows(g, B, T, H, D), _rows(g, B, T, H, D)], 2)
        st["start"] = torch.randint(0, cap - T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        st["slots"] = st["start"][:, None] + torch.arange(T, device="cuda", dtype=torch.int32)
        return st
    Tq, fill = case["Tq"], case["fill"]
    for n in ("k", "v"):
        st[n], st[n + "_scale"] = _filled(g, B, H, cap, D)
    st["q"] = torch.randn(B, Tq, case["Hq"], D, generator=g, device="cuda", dtype=torch.bfloat16)
    u = torch.rand(B, Tq, generator=g, device="cuda")
    n = (fill * (0.5 + 0.5 * u)).to(torch.int32).clamp(min=1)
    n[0, 0] = fill
    at = ((fill - n) * torch.rand(B, Tq, generator=g, device="cuda")).to(torch.int32)
    if Tq > 1:                 # the later queries: a short slice, and none for every other sequence
        n[:, 1:] = torch.clamp(n[:, 1:] // 8, min=1)
        n[1::2, 1:] = 0
        at[:, 1:] = 0
    st["start"], st["length"] = at, n
    return st


# ------------------------------------------------------------------------------------------------- one pass
def run(st):
    case = st["case"]
    if own:
        return _own(st, case)
    if case["kind"] == "linear":
        return (st["x"].float() @ _weight(st["codes"], st["scale"]).t()).bfloat16()
    if case["kind"] == "cache":
        H, out = case["H"], []
        b = torch.arange(case["B"], device="cuda")[:, None]
        at = st["slots"].long()
        for n, rows in (("k", st["rows"][:, :, :H]), ("v", st["rows"][:, :, H:])):
            c, s, o = _quantize(rows, GROUP)
            st[n][b, :, at] = _pack(c)
            st[n + "_scale"][b, :, at] = torch.stack([s, o], -1)
            meta = st[n + "_scale"][b, :, at]
            out.append(_values(st[n][b, :, at], meta[..., 0], meta[..., 1]).bfloat16().transpose(1, 2).contiguous())
        return out
    r = case["Hq"] // case["H"]
    q = st["q"].float().unflatten(2, (case["H"], r))
    slot = torch.arange(case["cap"], device="cuda")
    seen = (slot >= st["start"][..., None]) & (slot < (st["start"] + st["length"])[..., None])       # [B, Tq, cap]
    z = torch.einsum("bthrd,bhkd->bthrk", q, _values(st["k"], st["k_scale"][..., 0], st["k_scale"][..., 1])) / math.sqrt(case["D"])
    z = z.masked_fill(~seen[:, :, None, None], -math.inf)
    p = torch.exp(z - z.amax(-1, keepdim=True).clamp(min=-1e30))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    out = torch.einsum("bthrk,bhkd->bthrd", p, _values(st["v"], st["v_scale"][..., 0], st["v_scale"][..., 1]))
    return out.flatten(2, 3).bfloat16()


def _own(st, case):
    from ksa_b200 import ops
    if case["kind"] == "linear":
        return ops.int4_linear(st["x"], ops.Int4Weight(st["codes"], st["scale"]))
    cache = ops.Int4Cache(st["k"], st["k_scale"], st["v"], st["v_scale"])
    if case["kind"] == "cache":
        H = case["H"]
        ops.int4_cache_write(cache, st["rows"][:, :, :H], st["rows"][:, :, H:], st["slots"])
        return list(ops.int4_cache_read(cache, st["start"], case["T"]))
    return ops.int4_decode_attention(st["q"], cache, st["start"], st["length"])


# ------------------------------------------------------------------------------------------------- what a pass needs
def work(case):
    if case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": N * K * (0.5 + 4.0 / case["group"]) + 2.0 * M * (K + N), "flops": 2.0 * M * N * K}
    H, D = case["H"], case["D"]
    if case["kind"] == "cache":
        n = 2 * case["B"] * case["T"] * H * D
        return {"bytes": n * (2 + 0.625 + 0.625 + 2.0) + 4.0 * case["B"] * case["T"], "flops": 12.0 * n}
    # the slices' lengths come from the seed: the first is the longest, the others half of it to all of it, three quarters on average;
    # the short slices of the later queries lie within or beside them
    B, Tq = case["B"], case["Tq"]
    slots = case["fill"] * (1 + 0.75 * (B - 1)) + (Tq - 1) * ((B + 1) // 2) * case["fill"] * 0.75 / 8
    return {"bytes": slots * H * 2 * D * 0.625 + 4.0 * B * Tq * case["Hq"] * D, "flops": 4.0 * slots * case["Hq"] * D}


# ------------------------------------------------------------------------------------------------- the same in 64 bits
ORDER = (0, 2, 4, 6, 1, 3, 5, 7)             # the value that nibble 0, 1, ... of a word holds


def _bf16(x):
    """64-bit values rounded to eight significant bits, ties to even."""
    m, e = torch.frexp(x)
    return torch.ldexp(torch.round(m * 256), e - 8)


def _decode64(codes, s, o):
    """Words of eight codes -> 64-bit values: each value is looked up by its nibble's place in the word."""
    words = codes.contiguous().view(torch.int32).long() & 0xFFFFFFFF
    c = torch.empty(*words.shape, 8, dtype=torch.float64, device=codes.device)
    for nibble, value in enumerate(ORDER):
        c[..., value] = (words >> (4 * nibble)) & 15
    c = c.flatten(-2)
    n = c.shape[-1] // s.shape[-1]
    s, o = s.double().repeat_interleave(n, -1), o.double().repeat_interleave(n, -1)
    return _bf16(o + s + s * c / 16)


def _round_trip64(x):
    """What the values of the last axis become in the cache, from the definition of the format."""
    v = x.double().reshape(-1, GROUP)
    lo, hi = v.min(1, keepdim=True).values, v.max(1, keepdim=True).values
    s = _bf16((hi - lo) * 16 / 15)
    s = s * (s >= LEAST)
    o = _bf16(lo - s)
    c = torch.round((v - o) * 16 / s.clamp(min=LEAST)).clamp(16, 31) * (s > 0)
    return _bf16(o + s * c / 16).reshape(x.shape)


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "linear":
        N = case["N"]
        y = torch.empty(case["M"], N, dtype=torch.float64, device="cuda")
        step = max(1, (1 << 27) // case["K"])
        for lo in range(0, N, step):
            hi = min(N, lo + step)
            w = _decode64(st["codes"][lo:hi], st["scale"][:, lo:hi, 0].t(), st["scale"][:, lo:hi, 1].t())
            y[:, lo:hi] = st["x"].double() @ w.t()
        return y
    if case["kind"] == "cache":
        H = case["H"]
        return [_round_trip64(st["rows"][:, :, i * H:(i + 1) * H]).transpose(1, 2).contiguous() for i in range(2)]
    B, Tq, Hq, H, D = (case[n] for n in ("B", "Tq", "Hq", "H", "D"))
    out = torch.zeros(B, Tq, Hq, D, dtype=torch.float64, device="cuda")
    starts, lengths = st["start"].tolist(), st["length"].tolist()
    for b in range(B):
        k, v = (_decode64(st[n][b], st[n + "_scale"][b, ..., 0], st[n + "_scale"][b, ..., 1]) for n in ("k", "v"))
        for t in range(Tq):
            lo, n = starts[b][t], lengths[b][t]
            if n == 0:
                continue
            q = st["q"][b, t].double().view(H, Hq // H, D)
            w = torch.softmax(q @ k[:, lo:lo + n].transpose(1, 2) / math.sqrt(D), -1)
            out[b, t] = (w @ v[:, lo:lo + n]).reshape(Hq, D)
    return out
