"""Performance cases of a post-training step: log probabilities of given tokens under the output head, the clipped policy loss
with a KL term, the preference loss of pairs, and the global gradient norm with clipping.

A case has one of four kinds:

==============  ======================================================================================================
``log_probs``   ``y_t = log softmax(h_t W^T / tau)[label_t]`` of ``T`` rows, 0 where the label is -100; ``train``: with the
                gradients of ``h`` and ``W`` for a given gradient of ``y``
``policy``      clipped policy loss with a KL term against a reference model, and its gradient for every token
``preference``  loss of paired answers (sequences 2 i and 2 i + 1: preferred and rejected), and its gradient for every token
``norm``        global 2-norm of many gradients; ``place``: clipped in place, ``out``: the clipped ones into other buffers
==============  ======================================================================================================

Formulas.  Policy: ``d = y - y_old``, ``r = exp(d)``, ``L = -min(r A, clip(r, 1 - low, 1 + high) A)``, ``x = y_ref - y``,
``K = exp(x) - 1 - x``; the loss is the mean of ``L + kl_coef K`` over valid tokens, or the mean over the sequences that have
one of each sequence's mean.  Statistics: the means of ``L``, ``K`` and of ``L`` being cut off.  Preference: ``D_s`` is the sum
of ``y - y_ref`` over the valid tokens of sequence ``s``, ``z_i = beta (D_2i - D_2i+1)``, and the loss the mean of
``softplus(-z_i) + smoothing z_i``; rewards are ``beta D_s``.  Clipping: gradients times ``min(1, most / (norm + 1e-6))``.

Widths and vocabularies are those of the presets "ksa-4b" (2560, 151936), "qwen3-1.9b-ksa" (2048, 151936) and "qwen3-ksa-tiny"
(256, 4096).
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

IGNORE = -100


def listed():
    return [
        # one answer token of one user is scored under a reference model: the weights are the whole cost
        {"name": "score_1", "kind": "log_probs", "T": 1, "D": 2560, "V": 151936, "answer": 1.0, "turns": 1, "tau": 1.0, "train": False},
        # a few short answers of a ragged batch, sampled at another temperature
        {"name": "score_77", "kind": "log_probs", "T": 77, "D": 2048, "V": 151936, "answer": 0.8, "turns": 3, "tau": 0.7, "train": False},
        # a long rollout under the old policy: what the step's ratios are taken against
        {"name": "score_8192", "kind": "log_probs", "T": 8192, "D": 2048, "V": 151936, "answer": 1.0, "turns": 1, "tau": 1.0, "train": False},
        # a small model's step on a ragged batch
        {"name": "train_333_small", "kind": "log_probs", "T": 333, "D": 256, "V": 4096, "answer": 0.7, "turns": 4, "tau": 1.0, "train": True},
        # a training step on conversations: prompts and tool answers are masked
        {"name": "train_8192", "kind": "log_probs", "T": 8192, "D": 2048, "V": 151936, "answer": 0.6, "turns": 5, "tau": 1.0, "train": True},
        # a small rollout batch, padded: one advantage for each sequence, no reference model
        {"name": "policy_4x257", "kind": "policy", "S": 4, "L": 257, "packed": False, "ref": False, "by_sequence": True, "adv": "sequence"},
        # a large rollout batch: many long answers packed behind one another, with the KL term
        {"name": "policy_256x16000", "kind": "policy", "S": 256, "L": 16000, "packed": True, "ref": True, "by_sequence": False, "adv": "token"},
        # a few pairs, packed
        {"name": "preference_4", "kind": "preference", "S": 8, "L": 611, "packed": True, "ref": True, "smooth": 0.0},
        # many long pairs, padded, with uncertain labels
        {"name": "preference_64x8192", "kind": "preference", "S": 128, "L": 8192, "packed": False, "ref": True, "smooth": 0.1},
        # the flat fp32 buffers of a trained model's layers: the norm that the optimizer clips by
        {"name": "norm_units", "kind": "norm", "n": 30, "total": 1_900_000_000, "ragged": False, "dtype": "float32", "to": "norm"},
        # every parameter of a small model by itself, in two types, clipped in place
        {"name": "clip_parameters_61", "kind": "norm", "n": 61, "total": 2_500_000, "ragged": True, "dtype": "mixed", "to": "place"},
        # every parameter of a large model, clipped into the optimizer's buffers
        {"name": "clip_parameters_400", "kind": "norm", "n": 400, "total": 1_200_000_000, "ragged": True, "dtype": "bfloat16", "to": "out"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["log_probs", "log_probs", "policy", "preference", "norm"])
    if kind == "log_probs":
        D = 8 * _log(rng, 16, 320)
        V = _log(rng, 1000, 151936)
        T = _log(rng, 1, max(2, min(32768, 8192 * 151936 // V)))
        return {"kind": kind, "T": T, "D": D, "V": V, "answer": rng.choice([1.0, 0.9, 0.5, 0.2]), "turns": rng.randint(1, 6),
                "tau": rng.choice([1.0, 1.0, 0.6]), "train": rng.random() < 0.5}
    if kind == "policy":
        S = _log(rng, 1, 512)
        return {"kind": kind, "S": S, "L": _log(rng, 1, max(2, min(65536, 256 * 16000 // S))), "packed": rng.random() < 0.5, "ref": rng.random() < 0.5,
                "by_sequence": rng.random() < 0.5, "adv": rng.choice(["token", "sequence"])}
    if kind == "preference":
        S = 2 * _log(rng, 1, 128)
        return {"kind": kind, "S": S, "L": _log(rng, 1, max(2, min(65536, 128 * 8192 // S))), "packed": rng.random() < 0.5, "ref": rng.random() < 0.8,
                "smooth": rng.choice([0.0, 0.1])}
    n = _log(rng, 1, 500)
    return {"kind": kind, "n": n, "total": max(n, _log(rng, 100, 1_200_000_000)), "ragged": rng.random() < 0.6,
            "dtype": rng.choice(["float32", "bfloat16", "float16", "mixed"]), "to": rng.choice(["norm", "place", "out"])}


# ------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _answered(case):
    """Which rows have a label: the last part of every turn (a fixed number of rows, whatever the seed)."""
    T, turn = case["T"], -(-case["T"] // case["turns"])
    return (np.arange(T) % turn) >= int(turn * (1 - case["answer"]))


def _lengths(case):
    """Lengths of the sequences: packed ones differ, and some have no token at all; padded ones have rows of one length."""
    S, L = case["S"], case["L"]
    if not case["packed"]:
        return np.full(S, L)
    lengths = np.maximum(1, L * (np.arange(S) * 7 % 11 + 3) // 13)
    lengths[4::50] = 0
    return lengths


def _log_probs_inputs(case, g):
    T, D, V = case["T"], case["D"], case["V"]
    w = (0.02 * torch.randn(V, D, generator=g, device="cuda")).bfloat16()
    given = torch.randint(0, V, (T,), generator=g, device="cuda")
    # a trained model gives the tokens that it sampled a high score, some of them nearly the whole mass
    pull = torch.rand(T, 1, generator=g, device="cuda") * 8 / (D * 4e-4) * case["tau"]
    h = (torch.randn(T, D, generator=g, device="cuda") * (100 / math.sqrt(D)) + pull * w[given].float()).bfloat16()
    labels = torch.where(torch.from_numpy(_answered(case)).cuda(), given, torch.full_like(given, IGNORE))
    s = {"kind": "log_probs", "h": h, "w": w, "labels": labels, "tau": case["tau"], "train": case["train"]}
    if case["train"]:
        s["dy"] = torch.randn(T, generator=g, device="cuda") / T
        s["h"].requires_grad_(True)
        s["w"].requires_grad_(True)
    return s


def _token_inputs(case, g):
    """Log probabilities of the answers' tokens under the policy, and under an older and a reference model."""
    lengths = _lengths(case)
    S, n = len(lengths), int(lengths.sum())
    behind = 5 if case["packed"] else 0                        # tokens behind the last sequence belong to none
    y = -torch.rand(n + behind, generator=g, device="cuda").pow(3) * 9
    drift = lambda by: (y + by * torch.randn(y.shape, generator=g, device="cuda")).clamp(max=0)  # noqa: E731
    s = {"y": y, "old": drift(0.12), "ref": drift(0.25) if case["ref"] else None,
         "mask": torch.rand(y.shape, generator=g, device="cuda") < 0.85, "cu": None}
    s["of"] = torch.repeat_interleave(torch.arange(S, device="cuda"), torch.from_numpy(lengths).cuda())
    if case["packed"]:
        s["cu"] = torch.from_numpy(np.concatenate([[0], np.cumsum(lengths)])).to(device="cuda", dtype=torch.int32)
    else:
        for k in ("y", "old", "ref", "mask"):
            s[k] = None if s[k] is None else s[k].view(S, case["L"])
    s["y"].requires_grad_(True)
    s["S"] = S
    return s


def _gradient_inputs(case, g):
    n, total = case["n"], case["total"]
    if case["ragged"]:              # norm weights beside matrices, lengths of no round number, one of nothing
        share = np.array([(1.0 if k % 4 else 1e-3) * (1 + k * 5 % 7) for k in range(n)])
        sizes = np.maximum(1, (share / share.sum() * total).astype(np.int64))
        if n > 3:
            sizes[3] = 0
    else:
        sizes = np.full(n, max(1, total // n))
    types = [torch.bfloat16 if case["dtype"] == "mixed" and k % 3 == 0 else torch.float32 if case["dtype"] == "mixed" else getattr(torch, case["dtype"])
             for k in range(n)]
    # all gradients of a type lie in one buffer, as an optimizer over flat buffers keeps them: odd sizes begin at odd places
    step = 1 if case["ragged"] else 128
    flat, views = {}, []
    for t in sorted(set(types), key=str):
        at, begin = 0, {}
        for k in range(n):
            if types[k] == t:
                begin[k], at = at, at + -(-int(sizes[k]) // step) * step
        flat[str(t)] = (0.02 * torch.randn(at, generator=g, device="cuda")).to(t)
        views += [(k, flat[str(t)][b:b + int(sizes[k])]) for k, b in begin.items()]
    grads = [v for _, v in sorted(views, key=lambda x: x[0])]
    s = {"grads": grads, "flat": flat, "most": 0.3 * 0.02 * math.sqrt(total), "to": case["to"]}         # about a third of the norm
    if case["to"] == "out":
        s["flat"] = {t: torch.zeros_like(b) for t, b in flat.items()}
        s["out"] = [s["flat"][str(x.dtype)][x.storage_offset():x.storage_offset() + x.numel()] for x in grads]
    return s


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    if kind == "log_probs":
        return _log_probs_inputs(case, g)
    if kind == "norm":
        return {"kind": kind, **_gradient_inputs(case, g)}
    s = _token_inputs(case, g)
    s["kind"] = kind
    if kind == "policy":
        s["by"], s["kl"] = ("sequence" if case["by_sequence"] else "token"), (0.04 if case["ref"] else 0.0)
        s["adv"] = torch.randn(s["S"] if case["adv"] == "sequence" else s["y"].shape, generator=g, device="cuda")
    else:
        s["smooth"], s["beta"] = case["smooth"], 0.5 / math.sqrt(case["L"])
    return s


# ------------------------------------------------------------------------------------------------- plain forms
def _plain_log_probs(s):
    with torch.no_grad():
        h, w, at = s["h"].float(), s["w"].float(), s["labels"].clamp(min=0)[:, None]
        said = s["labels"] != IGNORE
        x = h @ w.T / s["tau"]
        x -= x.amax(1, keepdim=True)
        total = x.exp().sum(1, keepdim=True)
        y = torch.where(said, (x.gather(1, at) - total.log())[:, 0], torch.zeros((), device=h.device))
        if not s["train"]:
            return {"y": y}
        g = torch.where(said, s["dy"], torch.zeros((), device=h.device))[:, None] / s["tau"]
        dx = x.exp_().div_(total).mul_(-g).scatter_add_(1, at, g)
        return {"y": y, "dh": (dx @ w).bfloat16(), "dw": (dx.T @ h).bfloat16()}


def _plain_policy(s):
    """The clipped policy loss.  The differences are taken in 64 bits: a token on the border of the clipped range falls on one side of it."""
    with torch.no_grad():
        n, S, of = s["of"].numel(), s["S"], s["of"]
        flat = lambda t: t.reshape(-1)[:n].double()  # noqa: E731
        y, m = flat(s["y"]), s["mask"].reshape(-1)[:n]
        a = s["adv"].double()[of] if s["adv"].numel() == S and s["adv"].shape != s["y"].shape else flat(s["adv"])
        d = y - flat(s["old"])
        cut = ((a > 0) & (d > math.log1p(0.2))) | ((a < 0) & (d < math.log1p(-0.2)))
        r = d.exp()
        L = -torch.minimum(r * a, r.clamp(0.8, 1.2) * a)
        dL = torch.where(cut, torch.zeros_like(r), -r * a)
        x = flat(s["ref"]) - y if s["ref"] is not None else torch.zeros_like(y)
        K, dK = torch.expm1(x) - x, -torch.expm1(x)
        if s["by"] == "token":
            weight = m / m.sum().clamp(min=1)
        else:
            count = torch.zeros(S, dtype=torch.float64, device=y.device).index_add_(0, of, m.double())
            weight = m / (count.clamp(min=1) * (count > 0).sum().clamp(min=1))[of]
        mean = lambda v: torch.where(m, v * weight, torch.zeros_like(v)).sum()  # noqa: E731
        stats = torch.stack([mean(L), mean(K), mean(cut.double())])
        dy = torch.zeros(s["y"].numel(), dtype=torch.float32, device=y.device)
        dy[:n] = torch.where(m, (dL + s["kl"] * dK) * weight, torch.zeros_like(y)).float()
        return {"loss": (stats[0] + s["kl"] * stats[1]).float(), "stats": stats.float(), "dy": dy.view(s["y"].shape)}


def _plain_preference(s):
    """The loss of pairs.  Sums over long answers are taken in 64 bits: what counts is the difference of two of them."""
    with torch.no_grad():
        n, S, of = s["of"].numel(), s["S"], s["of"]
        flat = lambda t: t.reshape(-1)[:n].double()  # noqa: E731
        m = s["mask"].reshape(-1)[:n]
        v = flat(s["y"]) - (flat(s["ref"]) if s["ref"] is not None else 0.0)
        total = torch.zeros(S, dtype=torch.float64, device=v.device).index_add_(0, of, torch.where(m, v, torch.zeros_like(v)))
        rewards = s["beta"] * total.view(S // 2, 2)
        z = rewards[:, 0] - rewards[:, 1]
        loss = (torch.log1p(torch.exp(-z.abs())) + (-z).clamp(min=0) + s["smooth"] * z).mean()
        dz = (s["smooth"] - 1 / (1 + torch.exp(z))) * s["beta"] / (S // 2)
        per = torch.stack([dz, -dz], 1).view(-1)
        dy = torch.zeros(s["y"].numel(), dtype=torch.float32, device=v.device)
        dy[:n] = torch.where(m, per[of], torch.zeros_like(v)).float()
        return {"loss": loss.float(), "rewards": rewards.float(), "dy": dy.view(s["y"].shape)}


def _plain_norm(s):
    norm = torch.stack([x.float().square().sum() for x in s["grads"]]).sum().sqrt()
    if s["to"] == "norm":
        return {"norm": norm}
    factor = (s["most"] / (norm + 1e-6)).clamp(max=1.0)
    to = s["grads"] if s["to"] == "place" else s["out"]
    [o.copy_(x.float() * factor) for o, x in zip(to, s["grads"])]
    return {"norm": norm, "clipped": s["flat"]}


# ------------------------------------------------------------------------------------------------- one pass
def _own_log_probs(s):
    from ksa_b200 import ops
    if not s["train"]:
        with torch.no_grad():
            return {"y": ops.linear_log_probs(s["h"], s["w"], s["labels"], temperature=s["tau"])}
    y = ops.linear_log_probs(s["h"], s["w"], s["labels"], temperature=s["tau"])
    dh, dw = torch.autograd.grad(y, (s["h"], s["w"]), s["dy"])
    return {"y": y.detach(), "dh": dh, "dw": dw}


def _own_policy(s):
    from ksa_b200 import ops
    loss, stats = ops.policy_loss(s["y"], s["old"], s["adv"], ref_log_probs=s["ref"], mask=s["mask"], cu_seqlens=s["cu"],
                                  clip_low=0.2, clip_high=0.2, kl_coef=s["kl"], reduction=s["by"])
    dy, = torch.autograd.grad(loss, s["y"])
    return {"loss": loss.detach(), "stats": stats, "dy": dy}


def _own_preference(s):
    from ksa_b200 import ops
    loss, rewards = ops.preference_loss(s["y"], s["ref"], mask=s["mask"], cu_seqlens=s["cu"], beta=s["beta"], label_smoothing=s["smooth"])
    dy, = torch.autograd.grad(loss, s["y"])
    return {"loss": loss.detach(), "rewards": rewards, "dy": dy}


def _own_norm(s):
    from ksa_b200 import ops
    if s["to"] == "norm":
        return {"norm": ops.grad_norm(s["grads"])}
    return {"norm": ops.clip_grad_norm_(s["grads"], s["most"], out=s["out"] if s["to"] == "out" else None), "clipped": s["flat"]}


def run(state):
    kind = state["kind"]
    if own:
        return {"log_probs": _own_log_probs, "policy": _own_policy, "preference": _own_preference, "norm": _own_norm}[kind](state)
    return {"log_probs": _plain_log_probs, "policy": _plain_policy, "preference": _plain_preference, "norm": _plain_norm}[kind](state)


def work(case):
    kind = case["kind"]
    if kind == "log_probs":
        n, T, D, V = int(_answered(case).sum()), case["T"], case["D"], case["V"]
        nbytes, flops = 2 * n * D + 2 * V * D + 12 * T, 2 * n * V * D
        if case["train"]:
            nbytes, flops = nbytes + 2 * T * D + 2 * V * D + 4 * T, 3 * flops
        return {"bytes": nbytes, "flops": flops}
    if kind == "norm":
        size = {"float32": 4, "bfloat16": 2, "float16": 2, "mixed": 10 / 3}[case["dtype"]]
        return {"bytes": case["total"] * size * (2 if case["to"] == "out" else 1), "flops": 2 * case["total"]}
    n = int(_lengths(case).sum())
    arrays = (4 if kind == "policy" and case["adv"] == "token" else 3 if kind == "policy" else 2) + case["ref"]
    return {"bytes": n * (4 * arrays + 1), "flops": 30 * n if kind == "policy" else 4 * n}


# ------------------------------------------------------------------------------------------------- in 64 bits
def _exact_log_probs(s):
    rows = torch.nonzero(s["labels"] != IGNORE)[:, 0]
    h, w = s["h"].detach()[rows].double(), s["w"].detach().double()
    x = torch.mm(h, w.t()).div_(s["tau"])
    lse = torch.logsumexp(x, dim=1)
    T, at = s["labels"].shape[0], torch.arange(rows.numel(), device=h.device)
    y = torch.zeros(T, dtype=torch.float64, device=h.device)
    y[rows] = x[at, s["labels"][rows]] - lse
    if not s["train"]:
        return {"y": y}
    dx = torch.exp_(x.sub_(lse[:, None])).neg_()
    dx[at, s["labels"][rows]] += 1
    dx *= (s["dy"][rows].double() / s["tau"])[:, None]
    dh = torch.zeros(T, h.shape[1], dtype=torch.float64, device=h.device)
    dh[rows] = torch.mm(dx, w)
    return {"y": y, "dh": dh, "dw": torch.mm(dx.t(), h)}


def _bounds(s):
    return [0] + np.cumsum(np.bincount(s["of"].cpu().numpy(), minlength=s["S"])).tolist()


def _exact_policy(s):
    host = lambda t: None if t is None else t.detach().reshape(-1).cpu().numpy().astype(np.float64)  # noqa: E731
    y, old, ref, m, a = host(s["y"]), host(s["old"]), host(s["ref"]), host(s["mask"]) > 0, host(s["adv"])
    bounds = _bounds(s)
    per_sequence = s["adv"].shape != s["y"].shape
    dy, sums, counts = np.zeros(y.size), [], []
    for k, (lo, hi) in enumerate(zip(bounds[:-1], bounds[1:])):
        at = lo + np.flatnonzero(m[lo:hi])
        A = a[k] if per_sequence else a[at]
        d = y[at] - old[at]
        over = np.where(A >= 0, d > np.log(1.2), d < np.log(0.8)) & (A != 0)
        ratio = np.exp(np.where(over, np.where(d > 0, np.log(1.2), np.log(0.8)), d))
        K, dK = np.zeros(at.size), np.zeros(at.size)
        if ref is not None:
            x = ref[at] - y[at]
            K, dK = np.expm1(x) - x, -np.expm1(x)
        dy[at] = np.where(over, 0.0, -A * np.exp(d)) + s["kl"] * dK
        sums.append([(-A * ratio).sum(), K.sum(), over.sum()])
        counts.append(at.size)
    sums, counts = np.array(sums), np.array(counts)
    if s["by"] == "token":
        means, scale = sums.sum(0) / max(counts.sum(), 1), np.full(len(counts), 1.0 / max(counts.sum(), 1))
    else:
        scale = 1.0 / (np.maximum(counts, 1) * max((counts > 0).sum(), 1))
        means = (sums * scale[:, None]).sum(0)
    dy[:bounds[-1]] *= np.repeat(scale, np.diff(bounds))
    return {"loss": np.array(means[0] + s["kl"] * means[1]), "stats": means, "dy": dy.reshape(tuple(s["y"].shape))}


def _exact_preference(s):
    host = lambda t: None if t is None else t.detach().reshape(-1).cpu().numpy().astype(np.float64)  # noqa: E731
    y, ref, m = host(s["y"]), host(s["ref"]), host(s["mask"])
    bounds = _bounds(s)
    v = (y if ref is None else y - ref) * m
    rewards = s["beta"] * np.array([math.fsum(v[lo:hi]) for lo, hi in zip(bounds[:-1], bounds[1:])]).reshape(-1, 2)
    z = rewards[:, 0] - rewards[:, 1]
    loss = np.mean((1 - s["smooth"]) * np.logaddexp(0, -z) + s["smooth"] * np.logaddexp(0, z))
    dz = s["smooth"] * np.exp(-np.logaddexp(0, -z)) - (1 - s["smooth"]) * np.exp(-np.logaddexp(0, z))
    per = s["beta"] / len(z) * np.stack([dz, -dz], 1).reshape(-1)
    dy = m * np.concatenate([np.repeat(per, np.diff(bounds)), np.zeros(y.size - bounds[-1])])
    return {"loss": np.array(loss), "rewards": rewards, "dy": dy.reshape(tuple(s["y"].shape))}


def _exact_norm(s):
    norm = math.sqrt(math.fsum(float((x.double() ** 2).sum()) for x in s["grads"]))
    if s["to"] == "norm":
        return {"norm": np.array(norm)}
    by = min(1.0, s["most"] / (norm + 1e-6))
    if s["to"] == "place":
        return {"norm": np.array(norm), "clipped": {t: b.double() * by for t, b in s["flat"].items()}}
    clipped = {t: torch.zeros_like(b, dtype=torch.float64) for t, b in s["flat"].items()}
    for x in s["grads"]:
        clipped[str(x.dtype)][x.storage_offset():x.storage_offset() + x.numel()] = x.double() * by
    return {"norm": np.array(norm), "clipped": clipped}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"log_probs": _exact_log_probs, "policy": _exact_policy, "preference": _exact_preference, "norm": _exact_norm}[case["kind"]](s)
