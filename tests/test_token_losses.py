"""The policy and preference losses against their formulas in 64 bits, written out token by token, on the CPU and (marked) on the GPU.

Tolerances: a token's terms are a product of an exponential and the advantage, each rounded a few times in 32 bits: ``(|d| + 8) 2^-24`` of
the term's magnitude (the difference's rounding counts ``|d|`` times in its exponential), and a gradient that is returned in another type is rounded to
it, half a step.  Means are off by the mean of their terms' errors and one rounding.
"""
import math

import pytest
import torch

from ksa_b200 import ops
from ksa_b200.losses import PolicyLoss, PreferenceLoss

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
E = 2.0 ** -24


def _tokens(lengths, packed, behind=0, seed=0, dtypes=(torch.float32,) * 4, odd=0, adv="token"):
    """y, old, ref, advantages, mask, cu, each packed sequence's slice; ``odd``: values in front of every array, off its alignment."""
    g = torch.Generator().manual_seed(seed)
    n = sum(lengths) + behind
    mk = lambda v, t: torch.cat([torch.full((odd,), float("nan")), v]).to(t)[odd:]  # noqa: E731
    y = -torch.rand(n, generator=g).pow(3) * 9
    old = y + 0.3 * torch.randn(n, generator=g)
    ref = y + 0.5 * torch.randn(n, generator=g)
    a = torch.randn(n if adv == "token" else len(lengths), generator=g)
    mask = torch.rand(n + odd, generator=g)[odd:] < 0.8
    out = [mk(v, t) for v, t in zip((y, old, ref, a), dtypes)]
    cu = torch.tensor([0] + torch.tensor(lengths, dtype=torch.long).cumsum(0).tolist(), dtype=torch.int32)
    if not packed:
        shape = (len(lengths), lengths[0] if lengths else 0)
        out = [v.view(shape) if v.numel() == n and adv == "token" or i < 3 else v for i, v in enumerate(out)]
        mask, cu = mask.view(shape), None
    return (*out, mask, cu)


def _slices(y, cu):
    if cu is not None:
        return [(int(a), int(b)) for a, b in zip(cu[:-1], cu[1:])]
    if y.dim() == 1:
        return [(0, y.numel())]
    return [(s * y.shape[1], (s + 1) * y.shape[1]) for s in range(y.shape[0])]


def _policy(y, old, ref, adv, mask, cu, low, high, beta, by_sequence):
    """(loss, stats, gradient) and their tolerances, by loops in 64 bits."""
    flat = lambda t: t.detach().cpu().double().reshape(-1)  # noqa: E731
    yf, of = flat(y), flat(old)
    per_token = adv.shape == y.shape
    spans, n = _slices(y, cu), y.numel()
    dy, tol = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
    rows = []
    for s, (lo, hi) in enumerate(spans):
        at = torch.arange(lo, hi)
        if mask is not None:
            at = at[mask.cpu().reshape(-1)[lo:hi] != 0]
        A = flat(adv)[at] if per_token else flat(adv)[s].expand(at.numel())
        d = yf[at] - of[at]
        r = d.exp()
        cut = ((A > 0) & (d > math.log1p(high))) | ((A < 0) & (d < (math.log1p(-low) if low < 1 else -math.inf)))
        L = -torch.minimum(r * A, r.clamp(1 - low, 1 + high) * A)
        x = flat(ref)[at] - yf[at] if ref is not None else torch.zeros_like(d)
        K = torch.expm1(x) - x
        g = torch.where(cut, torch.zeros_like(r), -r * A) - beta * torch.expm1(x)
        e = (r * A).abs() * (d.abs() + 8) * E
        eK = (K + x.abs() * 0.0) * (x.abs() + 16) * E
        dy[at] = g
        tol[at] = torch.where(cut, torch.zeros_like(e), e) + beta * torch.expm1(x).abs() * (x.abs() + 8) * E + g.abs() * 8 * E
        rows.append((at, torch.stack([L.sum(), K.sum(), cut.double().sum()]), torch.stack([e.sum() + (L.abs() * 4 * E).sum(), eK.sum(), e.sum() * 0])))
    counts = torch.tensor([r[0].numel() for r in rows], dtype=torch.float64)
    live = (counts > 0).double().sum().clamp(min=1)
    stats, off = torch.zeros(3, dtype=torch.float64), torch.zeros(3, dtype=torch.float64)
    for (at, total, err), c in zip(rows, counts):
        w = (1 / (c.clamp(min=1) * live)) if by_sequence else 1 / counts.sum().clamp(min=1)
        dy[at] *= w
        tol[at] *= w
        stats, off = stats + total * w, off + err * w
    loss = stats[0] + (beta * stats[1] if beta else 0)
    loss_off = off[0] + beta * off[1] + loss.abs() * 4 * E + 1e-12
    return loss, loss_off, stats, off + stats.abs() * 4 * E + 1e-12, dy.view(y.shape), tol.view(y.shape) + 1e-30


def _half_step(t):
    return {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[t]


def _name(lengths):
    return f"{len(lengths)} of {sum(lengths)}"


LENGTHS = [[1], [7], [2048], [2049], [4096], [3, 5], [257] * 4, [0, 0, 3], [5, 0, 0, 4100, 1, 2047, 2048, 0], [1] * 300, [6000, 1, 9000],
           [4095, 4097, 8193], [33001, 2], [2] * 1100, []]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lengths", LENGTHS, ids=_name)
@pytest.mark.parametrize("by_sequence", [False, True])
def test_policy_loss(device, lengths, by_sequence):
    for packed in (True, False):
        if not packed and (not lengths or len(set(lengths)) > 1):
            continue
        for beta, adv, behind, wide in ((0.0, "token", 0, False), (0.05, "sequence", 3 if packed else 0, True)):
            y, old, ref, a, mask, cu = _tokens(lengths, packed, behind, seed=len(lengths), adv=adv)
            if cu is not None and wide:
                cu = cu.long()
            use_ref = ref if beta else None
            want = _policy(y, old, use_ref, a, mask, cu, 0.2, 0.28, beta, by_sequence)
            y, old, use_ref, a, mask, cu = (None if t is None else t.to(device) for t in (y, old, use_ref, a, mask, cu))
            y.requires_grad_(True)
            loss, stats = ops.policy_loss(y, old, a, use_ref, mask, cu, clip_low=0.2, clip_high=0.28, kl_coef=beta,
                                          reduction="sequence" if by_sequence else "token")
            assert loss.dtype == stats.dtype == torch.float32 and not stats.requires_grad
            assert abs(float(loss.detach()) - float(want[0])) <= want[1]
            assert ((stats.cpu().double() - want[2]).abs() <= want[3]).all()
            dy, = torch.autograd.grad(loss, y, torch.tensor(2.0, device=device))
            assert dy.shape == y.shape and ((dy.cpu().double() / 2 - want[4]).abs() <= want[5]).all()
            module = PolicyLoss(0.2, 0.28, beta, "sequence" if by_sequence else "token")
            assert torch.equal(module(y, old, a, use_ref, mask, cu)[0], loss)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("odd", [0, 1, 2])
@pytest.mark.parametrize("dtypes", [(torch.bfloat16,) * 4, (torch.float16, torch.float32, torch.bfloat16, torch.float32),
                                    (torch.float32, torch.bfloat16, torch.float32, torch.float16)], ids=["bf16", "fp16 first", "mixed"])
def test_policy_loss_of_other_types_and_alignments(device, odd, dtypes):
    y, old, ref, a, mask, cu = _tokens([100, 2051, 3], True, 2, seed=odd, dtypes=dtypes)
    want = _policy(y, old, ref, a, mask, cu, 0.2, 0.2, 0.1, False)
    # on the device the arrays begin off their alignment too
    move = lambda t: torch.cat([t[:odd], t]).to(device)[odd:]  # noqa: E731
    y, old, ref, a, mask = (move(t) for t in (y, old, ref, a, mask))
    y = y.detach().requires_grad_(True)
    loss, _ = ops.policy_loss(y, old, a, ref, mask, cu.to(device), kl_coef=0.1)
    dy, = torch.autograd.grad(loss, y)
    assert abs(float(loss.detach()) - float(want[0])) <= want[1]
    assert dy.dtype == dtypes[0]
    # (a gradient below the smallest normal number of fp16 is off by half its spacing, 2^-25)
    assert ((dy.cpu().double() - want[4]).abs() <= want[5] + _half_step(dtypes[0]) * want[4].abs() * 1.01 + (2.0 ** -25 if dtypes[0] == torch.float16 else 0)).all()


@pytest.mark.parametrize("device", DEVICES)
def test_masked_tokens_may_hold_anything(device):
    y, old, ref, a, mask, cu = (t.to(device) for t in _tokens([50, 2060, 7], True, 9, seed=5))
    y.requires_grad_(True)
    kw = dict(clip_low=0.2, clip_high=0.2, kl_coef=0.1, reduction="sequence")
    for bad in (float("nan"), float("inf"), -float("inf"), torch.finfo(torch.float32).min):
        spoil = lambda t: torch.where(mask, t, torch.full_like(t, bad)) if t.shape == mask.shape else t  # noqa: E731
        y2, old2, ref2, a2 = (spoil(t.detach()) for t in (y, old, ref, a))
        for t in (y2, old2, ref2, a2):
            t[int(cu[-1]):] = bad                             # behind the last sequence
        y2.requires_grad_(True)
        one, two = ops.policy_loss(y, old, a, ref, mask, cu, **kw), ops.policy_loss(y2, old2, a2, ref2, mask, cu, **kw)
        assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
        assert torch.equal(torch.autograd.grad(one[0], y)[0], torch.autograd.grad(two[0], y2)[0])
    pairs = torch.cat([cu[:3], cu[2:3] + 4, cu[3:]])
    one, two = ops.preference_loss(y, ref, mask, pairs), ops.preference_loss(y2, ref2, mask, pairs)
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
    assert torch.equal(torch.autograd.grad(one[0], y)[0], torch.autograd.grad(two[0], y2)[0])


@pytest.mark.parametrize("device", DEVICES)
def test_nothing_valid_is_no_loss(device):
    y, old, ref, a, mask, cu = (t.to(device) for t in _tokens([50, 60], True, seed=6))
    y.requires_grad_(True)
    for reduction in ("token", "sequence"):
        loss, stats = ops.policy_loss(y, old, a, ref, torch.zeros_like(mask), cu, kl_coef=0.1, reduction=reduction)
        assert float(loss.detach()) == 0 and not stats.any() and not torch.autograd.grad(loss, y)[0].any()
    loss, rewards = ops.preference_loss(y, ref, torch.zeros_like(mask), cu)
    assert abs(float(loss.detach()) - math.log(2)) < 1e-7 and not rewards.any() and not torch.autograd.grad(loss, y)[0].any()


@pytest.mark.parametrize("device", DEVICES)
def test_border_of_the_clipped_range(device):
    """Ratios next to 1 + high and 1 - low: cut off strictly outside.  log(1.25) falls between two fp32 numbers."""
    edge = torch.tensor(math.log(1.25), dtype=torch.float64)
    near = edge.float()
    steps = torch.stack([torch.nextafter(near, torch.tensor(v)) for v in (-1.0, 1.0)] + [near])
    d = torch.cat([steps, -steps])
    y = d.to(device).requires_grad_(True)
    for A in (1.0, -1.0):
        loss, stats = ops.policy_loss(y, torch.zeros_like(y), torch.full((6,), A, device=device), clip_low=0.2, clip_high=0.25)
        cut = (d.double() > edge) if A > 0 else (d.double() < math.log1p(-0.2))
        dy, = torch.autograd.grad(loss, y)
        assert torch.equal(dy.cpu() == 0, cut) and abs(float(stats[2]) - cut.double().mean()) < 1e-7


@pytest.mark.parametrize("device", DEVICES)
def test_extreme_differences(device):
    """Ratios that overflow, vanish, or have no number; a KL term next to zero keeps its digits."""
    y = torch.tensor([0.0, -200.0, -1.0, -1.0, -math.inf], device=device, requires_grad=True)
    old = torch.tensor([-200.0, 0.0, -1.0, -1.0, -1.0], device=device)
    a = torch.tensor([1.0, 1.0, 0.0, -1.0, 1.0], device=device)
    loss, stats = ops.policy_loss(y, old, a)
    dy, = torch.autograd.grad(loss, y)
    assert abs(float(loss.detach()) - (-1.2 + 0 + 0 + 1 + 0) / 5) < 1e-6 and float(stats[2]) == pytest.approx(0.2)
    assert torch.equal(dy.cpu(), torch.tensor([0.0, 0.0, 0.0, 0.2, 0.0]))
    x = torch.tensor([1e-3, -1e-4, 3e-6, 0.99, -1.01, 5.0, -30.0, 0.0], dtype=torch.float32)
    y = torch.zeros(8, device=device, requires_grad=True)
    for i in range(8):
        keep = torch.zeros(8, dtype=torch.bool, device=device)
        keep[i] = True
        loss, stats = ops.policy_loss(y, torch.zeros_like(y), torch.zeros_like(y), x.to(device), keep, kl_coef=1.0)
        v = x[i].double()
        # the series in 32 bits is off by some roundings of itself; beyond one the difference by those of its largest term
        K = torch.expm1(v) - v if v.abs() > 1e-2 else v * v * (0.5 + v / 6 + v * v / 24)
        assert abs(float(loss.detach()) - K) <= 16 * E * K + (4 * E * (v.exp() + v.abs() + 1) if v.abs() >= 1 else 0)
        g = torch.autograd.grad(loss, y)[0][i]
        assert abs(float(g) + torch.expm1(v)) <= 4 * E * torch.expm1(v).abs()


@pytest.mark.parametrize("device", DEVICES)
def test_policy_gradient_against_differences(device):
    y, old, ref, a, mask, cu = _tokens([40, 33], True, seed=7)
    dev = [t.to(device) for t in (y, old, ref, a, mask, cu)]
    dev[0].requires_grad_(True)
    loss, _ = ops.policy_loss(dev[0], dev[1], dev[3], dev[2], dev[4], dev[5], kl_coef=0.1, reduction="sequence")
    dy = torch.autograd.grad(loss, dev[0])[0].cpu().double()
    h = 1e-6
    for i in range(0, 73, 7):
        step = torch.zeros(73, dtype=torch.float64)
        step[i] = h
        f = [_policy(y.double() + s * step, old, ref, a, mask, cu, 0.2, 0.2, 0.1, True)[0] for s in (1, -1)]
        assert abs((f[0] - f[1]) / (2 * h) - dy[i]) < 1e-7          # (no token is within 1e-6 of the border)


def _preference(y, ref, mask, cu, beta, eps):
    flat = lambda t: t.detach().cpu().double().reshape(-1)  # noqa: E731
    v = flat(y) - (flat(ref) if ref is not None else 0)
    m = torch.ones(v.numel(), dtype=torch.bool) if mask is None else mask.cpu().reshape(-1) != 0
    spans = _slices(y, cu)
    D = torch.stack([v[lo:hi][m[lo:hi]].sum() for lo, hi in spans]) if spans else torch.zeros(0, dtype=torch.float64)
    r = beta * D.view(-1, 2)
    z = r[:, 0] - r[:, 1]
    loss = ((1 - eps) * torch.nn.functional.softplus(-z) + eps * torch.nn.functional.softplus(z)).sum() / max(len(z), 1)
    per = beta * (eps * torch.sigmoid(z) - (1 - eps) * torch.sigmoid(-z)) / max(len(z), 1)
    dy = torch.zeros(v.numel(), dtype=torch.float64)
    for s, (lo, hi) in enumerate(spans):
        dy[lo:hi] = torch.where(m[lo:hi], per[s // 2] * (1 if s % 2 == 0 else -1), dy[lo:hi])
    return loss, r, dy.view(y.shape)


PAIRS = [[1, 1], [2048, 2049], [0, 5], [0, 0], [257] * 4, [1] * 300, [4097, 3, 0, 6000, 2048, 1], [33001, 4096], [2] * 1026, [1] * 2500, []]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lengths", PAIRS, ids=_name)
@pytest.mark.parametrize("use_ref,use_mask,eps", [(True, True, 0.0), (False, False, 0.1), (True, False, 1.0)])
def test_preference_loss(device, lengths, use_ref, use_mask, eps):
    for packed in (True, False):
        if not packed and (not lengths or len(set(lengths)) > 1):
            continue
        y, _, ref, _, mask, cu = _tokens(lengths, packed, 5 if packed else 0, seed=len(lengths) + 1)
        ref, mask = ref if use_ref else None, mask if use_mask else None
        # all is in 64 bits but beta and the smoothing, fp32 numbers (2^-24 each), and the rounding of the results
        beta = 0.03
        loss_w, r_w, dy_w = _preference(y, ref, mask, cu, beta, eps)
        y, ref, mask, cu = (None if t is None else t.to(device) for t in (y, ref, mask, cu))
        y.requires_grad_(True)
        loss, rewards = ops.preference_loss(y, ref, mask, cu, beta=beta, label_smoothing=eps)
        z = (r_w[:, 0] - r_w[:, 1]).abs().amax() if len(r_w) else torch.zeros(())
        assert abs(float(loss.detach()) - loss_w) <= (loss_w + z) * 4 * E
        assert rewards.shape == r_w.shape and ((rewards.cpu().double() - r_w).abs() <= r_w.abs() * 4 * E + 1e-30).all()
        dy, = torch.autograd.grad(loss, y)
        # (d(loss) / dz is a difference of the smoothing and a logistic value: off by z roundings of the latter, and of the smoothing)
        assert ((dy.cpu().double() - dy_w).abs() <= dy_w.abs() * 4 * E + beta / max(len(r_w), 1) * (z + 4) * E * (dy_w != 0)).all()
        assert torch.equal(PreferenceLoss(beta, eps)(y, ref, mask, cu)[0], loss)


@pytest.mark.parametrize("device", DEVICES)
def test_preference_of_far_apart_answers(device):
    for gap in (1e4, -1e4, math.inf, -math.inf):
        y = torch.tensor([0.0, -gap], device=device, requires_grad=True)
        cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=device)
        loss, rewards = ops.preference_loss(y, None, None, cu, beta=1.0)
        dy, = torch.autograd.grad(loss, y)
        assert float(loss.detach()) == (0 if gap > 0 else -gap) and torch.equal(dy.cpu(), torch.tensor([0.0, 0.0] if gap > 0 else [-1.0, 1.0]))


@pytest.mark.parametrize("device", DEVICES)
def test_other_layouts(device):
    y, old, ref, a, mask, _ = (None if t is None else t.to(device) for t in _tokens([12] * 6, False, seed=8))
    want = ops.policy_loss(y, old, a, ref, mask, kl_coef=0.1)
    spread = lambda t: torch.stack([t, t], -1)[..., 0]  # noqa: E731
    for f in (spread, lambda t: t.t().contiguous().t()):
        args = [f(t) for t in (y, old, a, ref, mask)]
        leaf = args[0].detach().requires_grad_(True)
        got = ops.policy_loss(leaf, *args[1:], kl_coef=0.1)
        assert torch.equal(got[0], want[0]) and torch.autograd.grad(got[0], leaf)[0].shape == y.shape
    rows = torch.randn(6, device=device)
    one = ops.policy_loss(y, old, rows, ref, mask)[0]
    assert torch.equal(one, ops.policy_loss(y, old, rows[:, None], ref, mask.to(torch.uint8))[0])
    assert torch.equal(one, ops.policy_loss(y, old, rows[:, None].expand(6, 12).contiguous(), ref, mask)[0])


@pytest.mark.parametrize("device", DEVICES)
def test_offsets_behind_the_last_token_count_as_it(device):
    y, old, ref, a, mask, cu = (t.to(device) for t in _tokens([50, 2060, 7, 0], True, seed=12))
    y.requires_grad_(True)
    far = cu.clone().long()
    far[3:] = 1 << 40
    for f in (lambda c: ops.policy_loss(y, old, a, ref, mask, c, kl_coef=0.1, reduction="sequence"), lambda c: ops.preference_loss(y, ref, mask, c)):
        one, two = f(cu), f(far)
        assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
        assert torch.equal(torch.autograd.grad(one[0], y)[0], torch.autograd.grad(two[0], y)[0])


@pytest.mark.parametrize("device", DEVICES)
def test_no_sequences(device):
    """Tokens that belong to none, and no rows: no loss, and gradients of zero."""
    y = torch.randn(10, device=device, requires_grad=True)
    cu = torch.zeros(1, dtype=torch.int32, device=device)
    empty = torch.randn(0, 5, device=device, requires_grad=True)
    for reduction in ("token", "sequence"):
        for t, c, adv in ((y, cu, torch.randn(10, device=device)), (empty, None, torch.randn(0, 5, device=device))):
            loss, stats = ops.policy_loss(t, t.detach(), adv, cu_seqlens=c, reduction=reduction)
            assert float(loss.detach()) == 0 and not stats.any() and not torch.autograd.grad(loss, t)[0].any()
    for t, c in ((y, cu), (empty, None)):
        loss, rewards = ops.preference_loss(t, None, None, c)
        assert float(loss.detach()) == 0 and rewards.shape == (0, 2) and not torch.autograd.grad(loss, t)[0].any()


@pytest.mark.gpu
def test_replayed_twice_at_once_and_on_another_stream():
    y, old, ref, a, mask, cu = (t.cuda() for t in _tokens([700, 0, 5000, 33], True, 4, seed=9))

    def step():
        leaf = y.detach().requires_grad_(True)
        p, _ = ops.policy_loss(leaf, old, a, ref, mask, cu, kl_coef=0.1, reduction="sequence")
        d, rewards = ops.preference_loss(leaf, ref, mask, cu)
        return p.detach(), d.detach(), rewards, torch.autograd.grad(p + d, leaf)[0]
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    side.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(other, want))
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    for shift in (0.25, 0.0):
        y.add_(shift) if shift else y.sub_(0.25)
        expect = step()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for s, graph in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(u, v) for u, v in zip(out, expect))


@pytest.mark.gpu
def test_many_tokens_agree_with_the_cpu():
    """Rows of several units each and a long packed sequence."""
    for lengths, packed in (([20000] * 5, False), ([1, 70000, 12345, 0, 2048], True)):
        y, old, ref, a, mask, cu = _tokens(lengths, packed, seed=10)
        want = _policy(y, old, ref, a, mask, cu, 0.2, 0.2, 0.1, True)
        y, old, ref, a, mask, cu = (None if t is None else t.cuda() for t in (y, old, ref, a, mask, cu))
        y.requires_grad_(True)
        loss, stats = ops.policy_loss(y, old, a, ref, mask, cu, kl_coef=0.1, reduction="sequence")
        dy, = torch.autograd.grad(loss, y)
        assert abs(float(loss.detach()) - float(want[0])) <= want[1] and ((dy.cpu().double() - want[4]).abs() <= want[5]).all()


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    y, old, ref, a, mask, cu = (t.to(device) for t in _tokens([5, 6], True, seed=11))
    bad = [dict(reduction="mean"), dict(clip_low=-0.1), dict(clip_low=1.1), dict(clip_high=-1.0), dict(kl_coef=float("nan")),
           dict(mask=mask[:-1]), dict(mask=mask.float()), dict(ref_log_probs=ref[:3]), dict(cu_seqlens=cu.float()), dict(cu_seqlens=cu[None]),
           dict(cu_seqlens=cu[:0])]
    for kw in bad:
        with pytest.raises(ValueError):
            ops.policy_loss(y, old, a, **kw)
    for args in ((y, old[:3], a), (y, old, a[:3]), (y.view(1, 1, -1), old.view(1, 1, -1), a.view(1, 1, -1))):
        with pytest.raises(ValueError):
            ops.policy_loss(*args)
    for t in (old, a, ref):
        with pytest.raises(ValueError):
            ops.policy_loss(y, *(u.detach().requires_grad_(u is t) for u in (old, a, ref)))
    with pytest.raises(TypeError):
        ops.policy_loss(y.double(), old, a)
    with pytest.raises(TypeError):
        ops.policy_loss(y, old, a.long())
    for args, kw in (((y,), {}), ((y, ref, mask, cu[:2]), {}), ((y, ref, mask, cu), dict(beta=float("inf"))), ((y, ref, mask, cu), dict(label_smoothing=1.5))):
        with pytest.raises(ValueError):
            ops.preference_loss(*args, **kw)
    if device == "cuda":
        with pytest.raises(ValueError):
            ops.policy_loss(y, old.cpu(), a)
        with pytest.raises(ValueError):
            ops.preference_loss(y, ref, mask.cpu(), cu)


@pytest.mark.gpu
def test_transforms_meet_an_error_and_not_the_kernels():
    """Whoever follows the calls themselves gets the autograd functions' own refusal, not numbers from a wrapper's memory."""
    y, old, ref, a, mask, cu = (t.cuda() for t in _tokens([50, 60], True, seed=13))
    h, w = torch.randn(110, 64, device="cuda").bfloat16(), torch.randn(30, 64, device="cuda").bfloat16()
    labels = torch.randint(0, 30, (110,), device="cuda")
    calls = [lambda t: ops.policy_loss(t, old, a, ref, mask, cu)[0], lambda t: ops.preference_loss(t, ref, mask, cu)[0],
             lambda t: ops.linear_log_probs(h * t[:, None].bfloat16(), w, labels).sum()]
    for f in calls:
        for transformed in (torch.func.grad(f), lambda t: torch.func.vmap(f)(torch.stack([t, t])), lambda t: torch.func.jvp(f, (t,), (t,))):
            with pytest.raises(RuntimeError):
                transformed(y)
        with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError):
            f(torch.autograd.forward_ad.make_dual(y, torch.ones_like(y)))
        assert torch.isfinite(f(y))                            # and the next ordinary call is one
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: ops.grad_norm([t]))(torch.randn(3, 50, device="cuda"))
