"""``ops.linear_log_probs`` where its arithmetic is at its limits, against the definition in 64 bits, on logits that are exact.

Rows and weights are small whole numbers and multiples of 2^-7, so that every partial sum of a logit is exact in 32 bits and in the tensor cores: what is
left are the errors of the softmax.  Row ``t`` has a column of its own with a one in it, and no weight has anything there: the logits' gradient of
that row can then be read from the weights' gradient, where it is a single product, as ``dx`` rounded to bf16.

Tolerances.  The distance below the maximum is taken in base 2 with one factor, ``log2(e) / tau`` in 32 bits: off by 2^-24 of the distance with its product.  The
log-sum is one 32-bit number: half a step, 2^-24 of it.  Exponentials (2^-22), the correction of a tile's sum for its rounded maximum (2^-22) and the
sum's roundings: 2^-20.  Kept logits: half a step of 2^-10 of a power of two, 2^-11.5 of the probability; not so the label's, which comes
from the exact logit by way of a distance that is rounded by itself.  dx is rounded to bf16, 2^-8.
"""
from types import SimpleNamespace

import pytest
import torch

from ksa_b200 import ops
from ksa_b200.ops import log_probs as impl
from test_log_probs_gpu import IGNORE, _close, _inputs, _oracle, _run

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["kept", "again"], autouse=True)
def logits(request, monkeypatch):
    """Every test with the logits kept for the backward pass and with them computed again, whatever the width."""
    monkeypatch.setattr(impl, "KEEP_WIDTH", 0 if request.param == "kept" else 1 << 20)
    return request.param


def _exact(T, V, D, factor, steps, unit, label_on_top, seed=0):
    """h, w, labels, dy and each row's own column.  Row t has its two largest logits in the columns 2 g and 2 g + 1, the first ``steps`` to
    its number times ``unit`` above the second; all others are far below."""
    assert V % 2 == 0 and D >= T + 48
    g = torch.Generator().manual_seed(seed)
    place = torch.randperm(D, generator=g)
    main, fine, own = place[:40], place[40], place[48:48 + T]
    w = torch.zeros(V, D)
    trits = torch.randint(-1, 2, (V // 2, 40), generator=g).float()
    w[:, main] = trits.repeat_interleave(2, 0)
    w[1::2, fine] = -1
    group = torch.randint(0, V // 2, (T,), generator=g)
    h = torch.zeros(T, D)
    h[:, main] = trits[group] * (factor * torch.randint(8, 16, (T, 1), generator=g))
    h[:, fine] = torch.randint(*steps, (T,), generator=g) * unit
    h[torch.arange(T), own] = 1
    labels = 2 * group if label_on_top else torch.randint(0, V, (T,), generator=g)
    dy = torch.randn(T, generator=g)
    assert torch.equal(h.bfloat16().float(), h)
    return h.bfloat16().cuda(), w.bfloat16().cuda(), labels.cuda(), dy.cuda(), own.cuda()


def _check(h, w, labels, dy, own, tau, kept):
    t32 = float(torch.tensor(tau, dtype=torch.float32))
    T = h.shape[0]
    i = torch.arange(T, device="cuda")
    x = h.double() @ w.double().T / t32
    lse = x.logsumexp(1, keepdim=True)
    p = (x - lse).exp()
    g = dy.double()[:, None] / t32
    dx = -p * g
    # (of the label next to a probability of one: by the sum of the others)
    rest = p.clone()
    rest[i, labels] = 0
    dx[i, labels] = rest.sum(1) * g[:, 0]
    gap = x.amax(1, keepdim=True) - x
    far = 2.0 ** -24 * gap + 2.0 ** -20                                     # of what is taken as a distance below the maximum
    off = p * (far + 2.0 ** -24 * (lse.abs() + 1) + (2.0 ** -11.5 if kept else 0)) + (2.0 ** -63 if kept else 2.0 ** -126)
    off[i, labels] = (p * far)[i, labels] + 2.0 ** -126
    tol = off * g.abs() * (1 + 2.0 ** -8) + 2.0 ** -8 * dx.abs()
    h, w = h.requires_grad_(), w.requires_grad_()
    y = ops.linear_log_probs(h, w, labels, temperature=tau)
    dh, dw = torch.autograd.grad(y, (h, w), dy)
    want = x[i, labels] - lse[:, 0]
    assert ((y.detach().double() - want).abs() <= 2.0 ** -23 * (want.abs() + 1) + 2.0 ** -20).all()
    got = dw[:, own].T.double()
    bad = (got - dx).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((got - dx).abs() / tol).max()))
    # dh adds up to two or three terms of any size in 32 bits, and is rounded once
    wd = w.detach().double()
    assert ((dh.double() - dx @ wd).abs() <= (tol @ wd.abs()) * (1 + 2.0 ** -8) + (dx.abs() @ wd.abs()) * 2.0 ** -18 + 2.0 ** -8 * (dx @ wd).abs()).all()


@pytest.mark.parametrize("T,V", [(90, 600), (200, 1002), (300, 5000)])
@pytest.mark.parametrize("factor,steps,unit,tau", [(16, (0, 12), 0.25, 1.0), (256, (0, 12), 0.25, 1.0), (1, (0, 4), 2.0 ** -7, 0.01)])
def test_probabilities_at_logits_of_thousands(T, V, factor, steps, unit, tau, logits):
    """The two largest logits share the row's probability however far from zero they are: by the hundreds, by the hundred thousand, at a
    sampling temperature of a hundredth."""
    h, w, labels, dy, own = _exact(T, V, -(-(T + 48) // 8) * 8, factor, steps, unit, False, seed=T)
    _check(h, w, labels, dy, own, tau, logits == "kept")


@pytest.mark.parametrize("T,V,D", [(64, 500, 136), (64, 500, 2056), (300, 1002, 1096)])
def test_gradient_of_a_label_next_to_probability_one(T, V, D, logits):
    """1 - p from 2e-2 down to 3e-6, with logits of a few hundred."""
    h, w, labels, dy, own = _exact(T, V, D, 1, (16, 52), 0.25, True, seed=T + D)
    _check(h, w, labels, dy, own, 1.0, logits == "kept")


@pytest.mark.parametrize("T,D,V,answer", [(1, 64, 1000, 1), (1, 2048, 3003, 1), (2, 136, 5000, 2), (9, 1032, 700, 9), (64, 128, 4096, 64),
                                              (65, 256, 300, 65), (128, 64, 2000, 128), (300, 136, 1000, 64), (1500, 64, 500, 128), (9000, 16, 300, 3)])
@pytest.mark.parametrize("which", ["both", "rows", "head", "slabs"])
def test_gradients_of_few_rows_are_rounded_once(T, D, V, answer, which, logits, monkeypatch):
    """Up to 128 rows with a label, wherever they are: the logits' gradient takes part with 16 bits, so that what the results are off by is
    their own rounding to bf16, 2^-8, and what the probabilities are (see test_log_probs_gpu)."""
    h, w, labels, dy = _inputs(T, D, V, 1.0, seed=T + D)
    labels[torch.randperm(T, device="cuda")[:T - answer]] = IGNORE
    if which == "slabs":
        monkeypatch.setattr(impl, "SLAB_BYTES", 1)
    x = h.double() @ w.double().T
    lse = x.logsumexp(1, keepdim=True)
    p = (x - lse).exp()
    live = labels != IGNORE
    one = torch.zeros_like(p)
    one[live, labels[live]] = 1
    g = torch.where(live, dy, torch.zeros_like(dy)).double()[:, None]
    dx = (one - p) * g
    ex = (D / 16 + 2) * 2.0 ** -22 * (h.double().abs() @ w.double().abs().T).amax(1, keepdim=True)
    kept = 2.0 ** -11.5 if logits == "kept" and which != "slabs" else 0.0
    off = p * (2 * ex + 2.0 ** -18 + kept) * g.abs() + 2.0 ** -16 * dx.abs() + 2.0 ** -120
    need = {"both": (True, True), "slabs": (True, True), "rows": (True, False), "head": (False, True)}[which]
    h.requires_grad_(need[0])
    w.requires_grad_(need[1])
    y = ops.linear_log_probs(h, w, labels)
    grads = iter(torch.autograd.grad(y, [t for t, n in zip((h, w), need) if n], dy))
    hd, wd = h.detach().double(), w.detach().double()
    for wanted, value, spread, sums in ((need[0], dx @ wd, off @ wd.abs(), (V / 16 + 80) * 2.0 ** -22 * (dx.abs() @ wd.abs())),
                                        (need[1], dx.T @ hd, off.T @ hd.abs(), (2 * T / 16 + 8) * 2.0 ** -22 * (dx.abs().T @ hd.abs()))):
        if wanted:
            got = next(grads).double()
            tol = 2.0 ** -8 * value.abs() + (spread + sums) * 1.01 + 1e-30
            bad = (got - value).abs() > tol
            assert not bad.any(), (int(bad.sum()), float(((got - value).abs() / tol).max()))


@pytest.mark.parametrize("T,D,V", [(1, 152, 99667), (70, 64, 4096), (300, 136, 1000), (333, 256, 4096), (600, 512, 20000), (1300, 1024, 30000), (4100, 128, 2000)])
@pytest.mark.parametrize("answer", [1.0, 0.4, 0.0])
@pytest.mark.parametrize("head", [True, False])
def test_parts_of_the_rows_gradient_are_those_that_were_written(T, D, V, answer, head, monkeypatch):
    """The products say how many parts they made, and so many are added up; the memory of the others holds anything."""
    h, w, labels, dy = _inputs(T, D, V, answer, seed=T)
    seen = []
    call = impl._lib.call

    def watched(name, *args):
        if name != "ksa_log_probs_bwd":
            return call(name, *args)
        parts, dh, planes, rows = args[11], args[12], args[22], args[0].shape[0]
        parts.fill_(float("nan"))
        call(name, *args)
        made = int(parts.view(torch.int32)[planes * rows * D])
        seen.append((made, planes))
        planes_of = parts[:planes * rows * D].view(planes, rows, D)
        count = int(args[5][0])
        assert (made == 0) if count == 0 else 1 <= made <= planes
        assert planes_of[made:].isnan().all() and planes_of[:made, :count].isfinite().all()
        total = torch.zeros(T, D, device="cuda", dtype=torch.float64)
        at = args[2][:count].long()
        used = planes_of[:made, :count]
        if count <= 128:                                                    # few rows: the products of both halves of the logits' gradient
            used = torch.cat([used, planes_of[:made, 128:128 + count]])
        total[at] = used.double().sum(0)
        # added up in 32 bits, in order or by eight at a time: 128 roundings of partial sums at most
        bound = torch.zeros_like(total)
        bound[at] = used.double().abs().sum(0)
        assert ((dh.double() - total).abs() <= 2.0 ** -8 * total.abs() + 2.0 ** -17 * bound + 2.0 ** -130).all()
    monkeypatch.setattr(impl._lib, "call", watched)
    monkeypatch.setattr(impl, "_native", SimpleNamespace(linear_log_probs=lambda *args: None))
    h.requires_grad_()
    w.requires_grad_(head)
    torch.autograd.grad(ops.linear_log_probs(h, w, labels), (h, w) if head else h, dy)
    assert len(seen) == 1


@pytest.mark.parametrize("T,D,V", [(1, 1032, 300), (33, 2048, 1003), (128, 2560, 300), (129, 1160, 1003), (300, 2048, 2600), (520, 2568, 700)])
@pytest.mark.parametrize("answer,tau", [(1.0, 1.0), (0.5, 0.7)])
def test_wide_rows(T, D, V, answer, tau):
    """Widths above 1024, where a logit is added up from several parts: the last one whole and ragged, tiles in halves, few rows and many."""
    h, w, labels, dy = _inputs(T, D, V, answer, seed=T, tau=tau)
    want = _oracle(h, w, labels, dy, tau)
    got = _run(h, w, labels, dy, tau)
    for name, g in zip(("y", "dh", "dw"), got):
        _close(g, want[name], name)
    with torch.no_grad():
        _close(ops.linear_log_probs(h, w, labels, temperature=tau), want["y"], "y alone")
    assert all(torch.equal(a, b) for a, b in zip(_run(h, w, labels, dy, tau), got))


@pytest.mark.parametrize("T", [8192, 8193, 8200, 16390, 20000])
def test_more_rows_than_one_round_of_the_selection(T):
    """Rows are chosen 8192 at a time; the places of a round begin where the one before it ended."""
    h, w, labels, dy = _inputs(T, 16, 40, 0.6, seed=T)
    labels[8190:8195] = torch.tensor([3, -100, 5, 39, -100], device="cuda")[:max(0, T - 8190)][:5]
    want = _oracle(h, w, labels, dy, 1.0)
    for name, g in zip(("y", "dh", "dw"), _run(h, w, labels, dy, 1.0)):
        _close(g, want[name], name)
    only = torch.full_like(labels, IGNORE)
    only[-1] = 7                                                            # a single label, in the last round
    want = _oracle(h, w, only, dy, 1.0)
    for name, g in zip(("y", "dh", "dw"), _run(h, w, only, dy, 1.0)):
        _close(g, want[name], name)


@pytest.mark.parametrize("T,D,V", [(1, 64, 1000), (128, 136, 1003), (129, 136, 1003), (300, 264, 1000), (1030, 64, 5000)])
@pytest.mark.parametrize("slab,planes", [(4 << 30, 512 << 20), (2 * 512 * 512, 512 << 20), (2 * 512 * 1024, 0), (1, 1 << 20)])
def test_both_ways_to_the_kernels_decide_alike(T, D, V, slab, planes, monkeypatch):
    """Calls by way of Python (which a head with a gradient buffer takes) and of native code give the same bits, wherever the
    rules for kept logits, slabs and parts put them."""
    monkeypatch.setattr(impl, "SLAB_BYTES", slab)
    monkeypatch.setattr(impl, "PLANE_BYTES", planes)
    h, w, labels, dy = _inputs(T, D, V, 0.7, seed=T)
    native = _run(h, w, labels, dy, 0.7)
    with torch.no_grad():
        alone = ops.linear_log_probs(h, w, labels, temperature=0.7)
    monkeypatch.setattr(impl, "_native", SimpleNamespace(linear_log_probs=lambda *args: None))
    assert all(torch.equal(a, b) for a, b in zip(_run(h, w, labels, dy, 0.7), native))
    with torch.no_grad():
        assert torch.equal(ops.linear_log_probs(h, w, labels, temperature=0.7), alone)
