"""Log probabilities of given tokens under the output head (``ops.linear_log_probs``) against their definition in 64 bits.

Tolerances, by arithmetic.  A logit is a sum of ``D`` products in the tensor cores' 32-bit accumulators: 16 products at a time, each
step off by at most 2^-22 of the sum of magnitudes ``S`` (a bit less than fp32 for what is aligned and cut off), so ``ex = (D / 16 + 2)
2^-22 S / tau``.  ``y`` is the difference of a logit and a log-sum that is off by no more than the logits are, both rounded a few times in base 2:
``2 ex + 8 2^-22 (1 + |x| + |lse|)``.  Probabilities are off by ``2 ex + 2^-18`` of themselves by the exponential's argument and function, and
by ln 2 times half a step of 2^-10, 2^-11.5, where they come from kept logits; the logits' gradient is rounded to bf16 (2^-8); the products with it add ``(n / 16 + 2) 2^-22`` of the sum of magnitudes, and the results are rounded to bf16 unless
they go into an fp32 buffer.
"""
import math

import pytest
import torch

from ksa_b200 import ops
from ksa_b200.ops import log_probs as impl

pytestmark = pytest.mark.gpu
IGNORE = -100


@pytest.fixture(params=["kept", "again"], autouse=True)
def _logits(request, monkeypatch):
    """Every test with the logits kept for the backward pass and with them computed again, whatever the width."""
    monkeypatch.setattr(impl, "KEEP_WIDTH", 0 if request.param == "kept" else 1 << 20)


def _inputs(T, D, V, answer, seed=0, tau=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = (torch.randn(V, D, generator=g, device="cuda") * 0.05).bfloat16()
    labels = torch.randint(0, V, (T,), generator=g, device="cuda")
    h = (torch.randn(T, D, generator=g, device="cuda") * (40 / math.sqrt(D)) + 6 / (D * 2.5e-3) * tau * w[labels].float()).bfloat16()
    keep = torch.rand(T, generator=g, device="cuda") < answer
    return h, w, torch.where(keep, labels, torch.full_like(labels, IGNORE)), torch.randn(T, generator=g, device="cuda")


def _oracle(h, w, labels, dy, tau):
    """y, dh, dw and their tolerances, all in 64 bits."""
    h, w, dy = h.detach().double(), w.detach().double(), dy.double()
    (T, D), V = h.shape, w.shape[0]
    rows = torch.nonzero((labels >= 0) & (labels < V))[:, 0]
    h, at, dy = h[rows], labels[rows], dy[rows]
    x = h @ w.T / tau
    ex = (D / 16 + 2) * 2.0 ** -22 * (h.abs() @ w.abs().T / tau).amax(1)
    lse = x.logsumexp(1)
    i = torch.arange(rows.numel(), device=h.device)
    yr = x[i, at] - lse
    p = (x - lse[:, None]).exp()
    dx = -p
    dx[i, at] += 1
    dx *= dy[:, None] / tau
    off = (p * (2 * ex + 2.0 ** -18 + 2.0 ** -11.5)[:, None] * dy.abs()[:, None] / tau) * (1 + 2.0 ** -8) + 2.0 ** -8 * dx.abs() + 2.0 ** -130
    out = {}
    full = lambda v: torch.zeros(T, *v.shape[1:], dtype=torch.float64, device=h.device).index_copy_(0, rows, v)  # noqa: E731
    out["y"] = full(yr), full(2 * ex + 8 * 2.0 ** -22 * (1 + x[i, at].abs() + lse.abs()))
    dh, dw = dx @ w, dx.T @ h
    acc = lambda n: (n / 16 + 2) * 2.0 ** -22  # noqa: E731
    out["dh"] = full(dh), full(off @ w.abs() + acc(V) * (dx.abs() @ w.abs()) * 1.1 + 2.0 ** -8 * dh.abs()) * 1.02 + 1e-30
    out["dw"] = dw, (off.T @ h.abs() + acc(max(rows.numel(), 1)) * (dx.abs().T @ h.abs()) * 1.1 + 2.0 ** -8 * dw.abs()) * 1.02 + 1e-30
    return out


def _close(got, want, what):
    value, tol = want
    assert got.shape == value.shape, what
    bad = ~((got.double() - value).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), float(((got.double() - value).abs() / tol.clamp_min(1e-300)).max()))


def _run(h, w, labels, dy, tau, **kw):
    h, w = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    y = ops.linear_log_probs(h, w, labels, temperature=tau, **kw)
    dh, dw = torch.autograd.grad(y, (h, w), dy)
    return y.detach(), dh, dw


SIZES = [(1, 8, 1), (1, 64, 1000), (2, 8, 7), (3, 72, 129), (17, 96, 128), (77, 256, 4096), (255, 64, 255), (256, 128, 257), (257, 136, 300),
         (300, 264, 1003), (600, 512, 5001), (1030, 64, 33000)]


@pytest.mark.parametrize("T,D,V", SIZES)
@pytest.mark.parametrize("answer,tau", [(1.0, 1.0), (0.5, 0.7)])
def test_values_and_gradients(T, D, V, answer, tau):
    h, w, labels, dy = _inputs(T, D, V, answer, seed=T, tau=tau)
    want = _oracle(h, w, labels, dy, tau)
    y, dh, dw = _run(h, w, labels, dy, tau)
    assert y.dtype == torch.float32 and dh.dtype == dw.dtype == torch.bfloat16
    for name, got in (("y", y), ("dh", dh), ("dw", dw)):
        _close(got, want[name], name)
    with torch.no_grad():           # (few rows have a kernel of their own without a gradient: another order of the log-sums)
        alone = ops.linear_log_probs(h, w, labels, temperature=tau)
    _close(alone, want["y"], "y alone")
    again = _run(h, w, labels, dy, tau)
    assert all(torch.equal(a, b) for a, b in zip(again, (y, dh, dw)))          # no order of summation varies


@pytest.mark.parametrize("T", [1, 2, 31, 32, 33, 63, 64, 65, 100, 128, 129])
@pytest.mark.parametrize("V", [1, 8, 31, 1000, 1185, 18944, 19001, 40000])
def test_few_rows_without_a_gradient(T, V):
    for answer, tau, D in ((1.0, 1.0, 72), (0.6, 0.7, 200)):
        h, w, labels, dy = _inputs(T, D, V, answer, seed=T + V, tau=tau)
        want = _oracle(h, w, labels, dy, tau)["y"]
        with torch.no_grad():
            y = ops.linear_log_probs(h, w, labels, temperature=tau)
            assert torch.equal(ops.linear_log_probs(h, w, labels, temperature=tau), y)
            _close(y, want, (T, V))
            h[labels == IGNORE] = float("nan")
            assert torch.equal(ops.linear_log_probs(h, w, labels, temperature=tau), y)


def test_bad_rows_without_a_gradient():
    h, w, labels, _ = _inputs(40, 64, 3000, 1.0, seed=18)
    with torch.no_grad():
        good = ops.linear_log_probs(h, w, labels)
        h[3, 5], h[9, 0] = float("nan"), float("inf")
        y = ops.linear_log_probs(h, w, labels)
        h[:] = (h * 0 + 1).nan_to_num(1, 1, 1) * 300
        far = ops.linear_log_probs(h, w, labels)
    rest = torch.tensor([i not in (3, 9) for i in range(40)], device="cuda")
    assert torch.isnan(y[3]) and torch.isnan(y[9]) and torch.equal(y[rest], good[rest])
    x = h.double() @ w.double().T
    want = (x - x.logsumexp(1, keepdim=True)).gather(1, labels[:, None])[:, 0]
    assert (far.double() - want).abs().max() <= 6 * 2.0 ** -22 * 64 * 300 * 0.3 + 8 * 2.0 ** -22 * x.abs().max() * 2


def test_every_row_without_a_label():
    h, w, labels, dy = _inputs(300, 64, 500, 0.0)
    y, dh, dw = _run(torch.full_like(h, float("nan")), w, labels, dy, 1.0)
    assert not y.any() and not dh.any() and not dw.any()


def test_what_rows_without_a_label_hold_reaches_nothing():
    h, w, labels, dy = _inputs(333, 128, 700, 0.6, seed=3)
    want = _run(h, w, labels, dy, 1.0)
    for bad in (float("nan"), float("inf"), -3e38):
        h2, dy2 = h.clone(), dy.clone()
        h2[labels == IGNORE] = bad
        dy2[labels == IGNORE] = bad
        assert all(torch.equal(a, b) for a, b in zip(_run(h2, w, labels, dy2, 1.0), want))
    odd = labels.clone()
    odd[labels == IGNORE] = torch.tensor([-1, 700, 1 << 40, -(1 << 40)], device="cuda").repeat(333)[:int((labels == IGNORE).sum())]
    assert all(torch.equal(a, b) for a, b in zip(_run(h, w, odd, dy, 1.0), want))
    zero = torch.where(labels == IGNORE, torch.zeros_like(labels), labels)      # the ignored number may be a token as well
    some = _run(h, w, torch.where(labels == 0, torch.full_like(labels, 1), zero), dy, 1.0, ignore_index=0)
    want0 = _run(h, w, torch.where(labels == 0, torch.full_like(labels, 1), labels), dy, 1.0)
    assert all(torch.equal(a, b) for a, b in zip(some, want0))


def test_a_bad_row_spoils_itself_and_the_weights_gradient_alone():
    h, w, labels, dy = _inputs(40, 64, 300, 1.0, seed=4)
    good = _run(h, w, labels, dy, 1.0)
    h2 = h.clone()
    h2[7, 3] = float("nan")
    y, dh, dw = _run(h2, w, labels, dy, 1.0)
    rest = torch.arange(40, device="cuda") != 7
    assert torch.isnan(y[7]) and torch.isnan(dh[7]).all() and torch.isnan(dw).any()
    assert torch.equal(y[rest], good[0][rest]) and torch.equal(dh[rest], good[1][rest])


def test_tokens_of_probability_one():
    """1 - p of a label that has nearly all of it comes from the exact logit: kept in 16 bits it would be lost."""
    h, w, labels, dy = _inputs(96, 128, 500, 1.0, seed=15)
    h = (h.float() * 0.05 + w[labels].float() * torch.linspace(20, 60, 96, device="cuda")[:, None]).bfloat16()
    x = h.double() @ w.double().T
    gap = 1 - (x - x.logsumexp(1, keepdim=True)).exp().gather(1, labels[:, None])[:, 0]
    assert gap.min() < 1e-4 and (gap > 1e-6).any()
    got = _run(h, w, labels, dy, 1.0)
    for name, g in zip(("y", "dh", "dw"), got):
        _close(g, _oracle(h, w, labels, dy, 1.0)[name], name)


def test_logits_far_below_the_maximum():
    """Columns more than 64 powers of two below the largest of their 128 count as nothing, and those of other columns keep their own scale."""
    h, w, labels, dy = _inputs(40, 64, 600, 1.0, seed=16)
    h = (h.float() * 6).bfloat16()
    want = _oracle(h, w, labels, dy, 1.0)
    x = h.double() @ w.double().T
    assert (x.amax(1) - x.amin(1)).min() > 64 * math.log(2)
    for name, g in zip(("y", "dh", "dw"), _run(h, w, labels, dy, 1.0)):
        _close(g, want[name], name)


def test_large_logits():
    """Differences of thousands between logits: probabilities of zero and one."""
    h, w, labels, dy = _inputs(64, 64, 1000, 1.0, seed=5)
    h = (h.float() * 100).bfloat16()
    want = _oracle(h, w, labels, dy, 1.0)
    y, dh, dw = _run(h, w, labels, dy, 1.0)
    _close(y, want["y"], "y")
    assert torch.isfinite(dh).all() and torch.isfinite(dw).all()


@pytest.mark.parametrize("layout", ["pitch", "odd", "columns", "expanded", "three", "int32"])
def test_layouts_of_rows_and_labels(layout):
    T, D, V = 66, 72, 400
    h, w, labels, dy = _inputs(T, D, V, 0.7, seed=6)
    want = _run(h, w, labels, dy, 1.0)
    shape = (T,)
    if layout == "pitch":
        x = torch.zeros(T, D + 56, device="cuda", dtype=torch.bfloat16)[:, 8:8 + D]
        x.copy_(h)
    elif layout == "odd":
        x = torch.zeros(T, D + 5, device="cuda", dtype=torch.bfloat16)[:, 3:3 + D]
        x.copy_(h)
    elif layout == "columns":
        x = h.t().contiguous().t()
    elif layout == "expanded":
        h = h[:1].expand(T, D)
        want = _run(h.contiguous(), w, labels, dy, 1.0)
        x = h
    elif layout == "three":
        shape = (2, 3, 11)
        x = h.view(2, 3, 11, D)
    else:
        x, labels = h, labels.to(torch.int32)
    y, dh, dw = _run(x, w, labels.view(shape), dy.view(shape), 1.0)
    assert y.shape == shape and dh.shape == x.shape
    for a, b in zip((y.reshape(T), dh.reshape(T, D), dw), want):
        assert torch.equal(a, b)


def test_a_single_row_without_a_dimension_of_its_own():
    h, w, labels, _ = _inputs(3, 72, 400, 1.0, seed=19)
    want = _run(h[1:2], w, labels[1:2], torch.ones(1, device="cuda"), 1.0)
    y, dh, dw = _run(h[1], w, labels[1], torch.ones((), device="cuda"), 1.0)
    assert y.shape == () and torch.equal(y, want[0][0]) and torch.equal(dh, want[1][0]) and torch.equal(dw, want[2])
    with torch.no_grad():
        assert torch.equal(ops.linear_log_probs(h[1], w, labels[1]), ops.linear_log_probs(h[1:2], w, labels[1:2])[0])


def test_two_threads_at_once():
    """Calls of two threads on streams of their own, on the same tensors: nothing of one call is another's."""
    import threading
    h, w, labels, dy = _inputs(200, 136, 3000, 0.7, seed=20)
    want = _run(h, w, labels, dy, 1.0)
    got = {}
    torch.cuda.synchronize()

    def work(k):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            outs = [_run(h, w, labels, dy, 1.0) for _ in range(5)]
        stream.synchronize()
        got[k] = outs
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for outs in got.values():
        assert len(outs) == 5 and all(torch.equal(a, b) for out in outs for a, b in zip(out, want))


@pytest.mark.parametrize("layout", ["pitch", "odd", "columns"])
def test_layouts_of_the_head(layout):
    T, D, V = 66, 72, 400
    h, w, labels, dy = _inputs(T, D, V, 0.7, seed=7)
    want = _run(h, w, labels, dy, 1.0)
    if layout == "columns":
        x = w.t().contiguous().t()
    else:
        wide = torch.zeros(V, D + 13 if layout == "odd" else D + 16, device="cuda", dtype=torch.bfloat16)
        x = wide[:, 5:5 + D] if layout == "odd" else wide[:, 8:8 + D]
        x.copy_(w)
    assert all(torch.equal(a, b) for a, b in zip(_run(h, x, labels, dy, 1.0), want))


@pytest.mark.parametrize("which", ["rows", "head"])
def test_one_gradient_alone(which):
    h, w, labels, dy = _inputs(70, 64, 300, 0.7, seed=8)
    want = _run(h, w, labels, dy, 1.0)
    leaf = (h if which == "rows" else w).requires_grad_(True)
    got, = torch.autograd.grad(ops.linear_log_probs(h, w, labels), leaf, dy)
    assert torch.equal(got, want[1 if which == "rows" else 2])


def test_main_grad_is_written_and_added_to():
    h, w, labels, dy = _inputs(70, 64, 300, 0.7, seed=9)
    want = _oracle(h, w, labels, dy, 1.0)["dw"]
    w = torch.nn.Parameter(w)
    w.main_grad = torch.full(w.shape, float("nan"), device="cuda")
    h.requires_grad_(True)
    ops.linear_log_probs(h, w, labels).backward(dy)
    assert w.grad is None and w._grad_written
    _close(w.main_grad, want, "written")
    ops.linear_log_probs(h, w, labels).backward(dy)
    _close(w.main_grad / 2, want, "added to")
    # nothing to add: what is there stays
    before = w.main_grad.clone()
    ops.linear_log_probs(h, w, torch.full_like(labels, IGNORE)).backward(dy)
    assert torch.equal(before, w.main_grad)


@pytest.mark.parametrize("V", [1000, 1283])
def test_slabs_of_the_vocabulary(V, monkeypatch):
    """The logits' gradient a part of the vocabulary at a time: disjoint parts of dw, and dh added up in fp32."""
    h, w, labels, dy = _inputs(300, 136, V, 0.8, seed=10)
    want = _oracle(h, w, labels, dy, 1.0)
    whole = _run(h, w, labels, dy, 1.0)
    for name, got in zip(("y", "dh", "dw"), whole):
        _close(got, want[name], name)
    monkeypatch.setattr(impl, "SLAB_BYTES", 2 * 512 * 256)
    assert impl._slab(512, V) == 256
    y, dh, dw = _run(h, w, labels, dy, 1.0)
    assert torch.equal(y, whole[0])
    _close(dh, want["dh"], "dh")
    _close(dw, want["dw"], "dw")
    bad = torch.where(labels[:, None] == IGNORE, torch.full_like(h, float("nan")), h)
    assert all(torch.equal(a, b) for a, b in zip(_run(bad, w, labels, dy, 1.0), (y, dh, dw)))
    p = torch.nn.Parameter(w)
    p.main_grad = torch.ones(w.shape, device="cuda")
    p._grad_written = True
    ops.linear_log_probs(h, p, labels).backward(dy)
    _close(p.main_grad - 1, (want["dw"][0], want["dw"][1] + 2.0 ** -23 * (1 + want["dw"][0].abs())), "added to")


@pytest.mark.parametrize("T,D,V", [(300, 136, 1000), (256, 64, 33000), (77, 256, 4096), (700, 512, 20000), (8000, 1024, 30000)])
def test_parts_of_the_vocabulary(T, D, V, monkeypatch):
    """dh in several parts, added up in order, against the same in one."""
    h, w, labels, dy = _inputs(T, D, V, 0.8, seed=17)
    want = _oracle(h, w, labels, dy, 1.0)
    one = _run(h, w, labels, dy, 1.0)
    monkeypatch.setattr(impl, "PLANE_BYTES", 0)
    for got in (one, _run(h, w, labels, dy, 1.0)):
        for name, g in zip(("y", "dh", "dw"), got):
            _close(g, want[name], name)


def test_gradients_against_differences():
    """Along directions of both inputs: (f(x + s) - f(x - s)) / 2 of the 64-bit definition, steps taken in bf16 numbers."""
    h, w, labels, dy = _inputs(50, 64, 200, 0.8, seed=11)
    _, dh, dw = _run(h, w, labels, dy, 1.0)
    g = torch.Generator(device="cuda").manual_seed(1)

    def f(hh, ww):
        return (_oracle(hh, ww, labels, dy, 1.0)["y"][0] * dy.double()).sum()
    for grad, at in ((dh, 0), (dw, 1)):
        base = [h.double(), w.double()]
        step = torch.randn(grad.shape, generator=g, device="cuda").double() * 1e-5
        plus, minus = list(base), list(base)
        plus[at], minus[at] = base[at] + step, base[at] - step
        num, ana = (f(*plus) - f(*minus)) / 2, (grad.double() * step).sum()
        # roundings to bf16, twice, of independent signs at most: the sum of magnitudes times 2^-7
        assert (num - ana).abs() <= 2.0 ** -7 * (grad.double().abs() * step.abs()).sum() + 1e-12


def test_replayed_and_on_other_streams():
    h, w, labels, dy = _inputs(130, 64, 700, 0.6, seed=12)
    h2, _, labels2, _ = _inputs(130, 64, 700, 0.3, seed=13)
    want, want2 = _run(h, w, labels, dy, 1.0), _run(h2, w, labels2, dy, 1.0)
    static = [t.clone() for t in (h, w, labels, dy)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = _run(*static, 1.0)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, want))
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_run(*static, 1.0))
        graphs.append(graph)
    for inputs, expect in (((h2, labels2), want2), ((h, labels), want)):
        static[0].copy_(inputs[0])
        static[2].copy_(inputs[1])
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for s, graph in zip(streams, graphs):                                    # both at once: neither shares a workspace
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(x, y) for x, y in zip(out, expect))


def test_a_graph_of_the_backward_pass_kept_and_used_twice():
    h, w, labels, dy = _inputs(60, 64, 300, 0.7, seed=14)
    h.requires_grad_(True)
    y = ops.linear_log_probs(h, w, labels)
    a, = torch.autograd.grad(y, h, dy, retain_graph=True)
    b, = torch.autograd.grad(y, h, dy)
    assert torch.equal(a, b)
    y = ops.linear_log_probs(h, w, labels)
    one, = torch.autograd.grad(y.sum(), h)                                       # an incoming gradient that is one number expanded
    y = ops.linear_log_probs(h, w, labels)
    assert torch.equal(one, torch.autograd.grad(y, h, torch.ones_like(dy))[0])


def test_no_rows_at_all():
    w = torch.randn(30, 64, device="cuda").bfloat16().requires_grad_(True)
    h = torch.randn(2, 0, 64, device="cuda").bfloat16().requires_grad_(True)
    y = ops.linear_log_probs(h, w, torch.zeros(2, 0, dtype=torch.long, device="cuda"))
    assert y.shape == (2, 0) and y.dtype == torch.float32
    dh, dw = torch.autograd.grad(y.sum(), (h, w))
    assert dh.shape == h.shape and dw.shape == w.shape and not dw.any()


def test_refusals():
    h, w, labels, _ = _inputs(5, 64, 30, 1.0)
    with pytest.raises(TypeError):
        ops.linear_log_probs(h.float(), w, labels)
    with pytest.raises(TypeError):
        ops.linear_log_probs(h, w.float(), labels)
    with pytest.raises(ValueError):
        ops.linear_log_probs(h[:, :60], w[:, :60], labels)
    with pytest.raises(ValueError):
        ops.linear_log_probs(h, w, labels.cpu())
    y = ops.linear_log_probs(h.requires_grad_(True), w, labels)
    first, = torch.autograd.grad(y.sum(), h, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.float().sum(), h)
