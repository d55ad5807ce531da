"""The plain form of ``ops.linear_log_probs``, its refusals, and the sizes that the kernels' callers work out."""
import pytest
import torch
import torch.nn.functional as F

from ksa_b200 import ops
from ksa_b200.ops import log_probs as impl


def _inputs(*rows, D=16, V=40):
    h, w = torch.randn(*rows, D, requires_grad=True), torch.randn(V, D, requires_grad=True)
    return h, w, torch.randint(0, V, rows)


@pytest.mark.parametrize("tau", [1.0, 0.7])
@pytest.mark.parametrize("rows", [(1,), (9,), (3, 5), (2, 1, 4)])
def test_plain_form(rows, tau):
    h, w, labels = _inputs(*rows)
    labels.view(-1)[0] = -100
    y = ops.linear_log_probs(h, w, labels, temperature=tau)
    full = F.log_softmax(h.double() @ w.double().T / tau, -1)
    want = torch.where(labels >= 0, full.gather(-1, labels.clamp(min=0)[..., None])[..., 0], torch.zeros((), dtype=torch.float64))
    assert y.dtype == torch.float32 and y.shape == rows and (y.double() - want).abs().max() < 1e-4
    dy = torch.randn(rows)
    for a, b in zip(torch.autograd.grad(y, (h, w), dy), torch.autograd.grad(want, (h, w), dy.double())):
        assert (a - b).abs().max() < 1e-4
    assert not torch.autograd.grad(ops.linear_log_probs(h, w, labels).sum(), h)[0].reshape(-1, 16)[0].any()


def test_labels_of_32_bits():
    h, w, labels = _inputs(9)
    assert torch.equal(ops.linear_log_probs(h, w, labels.int()), ops.linear_log_probs(h, w, labels))


def test_mean_of_the_labels_is_cross_entropy():
    h, w, labels = _inputs(30)
    labels[::3] = -100
    y = ops.linear_log_probs(h, w, labels)
    assert abs(float((-y.sum() / (labels >= 0).sum() - ops.linear_cross_entropy(h, w, labels)).detach())) < 1e-5


def test_rows_without_a_label_may_hold_anything():
    h, w, labels = _inputs(6)
    labels[2], labels[3], labels[4] = -100, 40, -1
    bad = h.detach().clone()
    bad[2:5] = float("nan")
    bad.requires_grad_(True)
    y = ops.linear_log_probs(bad, w, labels)
    assert torch.equal(y, ops.linear_log_probs(h, w, labels)) and not y[2:5].any()
    dh, dw = torch.autograd.grad(y.sum(), (bad, w))
    assert torch.isfinite(dh).all() and torch.isfinite(dw).all() and not dh[2:5].any()


def test_refusals():
    h, w, labels = _inputs(6)
    for args, kw in (((h, w[:, :8], labels), {}), ((h, w, labels[:5]), {}), ((h, w, labels.float()), {}), ((h, w[0], labels), {}),
                     ((h, w, labels), dict(temperature=0.0)), ((h, w, labels), dict(temperature=-1.0)), ((h, w, labels), dict(temperature=float("inf"))),
                     ((h, w, labels), dict(temperature=float("nan"))), ((h, w[:0], labels), {}), ((h[0], w, labels[0, None]), {})):
        with pytest.raises(ValueError):
            ops.linear_log_probs(*args, **kw)


def test_slabs_cover_the_vocabulary_in_multiples():
    for rows in (256, 512, 8192, 32768, 1 << 20, 1 << 24):
        for V in (1, 7, 255, 256, 4096, 151936):
            slab = impl._slab(rows, V)
            assert slab % 64 == 0 and (slab >= V or slab % 256 == 0) and slab <= -(-V // 64) * 64
            assert 2 * rows * slab <= max(impl.SLAB_BYTES, 2 * rows * 256)
