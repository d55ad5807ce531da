"""The policy and preference losses where a term is infinite or nothing, and with as many sequences as tokens, on the CPU and (marked) on the GPU."""
import math

import pytest
import torch

from ksa_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
INF = math.inf


def _on(device, *values):
    return [torch.tensor(v, device=device) for v in values]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("reduction", ["token", "sequence"])
@pytest.mark.parametrize("by_sequence", [False, True])
def test_no_advantage_is_no_policy_loss_whatever_the_ratio(device, reduction, by_sequence):
    """-min(r 0, clip(r) 0) is 0 for a ratio that overflows, is infinite or is zero; the other tokens keep loss and gradient."""
    y, old = _on(device, [[0.0, 0.0, 0.0, -INF], [-1.0, -1.0, -1.0, -1.0]], [[-100.0, -INF, 200.0, -1.0], [-1.0, -1.0, -1.0, -1.0]])
    y.requires_grad_(True)
    adv = torch.tensor([0.0, 1.0], device=device)
    if not by_sequence:
        adv = adv[:, None].expand(2, 4).contiguous()
    loss, stats = ops.policy_loss(y, old, adv, reduction=reduction)
    dy, = torch.autograd.grad(loss, y)
    assert float(loss.detach()) == -0.5 and stats.tolist() == [-0.5, 0.0, 0.0]
    assert torch.equal(dy.cpu(), torch.tensor([[0.0] * 4, [-0.125] * 4]))
    # a difference that is no number stays one
    with torch.no_grad():
        y[0, 0] = old[0, 0] = -INF
    assert math.isnan(float(ops.policy_loss(y, old, adv, reduction=reduction)[0].detach()))


@pytest.mark.parametrize("device", DEVICES)
def test_the_gradient_of_the_kl_term_stays_without_an_advantage(device):
    y, old, ref, adv = _on(device, [0.0, 0.0], [-100.0, 0.0], [0.5, -0.5], [0.0, 0.0])
    y.requires_grad_(True)
    loss, _ = ops.policy_loss(y, old, adv, ref, kl_coef=0.5)
    want = 0.5 * sum(math.expm1(x) - x for x in (0.5, -0.5)) / 2
    assert abs(float(loss.detach()) - want) <= 1e-6
    dy, = torch.autograd.grad(loss, y)
    assert all(abs(float(g) + 0.25 * math.expm1(x)) <= 1e-6 for g, x in zip(dy, (0.5, -0.5)))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("wide", [False, True])
def test_as_many_sequences_as_tokens(device, wide):
    """Two of the four sequences are empty.  A shape that is the log probabilities' own is a value for every token, any other one for every
    sequence: tokens 0 and 1 are sequence 1, tokens 2 and 3 are sequence 3."""
    cu = torch.tensor([0, 0, 2, 2, 4], device=device, dtype=torch.int64 if wide else torch.int32)
    y = torch.zeros(4, device=device)
    adv = torch.tensor([1.0, 2.0, 3.0, 4.0], device=device)
    by_token, by_sequence = -2.5, -3.0
    for rows, a, want in ((y, adv, by_token), (y, adv[:, None], by_sequence), (y[None], adv[None], by_token), (y[None], adv, by_sequence),
                          (y[None], adv[:, None], by_sequence)):
        for leaf in (rows, rows.clone().requires_grad_(True)):
            loss, stats = ops.policy_loss(leaf, torch.zeros_like(rows), a, cu_seqlens=cu)
            assert float(loss.detach()) == want and float(stats[0]) == want
            if leaf.requires_grad:
                dy, = torch.autograd.grad(loss, leaf)
                assert dy.reshape(-1).tolist() == ([-0.25, -0.5, -0.75, -1.0] if want == by_token else [-0.5, -0.5, -1.0, -1.0])
    # the tokens behind the last offset belong to no sequence
    loss, _ = ops.policy_loss(y, torch.zeros_like(y), adv[:, None], cu_seqlens=torch.tensor([0, 0, 1, 1, 3], device=device))
    assert abs(float(loss) + (2.0 + 4.0 + 4.0) / 3) <= 1e-6


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("smoothing", [0.0, 0.1, 1.0])
def test_preference_at_infinities(device, smoothing):
    """(1 - s) log(1 + exp(-z)) + s log(1 + exp(z)): infinite on the side that counts, and never infinity less infinity."""
    for better, worse, z in ((-INF, 0.0, -INF), (0.0, -INF, INF), (-1e30, 0.0, -1e30), (0.0, -1e30, 1e30)):
        y = torch.tensor([[better, 0.0], [worse, 0.0]], device=device, requires_grad=True)
        loss, rewards = ops.preference_loss(y, beta=1.0, label_smoothing=smoothing)
        weight = 1 - smoothing if z < 0 else smoothing
        want = weight * abs(z) if weight else 0.0
        assert float(loss.detach()) == want or abs(float(loss.detach()) - want) <= 2.0 ** -22 * want
        assert rewards.flatten().tolist() == [float(torch.tensor(better)), float(torch.tensor(worse))]
        g = smoothing - (1.0 if z < 0 else 0.0)
        dy, = torch.autograd.grad(loss, y)
        assert all(abs(float(a) - b) <= 2.0 ** -23 for a, b in zip(dy.flatten(), (g, g, -g, -g)))
    both = torch.full((2, 1), -INF, device=device)
    assert math.isnan(float(ops.preference_loss(both, label_smoothing=smoothing)[0]))


@pytest.mark.parametrize("device", DEVICES)
def test_an_infinite_kl_term(device):
    """exp(x) - 1 - x grows beyond all numbers on both sides."""
    for x in (INF, -INF, 200.0, -1e30):
        ref = torch.tensor([x], device=device)
        loss, stats = ops.policy_loss(torch.zeros(1, device=device), torch.zeros(1, device=device), torch.zeros(1, device=device), ref, kl_coef=1.0)
        assert float(loss) == float(stats[1]) and (float(loss) == INF if x != -1e30 else abs(float(loss) - 1e30) <= 1e24)


@pytest.mark.parametrize("device", DEVICES)
def test_gradient_of_an_infinite_kl_term(device):
    """-(exp(x) - 1): beyond all numbers where the reference has a token that the model has not, 1 where it is the other way round."""
    y = torch.zeros(3, device=device, requires_grad=True)
    ref, adv = _on(device, [INF, -INF, 0.0], [0.0, 0.0, 1.0])
    loss, stats = ops.policy_loss(y, torch.zeros_like(y), adv, ref, kl_coef=0.5)
    dy, = torch.autograd.grad(loss, y)
    assert float(loss.detach()) == INF and stats.tolist()[1] == INF
    assert float(dy[0]) == -INF and abs(float(dy[1]) - 0.5 / 3) <= 2.0 ** -24 and abs(float(dy[2]) + 1 / 3) <= 2.0 ** -24
    # without a coefficient the reference counts in the statistics alone
    loss, stats = ops.policy_loss(y, torch.zeros_like(y), adv, ref)
    assert abs(float(loss.detach()) + 1 / 3) <= 2.0 ** -24 and float(stats[1]) == INF
    assert torch.equal(torch.autograd.grad(loss, y)[0].cpu(), torch.tensor([0.0, 0.0, -1 / 3]))
