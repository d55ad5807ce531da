"""Where a post-training step is refused or takes another path, and that both ways to the kernels agree."""
from types import SimpleNamespace

import pytest
import torch

from ksa_b200 import ops
from ksa_b200.ops import token_losses as tl_impl
from ksa_b200.parallel import fsdp
from ksa_b200.training.engine import TrainEngine
from test_post_training import _batch, _model


def test_log_probs_of_a_shard_of_the_sequence_are_refused():
    """Under context parallelism a rank has parts of answers, and a loss of those is another loss."""
    model = _model("cpu")
    tokens, labels = _batch("cpu")
    model.cp = SimpleNamespace()
    with pytest.raises(ValueError, match="shard"):
        model(tokens, labels=labels, log_probs=True)


def test_log_probs_of_the_last_token_alone_are_refused():
    """Its logits would come back in their place."""
    model = _model("cpu")
    tokens, labels = _batch("cpu")
    with pytest.raises(ValueError, match="log_probs"):
        model(tokens, labels=labels, log_probs=True, last_token_only=True)


@pytest.mark.parametrize("clip_norm,comm,want", [(0.0, None, "fused"), (1.0, None, "collective"), (1.0, "collective", "collective"), (0.0, "collective", "collective")])
def test_clipping_by_the_norm_takes_the_back_end_that_has_it(clip_norm, comm, want, monkeypatch):
    """On the GPUs of one node, without a back end asked for."""
    class Reached(Exception):
        pass

    def stop(*args, **kw):
        raise Reached
    monkeypatch.setattr(TrainEngine, "__init__", stop)
    engine = fsdp.FsdpEngine.__new__(fsdp.FsdpEngine)
    with pytest.raises(Reached):
        engine.__init__(torch.nn.Linear(2, 2), device=torch.device("cuda"), world_size=2, rank=0, comm=comm, clip_norm=clip_norm)
    assert engine.comm == want


@pytest.mark.gpu
@pytest.mark.parametrize("most", [0.05, 1e6])
def test_replayed_steps_scale_by_the_clip_factor(most):
    """What AdamW multiplies the gradients by after every step, eager and replayed: 1/2 for two micro-batches, times the factor of the norm."""
    (t1, l1), (t2, l2) = _batch("cuda", 5, rows=2), _batch("cuda", 6, rows=2)
    for graphed in (False, True):
        engine = TrainEngine(_model("cuda"), lr=1e-3, clip_norm=most, grad_accum_steps=2)
        for _ in range(4):
            for t, lab in ((t1, l1), (t2, l2)):
                (engine.graphed_step if graphed else engine.train_step)(t, lab)
            norm = float(engine.grad_norm())
            want = 0.5 * min(1.0, most / (norm + 1e-6))
            # the norm comes back as the root of its square in 32 bits: some roundings
            assert abs(float(engine.hyper[3]) - want) <= 8 * 2.0 ** -24 * want
            assert (norm > most) == (most < 1)


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_both_ways_to_the_losses_decide_alike(packed, reduction, monkeypatch):
    """Calls by way of Python and of native code give the same bits."""
    g = torch.Generator(device="cuda").manual_seed(0)
    shape = (5003,) if packed else (6, 801)
    y, old, ref = (torch.randn(shape, generator=g, device="cuda") - 3 for _ in range(3))
    mask = torch.rand(shape, generator=g, device="cuda") < 0.8
    cu = torch.tensor([0, 7, 7, 2100, 4500, 4501, 4990], device="cuda") if packed else None
    y.requires_grad_()

    def run():
        outs = []
        for adv in (torch.linspace(-1, 1, 6, device="cuda"), old.detach() + 3):
            for kl in (0.0, 0.1):
                loss, stats = ops.policy_loss(y, old, adv, ref, mask, cu, kl_coef=kl, reduction=reduction)
                outs += [loss.detach(), stats, *torch.autograd.grad(loss, y)]
        for smoothing in (0.0, 0.2):
            loss, rewards = ops.preference_loss(y, ref, mask, cu, label_smoothing=smoothing)
            outs += [loss.detach(), rewards, *torch.autograd.grad(loss, y)]
        return outs
    native = run()
    monkeypatch.setattr(tl_impl, "_native", SimpleNamespace(policy_loss=lambda *args: None, preference_loss=lambda *args: None))
    assert all(torch.equal(a, b) for a, b in zip(run(), native))
