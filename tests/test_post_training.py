"""A post-training step as it is used: the model's log probabilities, a policy or preference loss, the engine's backward pass, clipping by the
global norm and AdamW; on the CPU and (marked) on the GPU."""
import copy
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from ksa_b200 import ops
from ksa_b200.config import get_preset
from ksa_b200.losses import PolicyLoss, PreferenceLoss
from ksa_b200.models import get_model_class
from ksa_b200.training.engine import TrainEngine

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _model(device, seed=0, **over):
    cfg = get_preset("qwen3-ksa-tiny").merge({"num_layers": 2, "summary_layer_freq": [1, 0], "embed_dim": 256, "vocab_size": 1000, **over})
    model = get_model_class(cfg.model_class)(cfg)
    model.init_weights(seed=seed)
    with torch.no_grad():
        for p in model.parameters():
            p.copy_(p.bfloat16().float())              # both devices start from the same values
    return model.to(device).to(torch.bfloat16) if device == "cuda" else model


def _batch(device, seed=1, rows=4, length=128):
    g = torch.Generator().manual_seed(seed)
    tokens = torch.randint(0, 1000, (rows, length + 1), generator=g)
    labels = tokens[:, 1:].clone()
    for r in range(rows):
        labels[r, :20 + 7 * r] = -100                  # the prompt
    return tokens[:, :-1].contiguous().to(device), labels.to(device)


@pytest.mark.parametrize("device", DEVICES)
def test_model_log_probs_are_those_of_its_logits(device):
    model = _model(device)
    tokens, labels = _batch(device)
    with torch.no_grad():
        logits = model(tokens).float() / 0.8
        y = model(tokens, labels=labels, log_probs=True, temperature=0.8)
    want = torch.log_softmax(logits, -1).gather(-1, labels.clamp(min=0)[..., None])[..., 0]
    want = torch.where(labels >= 0, want, torch.zeros_like(want))
    assert y.dtype == torch.float32 and y.shape == labels.shape
    # the logits are rounded to bf16 on the GPU (2^-8 of at most 4 / 0.8), the log probabilities are not
    assert (y - want).abs().max() <= (2 * 2.0 ** -8 * float(logits.abs().max()) if device == "cuda" else 1e-4)
    with pytest.raises(ValueError):
        model(tokens, log_probs=True)


def _policy_step(model, tokens, labels, old, ref, adv, scale=1.0):
    loss_fn = PolicyLoss(kl_coef=0.05, reduction="sequence")

    def step(t, lab):
        y = model(t, labels=lab, log_probs=True)
        loss, _ = loss_fn(y, old, adv, ref, lab >= 0)
        (loss * scale).backward()
        return loss.detach()
    return step


def _plain_log_probs(model, tokens, labels):
    return torch.log_softmax(model(tokens).float(), -1).gather(-1, labels.clamp(min=0)[..., None])[..., 0]


def _gradients_agree(device, model, plain):
    """The engine's fp32 gradients against autograd's of the plain definition.  On the GPU activations and logits are bf16 on either side, and not
    rounded at the same places: some roundings of 2^-8 through two layers."""
    wanted = {n: p.grad.float() for n, p in plain.named_parameters() if p.grad is not None}
    off = torch.stack([(p.main_grad - wanted[n]).square().sum() for n, p in model.named_parameters() if n in wanted]).sum().sqrt()
    norm = torch.stack([g.square().sum() for g in wanted.values()]).sum().sqrt()
    assert off <= (8e-2 if device == "cuda" else 1e-4) * norm


@pytest.mark.parametrize("device", DEVICES)
def test_policy_step(device):
    model = _model(device)
    tokens, labels = _batch(device)
    adv, m = torch.tensor([1.0, -1.0, 0.5, -0.5], device=device), labels >= 0
    with torch.no_grad():
        start = model(tokens, labels=labels, log_probs=True)
    old, ref = start + 0.1 * torch.randn(start.shape, device=device), start - 0.2 * torch.rand(start.shape, device=device)
    plain = copy.deepcopy(model)
    y = _plain_log_probs(plain, tokens, labels)
    ratio = torch.exp(y - old)
    per = (-torch.minimum(ratio * adv[:, None], ratio.clamp(0.8, 1.2) * adv[:, None]) * m).sum(1) / m.sum(1)
    kl = ((torch.exp(ref - y) - (ref - y) - 1) * m).sum(1) / m.sum(1)
    (per + 0.05 * kl).mean().backward()
    engine = TrainEngine(model, lr=1e-3, weight_decay=0.0, clip_norm=0.5)
    loss_fn = PolicyLoss(kl_coef=0.05, reduction="sequence")

    def step(t, lab):
        loss, _ = loss_fn(model(t, labels=lab, log_probs=True), old, adv, ref, lab >= 0)
        loss.backward()
        return loss.detach()
    engine.zero_grad()
    engine.forward_backward(tokens, labels, step_fn=step)
    engine._collect_autograd_grads()
    _gradients_agree(device, model, plain)
    for _ in range(2):
        assert torch.isfinite(engine.train_step(tokens, labels, step_fn=step)) and torch.isfinite(engine.grad_norm()).all()


@pytest.mark.parametrize("device", DEVICES)
def test_preference_step(device):
    model = _model(device)
    tokens, labels = _batch(device)
    with torch.no_grad():
        ref = model(tokens, labels=labels, log_probs=True)
    plain, m = copy.deepcopy(model), labels >= 0
    total = ((_plain_log_probs(plain, tokens, labels) - ref) * m).sum(1)
    torch.nn.functional.softplus(-0.5 * (total[0::2] - total[1::2])).mean().backward()
    engine = TrainEngine(model, lr=1e-3, weight_decay=0.0, clip_norm=1.0)
    loss_fn = PreferenceLoss(beta=0.5)

    def step(t, lab):
        loss, _ = loss_fn(model(t, labels=lab, log_probs=True), ref, lab >= 0)
        loss.backward()
        return loss.detach()
    engine.zero_grad()
    # the model is its own reference: no log ratio, so log 2 (on the GPU a forward pass for a gradient rounds as one without)
    assert abs(float(engine.forward_backward(tokens, labels, step_fn=step)) - 0.6931472) < 1e-3
    engine._collect_autograd_grads()
    _gradients_agree(device, model, plain)
    for _ in range(2):
        assert torch.isfinite(engine.train_step(tokens, labels, step_fn=step)) and torch.isfinite(engine.grad_norm()).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("most", [0.05, 1e6])
def test_clipping_by_the_norm_is_torchs(device, most):
    """Two micro-batches a step: the averaged gradients, clipped, reach AdamW."""
    (t1, l1), (t2, l2) = _batch(device, 2), _batch(device, 3)
    a, b = _model(device), _model(device)
    clipped = TrainEngine(a, lr=1e-2, weight_decay=0.1, clip_norm=most, grad_accum_steps=2)
    plain = TrainEngine(b, lr=1e-2, weight_decay=0.1, grad_accum_steps=2)
    for _ in range(2):
        for t, lab in ((t1, l1), (t2, l2)):
            clipped.train_step(t, lab)
        # by hand: the same gradients, then torch's clipping of their average in 64 bits (its sum in 32 is off by 1.4e-5 here)
        if plain.micro_step == 0:
            plain.zero_grad()
        plain._write_hyper()
        for t, lab in ((t1, l1), (t2, l2)):
            plain.forward_backward(t, lab)
        plain._collect_autograd_grads()
        holders = [torch.nn.Parameter(torch.empty_like(u.grad, dtype=torch.float64)) for u in plain.units]
        for h, u in zip(holders, plain.units):
            h.grad = u.grad.double() / 2
        norm = torch.nn.utils.clip_grad_norm_(holders, most)
        if device == "cpu":         # (on the GPU attention's backward adds in an order that varies: a few roundings of bf16 values)
            assert abs(float(clipped.grad_norm()) - float(norm)) <= 40 * 2.0 ** -24 * float(norm)
        assert abs(float(clipped.grad_norm()) - float(norm)) <= 1e-3 * float(norm)
        for h, u in zip(holders, plain.units):
            u.grad.copy_(h.grad * 2)
        plain.optimizer_step()
        plain.step_count += 1
        # AdamW divides by the second moment's root: on the CPU what differs is the scale's rounding, some 2^-22 of an update of the learning
        # rate (next to eps, 1e-8, gradients count by their size: 1e-3 of it); on the GPU signs of gradients next to nothing may too
        for u, v in zip(clipped.units, plain.units):
            off = (u.master - v.master).abs()
            assert off.max() <= (1e-2 * 1e-3 if device == "cpu" else 2 * 1e-2 * 1.2) and off.mean() <= 1e-2 * 1e-2
            v.master.copy_(u.master); v.compute.copy_(u.compute); v.exp_avg.copy_(u.exp_avg); v.exp_avg_sq.copy_(u.exp_avg_sq)


def test_refusals_of_clip_norm():
    from ksa_b200.parallel.fsdp import FsdpEngine
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            TrainEngine(_model("cpu"), clip_norm=bad)
    with pytest.raises(ValueError):
        TrainEngine(_model("cpu"), clip_norm=1.0, overlap_optimizer=True)
    with pytest.raises(ValueError, match="collective"):
        FsdpEngine(_model("cpu"), clip_norm=1.0, world_size=2, rank=0, comm="fused")
    assert not TrainEngine(_model("cpu"), clip_norm=1.0).overlap_optimizer


@pytest.mark.gpu
def test_replayed_step_with_clipping_agrees_with_the_eager_one():
    tokens, labels = _batch("cuda", 4, rows=2)
    results = []
    for graphed in (False, True):
        model = _model("cuda")
        engine = TrainEngine(model, lr=1e-3, weight_decay=0.1, clip_norm=0.1)
        for _ in range(4):
            (engine.graphed_step if graphed else engine.train_step)(tokens, labels)
        results.append((engine.grad_norm().clone(), [u.master.clone() for u in engine.units]))
    assert abs(float(results[0][0]) - float(results[1][0])) <= 1e-2 * float(results[0][0])
    for u, v in zip(results[0][1], results[1][1]):
        assert (u - v).abs().max() <= 4 * 1e-3 * 2            # (attention's backward adds in an order that varies)


@pytest.mark.gpu
def test_whole_step_of_the_losses_replayed():
    """Log probabilities, both losses, their gradients and the clipped norm in one captured graph."""
    g = torch.Generator(device="cuda").manual_seed(0)
    h = torch.randn(200, 128, generator=g, device="cuda").bfloat16().requires_grad_()
    w = (0.05 * torch.randn(700, 128, generator=g, device="cuda")).bfloat16().requires_grad_()
    labels = torch.randint(0, 700, (200,), generator=g, device="cuda")
    labels[::5] = -100
    cu = torch.tensor([0, 60, 90, 150, 190], dtype=torch.int32, device="cuda")
    ref, adv = torch.randn(200, generator=g, device="cuda") - 6, torch.randn(4, generator=g, device="cuda")

    def step():
        y = ops.linear_log_probs(h, w, labels)
        loss, stats = ops.policy_loss(y, ref, adv, ref, labels >= 0, cu, kl_coef=0.1)
        other, rewards = ops.preference_loss(y, ref, labels >= 0, cu)
        grads = torch.autograd.grad(loss + other, (h, w))
        out = [torch.empty_like(x) for x in grads]
        norm = ops.clip_grad_norm_(grads, 0.01, out=out)
        return (y.detach(), loss.detach(), stats, other.detach(), rewards, norm, *out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        h.mul_(1.5)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(out, step()):
        assert torch.equal(a, b)


def _free_port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _worker(rank, world, port, out_q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        from ksa_b200.parallel.fsdp import FsdpEngine
        eng = FsdpEngine(_model("cpu"), lr=1e-2, weight_decay=0.1, clip_norm=0.05, world_size=world, rank=rank)
        tokens, labels = _batch("cpu")
        for _ in range(2):
            eng.train_step(tokens[2 * rank:2 * rank + 2].contiguous(), labels[2 * rank:2 * rank + 2].contiguous())
        out_q.put((rank, float(eng.grad_norm()), {s.name: s.param.detach().numpy().copy() for u in eng.units for s in u.slots}))
    finally:
        dist.destroy_process_group()


def test_clipping_by_the_norm_over_two_ranks():
    world, ctx = 2, mp.get_context("spawn")
    q, port = ctx.Queue(), _free_port()
    procs = [ctx.Process(target=_worker, args=(r, world, port, q)) for r in range(world)]
    for p in procs:
        p.start()
    results = sorted([q.get(timeout=180) for _ in range(world)], key=lambda r: r[0])
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    engine = TrainEngine(_model("cpu"), lr=1e-2, weight_decay=0.1, clip_norm=0.05, grad_accum_steps=2)
    tokens, labels = _batch("cpu")
    for _ in range(2):
        for r in range(2):
            engine.train_step(tokens[2 * r:2 * r + 2].contiguous(), labels[2 * r:2 * r + 2].contiguous())
    for _, norm, params in results:
        assert abs(norm - float(engine.grad_norm())) <= 1e-4 * norm
        for u in engine.units:
            for s in u.slots:
                # sums of two ranks in another order, through AdamW's quotient: a small part of two updates of the learning rate
                assert (torch.from_numpy(params[s.name]) - s.param).abs().max() <= 2 * 1e-2 * 2e-2, s.name
