"""The global gradient norm and clipping against their definition in 64 bits, on the CPU and (marked) on the GPU.

Tolerances: squares are summed in 32 bits over at most 64 values of a thread, so a sum of positive terms is off by at most 66 2^-24 of itself, the
norm by half of that, and everything above is in 64 bits: 34 2^-24 with the result's rounding.  Clipped values are off by that, three
roundings of the factor and their own type's half step.
"""
import math

import pytest
import torch

from ksa_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
E = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}       # half the spacing of subnormal numbers


def _grads(sizes, dtype, device, seed=0, odd=False, std=0.02):
    """Views of one buffer for each type, each at the next free place (``odd``) or in memory of its own."""
    g = torch.Generator().manual_seed(seed)
    types = [torch.float32, torch.bfloat16, torch.float16]
    out = []
    for k, n in enumerate(sizes):
        t = types[k % 3] if dtype == "mixed" else dtype
        skip = (k * 5 + 1) % 8 if odd else 0
        v = (std * torch.randn(n + skip, generator=g)).to(t).to(device)
        out.append(v[skip:])
    return out


def _norm(grads, scale=1.0):
    return scale * math.sqrt(math.fsum(float(g.double().square().sum()) for g in grads))


def _check(grads, before, norm, most, scale=1.0):
    want = _norm(before, scale)
    assert norm.dtype == torch.float32 and norm.shape == () and abs(float(norm) - want) <= 34 * E * want + 2.0 ** -150
    factor = scale * min(1.0, most / (want + 1e-6))
    for g, b in zip(grads, before):
        exact = b.double() * factor
        assert g.dtype == b.dtype and ((g.double() - exact).abs() <= exact.abs() * (40 * E + HALF[g.dtype]) + TINY[g.dtype]).all()


SIZES = [[1], [0, 1, 0], [7, 1, 2, 3], [8192], [8191, 8193], [100003], [33] * 63, [17] * 64, [17] * 65, [5, 0] * 600, [9] * 1001, [9] * 2300,
         [1 << 20, 3, 12345], [400000] * 8]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, "mixed"], ids=str)
@pytest.mark.parametrize("odd", [False, True])
def test_norm_and_clipping(device, sizes, dtype, odd):
    grads = _grads(sizes, dtype, device, seed=len(sizes), odd=odd)
    before = [g.clone() for g in grads]
    want = _norm(before)
    norm = ops.grad_norm(grads)
    _check(grads, before, norm, math.inf)                                    # nothing has changed
    n2, factor = ops.grad_norm(iter(grads), scale=0.25, max_norm=want / 8)
    assert torch.equal(n2, norm * 0.25) and abs(float(factor) - 0.25 * min(1, want / 8 / (want / 4 + 1e-6))) <= 40 * E
    out = [torch.full_like(g, 7) for g in grads]
    _check(out, before, ops.clip_grad_norm_(grads, 0.3 * want, out=out), 0.3 * want)
    _check(grads, before, norm, math.inf)
    assert torch.equal(ops.clip_grad_norm_(grads, 2 * want + 1), norm)       # below the limit: as they are
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    _check(grads, before, ops.clip_grad_norm_(grads, 0.3 * want, scale=0.5), 0.3 * want, 0.5)
    assert all(torch.equal(a, b) for a, b in zip([g for g in grads], [g.clone() for g in grads]))


@pytest.mark.parametrize("device", DEVICES)
def test_neighbours_in_memory_stay(device):
    buffer = torch.arange(1, 4001, dtype=torch.float32, device=device).to(torch.bfloat16)
    grads = [buffer[1:1000], buffer[1001:1002], buffer[1003:1003], buffer[1500:3999]]
    want = buffer.clone()
    before = [g.clone() for g in grads]
    norm = ops.clip_grad_norm_(grads, 1.0)
    _check(grads, before, norm, 1.0)
    for lo, hi in ((0, 1), (1000, 1001), (1002, 1500), (3999, 4000)):
        assert torch.equal(buffer[lo:hi], want[lo:hi])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_magnitudes_whose_squares_leave_32_bits(device, dtype):
    for std in (1e-38, 1e-30, 1e-20, 1e18, 1e30, 1e34):
        grads = [t.to(device) for t in (torch.randn(5000).mul(std).to(dtype), torch.zeros(3000, dtype=dtype), torch.randn(3).mul(std).to(dtype))]
        want = _norm(grads)
        norm = ops.grad_norm(grads)
        # (numbers below 2^-126 are kept as they are)
        assert abs(float(norm) - want) <= 34 * E * want + 2.0 ** -150, std
    small, large = torch.full((4000,), 1e-25, device=device), torch.full((1,), 3e38, device=device)
    assert abs(float(ops.grad_norm([small, large])) - 3e38) <= 34 * E * 3e38
    assert float(ops.grad_norm([torch.full((10000,), 3e38, device=device)])) == math.inf       # the norm itself is no fp32 number


@pytest.mark.parametrize("device", DEVICES)
def test_infinities_and_what_is_no_number(device):
    for bad, norm in ((math.inf, math.inf), (-math.inf, math.inf), (math.nan, math.nan)):
        for at in (0, 5000, 9999):
            grads = [torch.ones(100, device=device), torch.ones(10000, device=device, dtype=torch.bfloat16)]
            grads[1][at] = bad
            got, factor = ops.grad_norm(grads, max_norm=1.0)
            assert str(float(got)) == str(norm) and (float(factor) == 0 if norm == math.inf else math.isnan(float(factor)))
            ops.clip_grad_norm_(grads, 1.0)
            if norm == math.inf:
                assert not grads[0].any() and torch.isnan(grads[1][at]) and not grads[1][:at].any()
            else:
                assert all(torch.isnan(g).all() for g in grads)


@pytest.mark.parametrize("device", DEVICES)
def test_no_gradients(device):
    assert float(ops.grad_norm([])) == 0 and float(ops.clip_grad_norm_([], 1.0)) == 0
    empty = [torch.empty(0, device=device), torch.empty(3, 0, device=device, dtype=torch.bfloat16)]
    norm, factor = ops.grad_norm(empty, max_norm=1.0)
    assert float(norm) == 0 and float(factor) == 1 and norm.device == empty[0].device
    zeros = [torch.zeros(50, device=device)]
    assert float(ops.clip_grad_norm_(zeros, 0.0)) == 0 and not zeros[0].any()
    ones = [torch.ones(50, device=device)]
    assert abs(float(ops.clip_grad_norm_(ones, 0.0)) - 50 ** 0.5) < 1e-5 and not ones[0].any()


@pytest.mark.parametrize("device", DEVICES)
def test_other_layouts(device):
    base = torch.randn(40, 60, device=device)
    grads = [base.clone().t(), base.clone()[:, ::2], base.clone()[3], base.clone().view(4, 10, 60).permute(2, 0, 1), torch.randn((), device=device),
             torch.ones(1, device=device).expand(5)]
    before = [g.clone() for g in grads]
    norm = ops.grad_norm(grads)
    assert abs(float(norm) - _norm(before)) <= 34 * E * _norm(before)
    _check(grads[:5], before[:5], ops.clip_grad_norm_(grads[:5], 2.0), 2.0)
    out = [torch.zeros_like(b, memory_format=torch.contiguous_format) for b in before]
    ops.clip_grad_norm_(before, 3.0, out=out)
    _check(out, before, norm, 3.0)
    apart = [torch.zeros(40, 120, device=device)[:, ::2]]
    ops.clip_grad_norm_([base], 3.0, out=apart)
    _check(apart, [base], ops.grad_norm([base]), 3.0)


@pytest.mark.parametrize("device", DEVICES)
def test_parameters_gradients_and_versions(device):
    p = torch.nn.Parameter(torch.randn(30, device=device))
    p.sum().backward()
    version = p.grad._version
    norm = ops.clip_grad_norm_((q.grad for q in (p,)), 1.0)
    assert not norm.requires_grad and p.grad._version > version
    assert abs(float(p.grad.norm()) - 1) < 1e-5
    leaf = torch.randn(20, device=device, requires_grad=True)                # what requires a gradient is a tensor like others
    ops.clip_grad_norm_([leaf], 1.0)
    assert abs(float(leaf.detach().norm()) - 1) < 1e-5


@pytest.mark.gpu
def test_same_bits_replayed_twice_at_once_and_on_another_stream():
    grads = _grads([300001, 77, 0, 40000], "mixed", "cuda", odd=True)
    out = [torch.empty_like(g) for g in grads]
    want = ops.clip_grad_norm_(grads, 1.0, out=out).clone()
    clipped = [o.clone() for o in out]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(ops.grad_norm(grads), want)
    graphs, outs = [], []
    for _ in range(2):
        mine = [torch.empty_like(g) for g in grads]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append((ops.clip_grad_norm_(grads, 1.0, out=mine), mine))
        graphs.append(graph)
    for by in (2.0, 0.5):
        for g in grads:
            g.mul_(by)
        expect = ops.clip_grad_norm_(grads, 1.0, out=out).clone()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for s, graph in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for norm, mine in outs:
            assert torch.equal(norm, expect) and all(torch.equal(a, b) for a, b in zip(mine, out))
    assert torch.equal(expect, want) and all(torch.equal(a, b) for a, b in zip(out, clipped))


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    a, b = torch.ones(10, device=device), torch.ones(6, device=device)
    for kw in (dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan"))):
        with pytest.raises(ValueError):
            ops.grad_norm([a], **kw)
    for most in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            ops.clip_grad_norm_([a], most)
        with pytest.raises(ValueError):
            ops.grad_norm([a], max_norm=most)
    for wrong in (a.double(), a.long(), None, 1.0, a.to_sparse()):
        with pytest.raises(TypeError):
            ops.grad_norm([a, wrong])
    for out in ([a], [a, a], [a, b.bfloat16()], [a, b[:5]]):
        with pytest.raises(ValueError):
            ops.clip_grad_norm_([a, b], 1.0, out=out)
    if device == "cuda":
        with pytest.raises(ValueError):
            ops.grad_norm([a, b.cpu()])
    for grads, out in (([a, a], None), ([a[:6], a[5:]], None), ([a[:5], a[5:]], [a[5:], a[:5]]), ([a], [a[:1].expand(10)]),
                       ([a[:5], a[:5]], [b[:5], b[1:]])):
        with pytest.raises(ValueError):
            ops.clip_grad_norm_(grads, 1.0, out=out)
    assert torch.equal(a, torch.ones_like(a))
    two = [torch.empty(10, device=device) for _ in range(2)]
    ops.clip_grad_norm_([a, a], 1.0, out=two)                                 # read twice: fine
    assert torch.equal(two[0], two[1])
