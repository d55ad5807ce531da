"""The four-bit format, the plain forms of its operators, and what they refuse."""
import pytest
import torch

from ksa_b200 import ops
from ksa_b200.ops import reference as ref


def _bf16(*shape):
    return torch.randn(*shape).bfloat16()


@pytest.mark.parametrize("group", [32, 64, 128])
def test_round_trip_is_within_half_a_step_and_the_roundings(group):
    x = _bf16(40, 2 * group)
    x[:8] *= 1e-3
    x[8:16] += 7
    x[16] = 2.5                                    # no range: exact
    codes, scale = ref.int4_quantize(x, group)
    assert codes.shape == (40, group) and scale.shape == (40, 2, 2)
    y = ref.int4_values(codes, scale).float()
    g = x.float().unflatten(-1, (-1, group))
    step = (g.amax(-1) - g.amin(-1)) / 15
    # the scale is off by 2^-8 of 16 steps, at most 31/16 of it count; the offset by 2^-8 of itself (at most |lo| + 17 steps); the result by 2^-8
    bound = step * (0.5 + 31 / 256 + 17 / 256) + g.abs().amax(-1) * 2 ** -7 * 1.01
    assert ((y - x.float()).unflatten(-1, (-1, group)).abs() <= bound[..., None]).all()
    assert torch.equal(y[16], x[16].float())


def test_order_of_codes_in_a_word():
    x = torch.arange(32.0).clamp(max=15)[None].repeat(1, 1)
    codes, scale = ref.int4_quantize(x, 32)
    word = int(codes[0, :4].contiguous().view(torch.int32)) & 0xFFFFFFFF
    got = [(word >> (4 * n)) & 15 for n in range(8)]
    c = [round((float(v) - float(scale[0, 0, 1])) / float(scale[0, 0, 0]) * 16) - 16 for v in x[0, :8]]
    assert got == [c[i] for i in (0, 2, 4, 6, 1, 3, 5, 7)]
    assert sorted(c) == c and c[0] == 0 and c[-1] > 4


def test_what_is_not_finite_or_too_large():
    x = _bf16(6, 64)
    x[0, 3], x[1, 40], x[2, 0] = float("inf"), float("nan"), float("-inf")
    x[3] = 3e38
    x[4, :32] = 1e-35
    x[4, 5] = -1e-35
    y = ref.int4_values(*ref.int4_quantize(x, 32)).float()
    assert y[0, :32].isnan().all() and y[0, 32:].isfinite().all()
    assert y[1, 32:].isnan().all() and y[1, :32].isfinite().all() and y[2, :32].isnan().all()
    assert (y[3] == 2.0 ** 126).all()
    assert (y[4, :32].abs() <= 2 ** -100).all()


def test_cache_write_read_and_slots():
    cache = ops.int4_cache(2, 3, 20, 64)
    assert cache.capacity == 32 and cache.bytes() == 2 * 2 * 3 * 32 * (32 + 8)
    k, v = _bf16(2, 4, 3, 64), _bf16(2, 4, 3, 64)
    slots = torch.tensor([[5, -1, 31, 5], [0, 32, 1 << 40, 2]])        # the last row of slot 5 stays; past the cache: not written
    ops.int4_cache_write(cache, k, v, slots)
    kr, vr = ops.int4_cache_read(cache, torch.tensor([0, -2]), 34)
    expect = ref.int4_values(*ref.int4_quantize(k, 32))
    assert torch.equal(kr[0, :, 5], expect[0, 3]) and torch.equal(kr[0, :, 31], expect[0, 2])
    assert torch.equal(kr[1, :, 2], expect[1, 0]) and torch.equal(kr[1, :, 4], expect[1, 3])
    assert torch.equal(vr[1, :, 4], ref.int4_values(*ref.int4_quantize(v, 32))[1, 3])
    written = torch.zeros(2, 34, dtype=torch.bool)
    written[0, [5, 31]] = written[1, [2, 4]] = True
    assert (kr.transpose(1, 2)[~written] == 0).all()
    assert [t.data_ptr() for t in cache.rows(slice(1, 2))] == [t[1:].data_ptr() for t in cache]


def test_norm_ahead_of_the_product():
    x, delta, norm = torch.randn(3, 64), torch.randn(2, 64), torch.rand(64) + 0.5
    w = ops.int4_quantize_weight(torch.randn(10, 64))
    for d in (None, delta):
        for glu in (False, True):
            res, y = ops.int4_norm_linear(x, d, norm, 1e-6, w, glu)
            expect = x if d is None else torch.cat([x[:2] + d, x[2:]])
            h = expect * (expect.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * norm
            assert torch.allclose(res, expect) and torch.allclose(y, (ops.int4_linear_swiglu if glu else ops.int4_linear)(h, w), atol=1e-4)
    with pytest.raises(ValueError):
        ops.int4_norm_linear(x, torch.randn(4, 64), norm, 1e-6, w)


def test_rotation_with_the_write():
    H, D, Hq = 2, 64, 4
    qkv, pos = torch.randn(3, (Hq + 2 * H) * D), torch.tensor([5, 0, 9])
    got, expect, slots = ops.int4_cache(2, H, 16, D), ops.int4_cache(2, H, 16, D), torch.tensor([3, 16])
    out = ops.int4_qk_norm_rope_decode(qkv, None, None, pos, Hq, 1e4, 1e-6, False, got, slots)
    assert torch.equal(out, ops.qk_norm_rope_packed(qkv, None, None, pos, Hq, H, D, 1e4, 1e-6, False))
    heads = out[:2, Hq * D:].view(2, 1, 2 * H, D)
    ops.int4_cache_write(expect, heads[:, :, :H], heads[:, :, H:], slots.view(2, 1))
    assert all(torch.equal(a, b) for a, b in zip(got, expect)) and got.k[0, :, 3].any() and not got.k[1].any()
    with pytest.raises(ValueError):
        ops.int4_qk_norm_rope_decode(qkv, None, None, pos, Hq, 1e4, 1e-6, False, got, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.int4_qk_norm_rope_decode(qkv[:, :-1], None, None, pos, Hq, 1e4, 1e-6, False, got, slots)


def test_attention_is_that_over_the_values_of_the_slice():
    cache = ops.int4_cache(2, 2, 48, 64)
    k, v = _bf16(2, 48, 2, 64), _bf16(2, 48, 2, 64)
    k[0, 7], v[0, 40] = float("nan"), float("inf")                     # outside every slice of the first sequence
    ops.int4_cache_write(cache, k, v, torch.arange(48).repeat(2, 1))
    q = torch.randn(2, 2, 6, 64)
    start, length = torch.tensor([[8, 20], [-3, 40]]), torch.tensor([[32, 0], [10, 100]])
    out = ops.int4_decode_attention(q, cache, start, length)
    kr, vr = (x.float() for x in ops.int4_cache_read(cache, torch.zeros(2, dtype=torch.int32), 48))
    for b, t, lo, hi in ((0, 0, 8, 40), (1, 0, 0, 7), (1, 1, 40, 48)):
        p = torch.softmax(torch.einsum("hgd,hkd->hgk", q[b, t].view(2, 3, 64), kr[b, :, lo:hi]) / 8, -1)
        assert torch.allclose(out[b, t], torch.einsum("hgk,hkd->hgd", p, vr[b, :, lo:hi]).reshape(6, 64), atol=1e-5)
    assert (out[0, 1] == 0).all()


def test_linear_is_that_with_the_values():
    w = _bf16(10, 192)
    for group in (32, 64):
        wq = ops.int4_quantize_weight(w, group)
        assert wq.shape == (10, 192) and wq.group == group and wq.scale.shape == (192 // group, 12, 2)
        x = torch.randn(3, 2, 192)
        assert torch.equal(ops.int4_linear(x, wq), x @ ops.int4_dequantize_weight(wq).float().t())
        assert torch.equal(ops.int4_dequantize_weight(wq), ref.int4_values(*ref.int4_quantize(w, group)))
    assert ops.int4_linear(torch.randn(0, 192), wq).shape == (0, 10)
    assert torch.equal(ops.int4_linear_swiglu(x, wq), ops.swiglu(ops.int4_linear(x, wq)))


def _refused(error, fn, *args, **kw):
    with pytest.raises(error):
        fn(*args, **kw)


def test_refusals():
    cache = ops.int4_cache(2, 2, 32, 64)
    k, q = _bf16(2, 3, 2, 64), torch.randn(2, 1, 4, 64)
    slots, one = torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, 1, dtype=torch.int32)
    _refused(ValueError, ops.int4_cache, 1, 1, 8, 40)
    _refused(ValueError, ops.int4_cache, 1, 1, 0, 64)
    _refused(ValueError, ops.int4_cache_write, cache, k, k[:, :2], slots)
    _refused(ValueError, ops.int4_cache_write, cache, k[:1], k[:1], slots[:1])
    _refused(ValueError, ops.int4_cache_write, cache, k[..., :32], k[..., :32], slots)
    _refused(ValueError, ops.int4_cache_write, cache, k, k, slots[:, :2])
    _refused(TypeError, ops.int4_cache_write, cache, k, k, slots.float())
    _refused(RuntimeError, ops.int4_cache_write, cache, k.clone().requires_grad_(), k, slots)
    _refused(ValueError, ops.int4_cache_read, cache, slots, 3)
    _refused(ValueError, ops.int4_cache_read, cache, slots[:, 0], -1)
    _refused(ValueError, ops.int4_decode_attention, q[:, :, :3], cache, one, one)
    _refused(ValueError, ops.int4_decode_attention, q[..., :32], cache, one, one)
    _refused(ValueError, ops.int4_decode_attention, q, cache, one[:, 0], one)
    _refused(ValueError, ops.int4_decode_attention, q, cache, one, one.repeat(1, 2))
    _refused(RuntimeError, ops.int4_decode_attention, q.clone().requires_grad_(), cache, one, one)
    _refused(TypeError, ops.int4_decode_attention, q, cache._replace(k=cache.k.int()), one, one)
    _refused(TypeError, ops.int4_decode_attention, q, cache._replace(v_scale=cache.v_scale.float()), one, one)
    _refused(ValueError, ops.int4_decode_attention, q, cache._replace(v=cache.v[:, :, :16]), one, one)
    _refused(ValueError, ops.int4_decode_attention, q, ops.Int4Cache(*(t[:, :, :24] for t in cache)), one, one)       # no multiple of 16
    _refused(ValueError, ops.int4_decode_attention, q, ops.Int4Cache(*(t.transpose(0, 1) for t in cache)), one, one)
    w = ops.int4_quantize_weight(_bf16(6, 128), 32)
    _refused(ValueError, ops.int4_quantize_weight, _bf16(6, 100), 32)
    _refused(ValueError, ops.int4_quantize_weight, _bf16(6, 128), 16)
    _refused(ValueError, ops.int4_linear, torch.randn(2, 64), w)
    _refused(ValueError, ops.int4_linear, torch.randn(2, 128), w._replace(scale=w.scale[:, :6].contiguous()))
    _refused(ValueError, ops.int4_linear, torch.randn(2, 128), w._replace(scale=w.scale[:3]))
    _refused(TypeError, ops.int4_linear, torch.randn(2, 128), w._replace(codes=w.codes.int()))
    _refused(RuntimeError, ops.int4_linear, torch.randn(2, 128, requires_grad=True), w)
    _refused(ValueError, ops.int4_linear_swiglu, torch.randn(2, 128), ops.int4_quantize_weight(_bf16(7, 128), 32))
    with torch.no_grad():
        ops.int4_linear(torch.randn(2, 128, requires_grad=True), w)
