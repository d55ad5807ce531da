"""Values of four bits at the ends of their range, on the CPU and as the kernels have them."""
import pytest
import torch

from ksa_b200 import ops
from ksa_b200.ops import reference as ref

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
def test_groups_as_wide_as_the_format_holds(device):
    """A group from -2^126 to 2^126: scale times 1 + c / 16 passes fp32 although the value does not.  Against the formula in 64 bits: a value is rounded to
    bf16 once, 2^-8 of it at most."""
    x = torch.randn(3, 4, 2, 64, generator=torch.Generator().manual_seed(0)).bfloat16()
    x[..., 7], x[..., 40] = 3e38, -3e38
    x[0, :, :, 3] = -2.0 ** 126
    x = x.to(device)
    cache = ops.int4_cache(3, 2, 16, 64, device)
    ops.int4_cache_write(cache, x, x, torch.arange(4, device=device, dtype=torch.int32).repeat(3, 1))
    for got, codes, scale in zip(ops.int4_cache_read(cache, torch.zeros(3, device=device, dtype=torch.int32), 4), cache[0::2], cache[1::2]):
        words = codes[:, :, :4].contiguous().view(torch.int32).long() & 0xFFFFFFFF
        c = torch.stack([(words >> (4 * n)) & 15 for n in (0, 4, 1, 5, 2, 6, 3, 7)], -1).flatten(-2).double().unflatten(-1, (2, 32))
        s, o = scale[:, :, :4, :, :1].double(), scale[:, :, :4, :, 1:].double()
        exact = (s * (1 + c / 16) + o).flatten(-2)
        assert exact.isfinite().all() and got.isfinite().all()
        assert ((got.double() - exact).abs() <= 2.0 ** -8 * exact.abs()).all()
        assert torch.equal(got, ref.int4_values(codes, scale)[:, :, :4])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D", [64, 128])
def test_rotation_of_rows_of_any_layout(device, D):
    """Rows that begin between two words, at an odd pitch, or with strided values, and strided positions: as contiguous ones, to the bit."""
    Hq, H, rows = 4, 2, 3
    W, g = (Hq + 2 * H) * D, torch.Generator().manual_seed(1)
    dtype = torch.bfloat16 if device == "cuda" else torch.float32
    draw = lambda *shape: torch.randn(*shape, generator=g).to(device, dtype)
    pos, slots = torch.tensor([5, 1, 900, 1, 77, 1], dtype=torch.int32, device=device)[::2], torch.tensor([3, 40, 9, 1], device=device)[::2]
    for qkv in (draw(rows, W + 3)[:, 1:W + 1], draw(rows, W + 1)[:, :W], draw(rows * W + 1)[1:].view(rows, W), draw(W, rows).t(), draw(1, W).expand(rows, W)):
        outs = []
        for x, p, s in ((qkv, pos, slots), (qkv.clone(memory_format=torch.contiguous_format), pos.clone(), slots.clone())):
            cache = ops.int4_cache(2, H, 16, D, device)
            outs.append((ops.int4_qk_norm_rope_decode(x, None, None, p, Hq, 1e4, 1e-6, False, cache, s), *cache))
            outs[-1] += (ops.qk_norm_rope_decode(x, None, None, p, Hq, H, D, 1e4, 1e-6, False),)
            k, v = (torch.zeros(2, H, 16, D, dtype=dtype, device=device) for _ in range(2))
            outs[-1] += (ops.qk_norm_rope_decode(x, None, None, p, Hq, H, D, 1e4, 1e-6, False, k, v, s), k, v)
        assert all(torch.equal(a, b) for a, b in zip(*outs))
        assert outs[0][1][0, :, 3].any()
    cache, qkv, ones = ops.int4_cache(2, H, 16, D, device), draw(rows, W), torch.ones(D, device=device, dtype=dtype)
    for bad in ((ones[:D // 2], None, pos), (None, torch.ones(2 * D, device=device, dtype=dtype), pos), (None, None, pos[:2]), (None, None, pos[:, None])):
        with pytest.raises(ValueError):
            ops.int4_qk_norm_rope_decode(qkv, *bad, Hq, 1e4, 1e-6, False, cache, slots)


@pytest.mark.parametrize("device", DEVICES)
def test_magnitudes_below_the_normal_ones_count_as_zero(device):
    x = torch.randn(2, 4, 1, 64, generator=torch.Generator().manual_seed(0)).bfloat16() * 1e-30
    x[0], x[0, 1], x[0, 2], x[0, 3, :, 5] = 0, -2e-39, 1e-39, 2e-39
    x[1, :, :, ::3] = 1e-39
    zeroed = torch.where(x.abs() < 2.0 ** -126, torch.zeros_like(x), x)
    assert not torch.equal(x, zeroed)
    slots, made = torch.arange(4).repeat(2, 1), []
    for rows, dev in ((x, device), (zeroed, "cpu")):
        cache = ops.int4_cache(2, 1, 16, 64, dev)
        ops.int4_cache_write(cache, rows.to(dev), rows.to(dev), slots.to(dev))
        made.append([t.cpu().float() for t in (*cache, *ops.int4_cache_read(cache, torch.zeros(2, dtype=torch.int32, device=dev), 4))])
    assert all(torch.equal(a, b) for a, b in zip(*made))
    assert made[0][4][0].count_nonzero() == 0
