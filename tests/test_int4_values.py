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
