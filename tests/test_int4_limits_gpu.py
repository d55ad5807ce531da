"""Operators in four bits at the ends of what they take: probabilities that need all their bits, scores and values at the ends of fp32,
infinite activations, rows of any pitch and alignment."""
import pytest
import torch

from ksa_b200 import ops
from ksa_b200.ops import _lib, reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = 2.0 ** -8                # a rounding to bf16, relative
FP32 = 2.0 ** -23               # an addition in a matrix instruction, which may truncate


def _randn(*shape, seed=0):
    return torch.randn(*shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)).bfloat16()


def _filled(k, v, cap):
    """A cache of ``cap`` slots that holds rows ``k`` and ``v`` ``[B, n, H, D]`` from slot 0 on."""
    B, n, H, D = k.shape
    cache = ops.int4_cache(B, H, cap, D, DEV)
    ops.int4_cache_write(cache, k, v, torch.arange(n, device=DEV, dtype=torch.int32).repeat(B, 1), distinct=True)
    return cache


def _exact(q, cache, lo, hi, scale):
    """Attention of ``q`` ``[B, 1, Hq, D]`` over slots lo .. hi in 64 bits: the result, sum p |v|, the scores and sum |q k|."""
    B, _, Hq, D = q.shape
    H = cache.k.shape[1]
    k, v = (ref.int4_values(c[:, :, lo:hi], s[:, :, lo:hi]).double() for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    qq = q.double().view(B, H, Hq // H, D)
    z = qq @ k.transpose(2, 3) * scale
    p = torch.softmax(z, -1)
    return tuple(x.reshape(B, Hq, -1) for x in (p @ v, p @ v.abs(), z, qq.abs() @ k.abs().transpose(2, 3) * abs(scale)))


# ------------------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 4, 128), (4, 2, 64), (32, 8, 128), (12, 2, 128), (16, 2, 64), (9, 1, 128), (32, 2, 64), (34, 2, 128)])
@pytest.mark.parametrize("cap", [96, 16400])             # on clusters, and by runs of tiles with a merge
@pytest.mark.parametrize("n", [1, 6, 40])
def test_probabilities_are_not_rounded_to_bf16(Hq, Hkv, D, cap, n):
    """Values that nearly cancel, so that a result's own rounding is small beside one of the probabilities.  Per output, A = sum p |v|: a score is off
    by its fp32 additions (D at most, of sum |q k|), two fp32 products and the exponential (2^-21), in the numerator and the denominator; a probability
    goes into the product as two bf16 terms, which leaves HALF * HALF of it; fp32 sums add 2^-23 for each of at most n + 64 additions in a row, above and below."""
    B = 2
    k, v = 0.5 * _randn(B, n, Hkv, D, seed=n), _randn(B, n, Hkv, D, seed=n + 1)
    k[:, 1::2] = k[:, 0:n - n % 2:2] + 0.02 * _randn(B, n // 2, Hkv, D, seed=n + 2)
    v[:, 1::2] = -v[:, 0:n - n % 2:2]
    cache, q = _filled(k, v, cap), 0.5 * _randn(B, 1, Hq, D, seed=n + 3)
    out = ops.int4_decode_attention(q, cache, torch.zeros(B, 1, device=DEV, dtype=torch.int32), torch.full((B, 1), n, device=DEV, dtype=torch.int32))
    _lib.check_status()
    expect, A, z, mag = _exact(q, cache, 0, n, D ** -0.5)
    score = D * FP32 * mag.amax(-1, keepdim=True) + 2 * FP32 * z.abs().amax(-1, keepdim=True) + 2.0 ** -21
    bound = HALF * expect.abs() + A * (HALF * HALF + 2.02 * score + 2 * (n + 64) * FP32)
    assert float(((out[:, 0].double() - expect).abs() / bound.clamp(min=1e-30)).max()) <= 1


@pytest.mark.parametrize("Hq,Hkv,D", [(4, 2, 128), (16, 2, 64), (32, 2, 128)])
@pytest.mark.parametrize("cap,n,low", [(96, 40, 16), (96, 90, 64), (16400, 300, 128), (16400, 300, 290)])
def test_scores_below_fp32_get_no_weight(Hq, Hkv, D, cap, n, low):
    """The scores of the first slots are products past -3.4e38; the plain form gives them no weight.  Bounds as in the test above, over the other slots."""
    k, v, q = 0.1 * _randn(1, n, Hkv, D, seed=1), _randn(1, n, Hkv, D, seed=2), _randn(1, 1, Hq, D, seed=3).abs() + 1
    k[:, :low] = -2.0 ** 126
    cache = _filled(k, v, cap)
    zero, whole = torch.zeros(1, 1, device=DEV, dtype=torch.int32), torch.full((1, 1), n, device=DEV, dtype=torch.int32)
    out = ops.int4_decode_attention(q, cache, zero, whole)
    expect, A, z, mag = _exact(q, cache, low, n, D ** -0.5)
    score = D * FP32 * mag.amax(-1, keepdim=True) + 2 * FP32 * z.abs().amax(-1, keepdim=True) + 2.0 ** -21
    bound = HALF * expect.abs() + A * (HALF + 2.02 * score + 2 * (n + 64) * FP32)
    assert ((out[:, 0].double() - expect).abs() <= bound).all()
    only = ops.int4_decode_attention(q, cache, zero, zero + low)                 # nothing has a weight: no number, as in the plain form
    assert only.isnan().all() and ref.int4_decode_attention(q.cpu(), *(t.cpu() for t in cache), zero.cpu(), zero.cpu() + low, D ** -0.5).isnan().all()
    assert (ops.int4_decode_attention(q, cache, zero, zero) == 0).all()


@pytest.mark.parametrize("Hq,Hkv,D", [(4, 2, 128), (16, 2, 64), (32, 2, 128)])
@pytest.mark.parametrize("cap,n", [(96, 90), (16400, 3000)])
def test_values_as_large_as_the_format_holds(Hq, Hkv, D, cap, n):
    """Values up to 2^126, and scores that rise by less than what moves the reference maximum: no sum of theirs may pass fp32."""
    v = (_randn(1, n, Hkv, D, seed=1).sign() * 2.0 ** 126).bfloat16()
    v[:, :, :, 0] = 2.0 ** 126
    k = torch.zeros(1, n, Hkv, D, device=DEV, dtype=torch.bfloat16)
    k[:, 16:, :, 0] = 10 / 8                                                       # e^10 = 2^14.4 times the weight of the first slots
    cache, q = _filled(k, v, cap), torch.zeros(1, 1, Hq, D, device=DEV, dtype=torch.bfloat16)
    q[..., 0] = 8
    out = ops.int4_decode_attention(q, cache, torch.zeros(1, 1, device=DEV, dtype=torch.int32), torch.full((1, 1), n, device=DEV, dtype=torch.int32), 1.0)
    expect, A, z, mag = _exact(q, cache, 0, n, 1.0)
    score = D * FP32 * mag.amax(-1, keepdim=True) + 2 * FP32 * z.abs().amax(-1, keepdim=True) + 2.0 ** -21
    assert out.isfinite().all()
    assert ((out[:, 0].double() - expect).abs() <= HALF * expect.abs() + A * (HALF + 2.02 * score + 2 * (n + 64) * FP32)).all()


# ------------------------------------------------------------------------------------------------- products
@pytest.mark.parametrize("N,K,group", [(300, 160, 32), (5, 32, 32), (64, 2080, 32), (1000, 320, 64), (777, 384, 128), (12000, 1568, 32)])
def test_infinite_activations(N, K, group):
    """An infinity times a weight is one, and a NaN only where the weight is zero, wherever in the row it stands and however many rows there are."""
    w = ops.int4_quantize_weight((_randn(N, K, seed=N) * 0.05).bfloat16(), group)
    wd = ops.int4_dequantize_weight(w).double().cpu()
    for M in (1, 5, 8, 11, 16, 20, 40):
        x = _randn(M, K, seed=M)
        for m, c in enumerate((3, K - 1, 31, K // 2, 0)):
            if m < M:
                x[m, c] = float("inf") if m % 2 == 0 else float("-inf")
        expect = x.double().cpu() @ wd.t()
        got = ops.int4_linear(x, w).double().cpu()
        assert torch.equal(got.isnan(), expect.isnan()) and torch.equal(got[expect.isinf()], expect[expect.isinf()]), M
        assert torch.equal(got.isfinite(), expect.isfinite())
        if N % 2 == 0:
            F = N // 2
            glu, finite = ops.int4_linear_swiglu(x, w), expect.isfinite()
            both = finite[:, :F] & finite[:, F:]
            assert glu.cpu()[both].isfinite().all()
    _lib.check_status()


def test_one_row_at_any_pitch():
    """A single row counts as contiguous at any pitch."""
    for N, K in ((200, 256), (12000, 1536)):
        w = ops.int4_quantize_weight(_randn(N, K, seed=1))
        wd = ops.int4_dequantize_weight(w).double()
        for x in (_randn(K, 1, seed=2).t(), _randn(1, K + 3, seed=3)[:, :K], _randn(4, K + 1, seed=4)[:1, :K], _randn(1, K, seed=5).as_strided((1, K), (0, 1))):
            assert x.is_contiguous()
            for xx in (x, x[0], x[None]):
                y = ops.int4_linear(xx, w)
                expect, mag = xx.double() @ wd.t(), xx.double().abs() @ wd.abs().t()
                assert y.shape == expect.shape
                assert ((y.double() - expect).abs() <= HALF * expect.abs() + (K / 16 + 64) * FP32 * mag).all()
            assert torch.equal(ops.int4_linear_swiglu(x, w), ops.int4_linear_swiglu(x.clone(), w))


def _layouts(M, K):
    """Rows between two vectors of 16 bytes, at an odd pitch, with strided values, one row for all, rows within one another."""
    return (_randn(M * K + 1, seed=2)[1:].view(M, K), _randn(M, K + 3, seed=3)[:, 1:K + 1], _randn(K, M, seed=4).t(), _randn(1, K, seed=5).expand(M, K),
            _randn(M * K, seed=6).as_strided((M, K), (8, 1)))


@pytest.mark.parametrize("N,K", [(96, 256), (2500, 2048)])
def test_many_rows_of_any_layout(N, K):
    w = ops.int4_quantize_weight((_randn(N, K, seed=1) * 0.1).bfloat16())
    for M in (12, 30, 200):
        for x in _layouts(M, K):
            plain = x.clone(memory_format=torch.contiguous_format)
            wd = ops.int4_dequantize_weight(w).double()
            expect, mag = plain.double() @ wd.t(), plain.double().abs() @ wd.abs().t()
            assert ((ops.int4_linear(x, w).double() - expect).abs() <= HALF * expect.abs() + (K / 16 + 64) * FP32 * mag).all()
            assert torch.equal(ops.int4_linear_swiglu(x, w), ops.int4_linear_swiglu(plain, w))


@pytest.mark.parametrize("M", [1, 3, 4, 9])
@pytest.mark.parametrize("K", [256, 8192, 9728, 40960])
def test_norm_ahead_of_the_product_takes_rows_of_any_layout_and_width(M, K):
    """Bounds as in the test of this operator: a rounding of the norm, 2^-20 of its fp32, and those of the product."""
    w = ops.int4_quantize_weight((_randn(64, K, seed=1) * 0.1).bfloat16())
    wd, norm_w = ops.int4_dequantize_weight(w).double(), (1 + _randn(2 * K + 1, seed=2) * 0.2).bfloat16()
    for x in _layouts(M, K):
        for delta in (None, _randn(M, K + 1, seed=7)[:, 1:], _randn(K, M // 2, seed=8).t()):
            for nw in (norm_w[1:K + 1], norm_w[:2 * K:2]):
                res, y = ops.int4_norm_linear(x, delta, nw, 1e-6, w)
                expect = x.clone(memory_format=torch.contiguous_format)
                if delta is not None:
                    n = delta.shape[0]
                    expect[:n] = (expect[:n].float() + delta.float()).bfloat16()
                assert torch.equal(res, expect)
                r = expect.double()
                h = r * (r.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * nw.double()
                p, mag = h @ wd.t(), h.abs() @ wd.abs().t()
                assert ((y.double() - p).abs() <= (HALF + 2.0 ** -20) * 1.01 * mag + HALF * p.abs() * 1.01 + (K / 16 + 64) * FP32 * mag * 1.01).all()
                assert torch.equal(ops.int4_norm_linear(x, delta, nw, 1e-6, w, True)[1].isfinite(), torch.ones(M, 32, device=DEV, dtype=torch.bool))
    _lib.check_status()
