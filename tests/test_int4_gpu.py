"""Cache writes, decode attention and products in four bits on the GPU against plain forms in 64 bits."""
import pytest
import torch

from ksa_b200 import ops
from ksa_b200.ops import _lib, reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = 2.0 ** -8                # a rounding to bf16, relative
FP32 = 2.0 ** -23               # an addition in a matrix instruction, which may truncate


def _gen(seed=0):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(*shape, seed=0):
    return torch.randn(*shape, device=DEV, generator=_gen(seed)).bfloat16()


def _same(a, b):
    assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


# ------------------------------------------------------------------------------------------------- cache
@pytest.mark.parametrize("B,T,H,D,cap", [(1, 1, 8, 128, 32), (3, 5, 2, 64, 48), (2, 17, 3, 96, 64), (5, 64, 1, 32, 80), (2, 65, 2, 128, 96),
                                         (1, 700, 4, 256, 704)])
def test_write_and_read_are_the_plain_form_to_the_bit(B, T, H, D, cap):
    rows = _randn(B, T, 2 * H + 3, D, seed=T)
    rows[..., :7] *= 30
    rows[0, 0, 0, 0] = float("nan")
    rows[B - 1, T - 1, H - 1, D - 1] = float("-inf")
    rows[0, T // 2, H, :32] = 1.5
    rows[0, T - 1, H, 5] = 3e38
    k, v = rows[:, :, :H], rows[:, :, H + 3:]                            # views of packed rows
    slots = torch.stack([torch.randperm(cap, device=DEV, generator=_gen(b))[:T] for b in range(B)]).to(torch.int32)
    cache = ops.int4_cache(B, H, cap, D, DEV)
    for t in cache:
        t.view(torch.uint8).fill_(0x5A)
    before = [t.clone() for t in cache]
    if T > 2:
        slots[:, 1] = -1
    ops.int4_cache_write(cache, k, v, slots)
    _lib.check_status()
    expect = [t.clone() for t in before]
    for rows_, c, s in ((k, 0, 1), (v, 2, 3)):
        codes, scale = ref.int4_quantize(rows_, 32)
        for b in range(B):
            for t in range(T):
                if slots[b, t] >= 0:
                    expect[c][b, :, slots[b, t]], expect[s][b, :, slots[b, t]] = codes[b, t], scale[b, t]
    for got, want in zip(cache, expect):                                 # untouched slots included
        _same(got.float(), want.float())
    start = torch.arange(B, device=DEV, dtype=torch.int32) * 3 - 2       # some slots outside the cache
    got = ops.int4_cache_read(cache, start, cap + 1)
    for x, c, s in ((got[0], cache.k, cache.k_scale), (got[1], cache.v, cache.v_scale)):
        for b in range(B):
            at = torch.arange(cap + 1, device=DEV) + start[b]
            inside = (at >= 0) & (at < cap)
            _same(x[b][:, inside], ref.int4_values(c[b], s[b])[:, at[inside]])
            assert (x[b][:, ~inside] == 0).all()


def test_codes_next_to_the_middle_between_two():
    """Rows on a coarse grid: many values lie exactly between two codes, or a rounding away from it."""
    g = _gen(7)
    B, T, H, D = 2, 600, 2, 128
    k = (torch.randint(-64, 65, (B, T, H, D), device=DEV, generator=g) / 16).bfloat16()
    scale = torch.exp2(torch.randint(-110, 110, (B, T, H, 1), device=DEV, generator=g).float())
    v = (torch.randint(-30, 31, (B, T, H, D), device=DEV, generator=g).float() * scale).bfloat16()
    cache = ops.int4_cache(B, H, T, D, DEV)
    ops.int4_cache_write(cache, k, v, torch.arange(T, device=DEV).repeat(B, 1), distinct=True)
    ties = 0
    for rows, codes, scales in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        c, s = ref.int4_quantize(rows.cpu(), 32)
        s_, o_ = s[..., 0].double().repeat_interleave(32, -1), s[..., 1].double().repeat_interleave(32, -1)
        y = (rows.cpu().double() - o_) / s_ * 16
        ties += int(((y - y.floor() - 0.5).abs() < 1e-9).sum())
        assert torch.equal(codes[:, :, :T].transpose(1, 2).cpu(), c)
        _same(scales[:, :, :T].transpose(1, 2).cpu().float(), s.float())
    assert ties > 1000                  # the inputs are what they are meant to be


@pytest.mark.parametrize("T", [2, 64, 65, 3000])
def test_the_last_row_of_a_slot_stays(T):
    B, H, D, cap = 2, 2, 64, 32
    k, v = _randn(B, T, H, D, seed=1), _randn(B, T, H, D, seed=2)
    slots = torch.randint(-2, cap + 2, (B, T), device=DEV, generator=_gen(3))        # int64, some outside
    slots[0, 0] = 1 << 33
    cache = ops.int4_cache(B, H, cap, D, DEV)
    ops.int4_cache_write(cache, k, v, slots)
    plain = ops.int4_cache(B, H, cap, D)
    ops.int4_cache_write(plain, k.cpu(), v.cpu(), slots.cpu())
    for a, b in zip(cache, plain):
        _same(a.cpu().float(), b.float())


@pytest.mark.parametrize("B,T,H,D,cap", [(3, 65, 1, 32, 48), (5, 100, 2, 32, 16), (2, 1501, 2, 64, 8192), (1, 2048, 1, 128, 80), (1, 2049, 1, 128, 80),
                                         (2, 300, 2, 64, 8208), (9, 1000, 8, 64, 1008), (3, 70, 1, 2048, 32)])
def test_the_last_row_of_a_slot_stays_however_it_is_found(B, T, H, D, cap):
    k, v = _randn(B, T, H, D, seed=1), _randn(B, T, H, D, seed=2)
    slots = torch.randint(-2, min(cap, T // 2) + 2, (B, T), device=DEV, generator=_gen(3), dtype=torch.int32)
    cache, once = ops.int4_cache(B, H, cap, D, DEV), ops.int4_cache(B, H, cap, D, DEV)
    ops.int4_cache_write(cache, k, v, slots)
    later = (slots[:, None, :] == slots[:, :, None]) & (torch.arange(T, device=DEV)[None, None, :] > torch.arange(T, device=DEV)[None, :, None])
    ops.int4_cache_write(once, k, v, torch.where(later.any(2), -1, slots).to(torch.int32), distinct=True)
    for a, b in zip(cache, once):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows,n,Hq,H,D", [(1, 1, 32, 8, 128), (5, 3, 4, 2, 128), (16, 16, 2, 1, 128), (4, 4, 4, 2, 64), (3, 0, 2, 1, 128)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norms", [False, True])
def test_rotation_with_the_write_is_both_to_the_bit(rows, n, Hq, H, D, interleaved, norms):
    qkv = _randn(rows, (Hq + 2 * H) * D + 16, seed=rows)[:, :(Hq + 2 * H) * D]
    q_w, k_w = (1 + _randn(D, seed=1) * 0.1, 1 + _randn(D, seed=2) * 0.1) if norms else (None, None)
    pos = torch.arange(rows, device=DEV) * 1000 + 3
    slots = torch.tensor([7, -1, 48, 47, -5, 31, 0, 1, 2, 3, 4, 5, 6, 8, 9, 10], device=DEV, dtype=torch.int32)[:n]
    got, expect = _cache(n + 1, H, 48, D, seed=3), _cache(n + 1, H, 48, D, seed=3)
    out = ops.int4_qk_norm_rope_decode(qkv, q_w, k_w, pos, Hq, 1e4, 1e-6, interleaved, got, slots)
    assert torch.equal(out, ops.qk_norm_rope_decode(qkv, q_w, k_w, pos, Hq, H, D, 1e4, 1e-6, interleaved))
    heads = out[:n, Hq * D:].view(n, 1, 2 * H, D)
    ops.int4_cache_write(expect.rows(slice(0, n)), heads[:, :, :H], heads[:, :, H:], slots.view(n, 1))
    for a, b in zip(got, expect):
        assert torch.equal(a, b)
    with pytest.raises(ValueError):
        ops.int4_qk_norm_rope_decode(qkv, q_w, k_w, pos, Hq, 1e4, 1e-6, interleaved, got, torch.zeros(rows + 1, device=DEV, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.int4_qk_norm_rope_decode(qkv, q_w, k_w, pos, Hq + 1, 1e4, 1e-6, interleaved, got, slots)


def test_write_takes_rows_of_any_layout():
    B, T, H, D = 2, 6, 2, 64
    base = _randn(B, H, D, T + 1, seed=4)
    k, v = base[..., :T].permute(0, 3, 1, 2), base[..., 1:].permute(0, 3, 1, 2)        # last dimension strided
    odd = _randn(B * T * H * D + 1, seed=5)[1:].view(B, T, H, D)                        # off the 16-byte grid
    slots = torch.arange(T, device=DEV, dtype=torch.int32).repeat(B, 1)
    for a, b in ((k, v), (odd, odd), (k, odd)):
        cache, plain = ops.int4_cache(B, H, 16, D, DEV), ops.int4_cache(B, H, 16, D, DEV)
        ops.int4_cache_write(cache, a, b, slots, distinct=True)
        ops.int4_cache_write(plain, a.contiguous().clone(), b.contiguous().clone(), slots)
        for x, y in zip(cache, plain):
            assert torch.equal(x, y)


# ------------------------------------------------------------------------------------------------- attention
def _cache(B, H, cap, D, seed=0):
    """A cache filled with channels of unlike spread and shift."""
    g = _gen(seed)
    spread = torch.exp(0.5 * torch.randn(D, device=DEV, generator=g))
    shift = 2 * torch.randn(D, device=DEV, generator=g)
    cache = ops.int4_cache(B, H, cap, D, DEV)
    for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        codes, scale = ref.int4_quantize((torch.randn(B, H, cap, D, device=DEV, generator=g) * spread + shift).bfloat16(), 32)
        c.copy_(codes)
        s.copy_(scale)
    return cache


def _check_attention(out, q, cache, start, length, scale):
    """Against 64 bits.  Per output, A = sum p |v| of the slice: a probability is rounded to bf16 (HALF), the result as well (HALF of itself); a
    score is off by its fp32 additions (D of them at most, of sum |q k|), by two fp32 products and the exponential (2^-21), in the
    numerator and the denominator; sums and merges of fp32 add 2^-23 for each of at most len / 8 + 600 additions in a row."""
    B, Tq, Hq, D = q.shape
    H, cap = cache.k.shape[1], cache.capacity
    worst = 0.0
    for b in range(B):
        for t in range(Tq):
            first = int(start[b, t])
            lo, hi = max(0, first), min(cap, first + max(0, int(length[b, t])))
            if hi <= lo:
                assert (out[b, t] == 0).all()
                continue
            k, v = (ref.int4_values(c[b, :, lo:hi], s[b, :, lo:hi]).double() for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
            qq = q[b, t].double().view(H, Hq // H, D)
            z = qq @ k.transpose(1, 2) * scale
            p = torch.softmax(z, -1)
            expect, A = p @ v, p @ v.abs()
            mag = (qq.abs() @ k.abs().transpose(1, 2) * abs(scale)).amax(-1, keepdim=True)
            score = D * FP32 * mag + 2 * FP32 * z.abs().amax(-1, keepdim=True) + 2.0 ** -21
            bound = HALF * expect.abs() + A * (HALF + 2 * score * 1.01 + ((hi - lo) / 8 + 600) * FP32 * 2)
            err = (out[b, t].double().view_as(expect) - expect).abs()
            assert torch.isfinite(err).all()
            worst = max(worst, float((err / bound.clamp(min=1e-30)).max()))
    assert worst <= 1.0, worst


@pytest.mark.parametrize("B,Tq,Hq,Hkv,D,cap", [(1, 1, 32, 8, 128, 1168), (2, 1, 8, 2, 128, 1504), (1, 2, 4, 2, 64, 304), (3, 1, 16, 8, 128, 9008),
                                               (2, 3, 8, 8, 128, 2208), (1, 2, 32, 2, 128, 640), (4, 1, 6, 2, 64, 144), (2, 1, 40, 1, 128, 400),
                                               (1, 1, 34, 2, 64, 96), (40, 1, 4, 2, 128, 80), (70, 2, 2, 1, 64, 48), (1, 1, 9, 1, 128, 70000)])
def test_attention(B, Tq, Hq, Hkv, D, cap):
    cache = _cache(B, Hkv, cap, D, seed=cap)
    q = _randn(B, Tq, Hq, D, seed=1)
    g = _gen(2)
    start = torch.randint(0, max(1, cap // 4), (B, Tq), device=DEV, generator=g, dtype=torch.int32)
    length = torch.randint(1, cap, (B, Tq), device=DEV, generator=g, dtype=torch.int32)
    out = ops.int4_decode_attention(q, cache, start, length)
    _lib.check_status()
    _check_attention(out, q, cache, start, length, D ** -0.5)
    for scale in (0.25, -0.1):
        _check_attention(ops.int4_decode_attention(q, cache, start, length, scale), q, cache, start, length, scale)


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (4, 2, 64), (32, 2, 128)])
def test_attention_of_odd_slices(Hq, Hkv, D):
    """Slices of no slot, of one, across tile ends, past the cache, before it, and of the whole cache, in one batch."""
    cap = 272
    spans = [(0, 0), (0, 1), (271, 1), (271, 50), (15, 2), (16, 16), (17, 31), (31, 33), (100, -5), (-4, 6), (-4, 4), (0, 272), (0, 2 ** 31 - 1),
             (300, 5), (2 ** 31 - 1, 2 ** 31 - 1), (-2 ** 31, 2 ** 31 - 1), (1, 271), (129, 128), (5, 64), (255, 17), (-2 ** 31, -2 ** 31)]
    B = len(spans)
    cache = _cache(B, Hkv, cap, D, seed=9)
    q = _randn(B, 1, Hq, D, seed=3)
    start = torch.tensor([s for s, _ in spans], device=DEV, dtype=torch.int32).view(B, 1)
    length = torch.tensor([n for _, n in spans], device=DEV, dtype=torch.int32).view(B, 1)
    _check_attention(ops.int4_decode_attention(q, cache, start, length), q, cache, start, length, D ** -0.5)
    one = ops.int4_decode_attention(q.view(1, B, Hq, D), cache.rows(slice(11, 12)), start.view(1, B), length.view(1, B))      # one sequence, many queries
    _check_attention(one, q.view(1, B, Hq, D), cache.rows(slice(11, 12)), start.view(1, B), length.view(1, B), D ** -0.5)
    zero = torch.zeros_like(length)
    assert (ops.int4_decode_attention(q, cache, start, zero) == 0).all()


@pytest.mark.parametrize("D", [64, 128])
def test_nothing_outside_a_slice_enters_a_result(D):
    B, Hq, Hkv, cap = 3, 8, 2, 208
    cache = _cache(B, Hkv, cap, D, seed=5)
    q = _randn(B, 2, Hq, D, seed=6)
    start = torch.tensor([[3, 90], [40, 0], [64, 97]], device=DEV, dtype=torch.int32)
    length = torch.tensor([[80, 30], [1, 35], [33, 100]], device=DEV, dtype=torch.int32)
    expect = ops.int4_decode_attention(q, cache, start, length)
    _check_attention(expect, q, cache, start, length, D ** -0.5)
    for t in range(2):                  # all that one query does not see is poisoned, also what the other one sees
        bad = ops.Int4Cache(*(x.clone() for x in cache))
        for b in range(B):
            seen = torch.zeros(cap, dtype=torch.bool, device=DEV)
            seen[start[b, t]:start[b, t] + length[b, t]] = True
            bad.k_scale[b, :, ~seen], bad.v_scale[b, :, ~seen] = float("nan"), float("inf")
            bad.k[b, :, ~seen] = 0xFF
        assert torch.equal(ops.int4_decode_attention(q, bad, start, length)[:, t], expect[:, t])
    cache.v_scale[1, 0, 40] = float("nan")                                 # inside: it shows
    out = ops.int4_decode_attention(q, cache, start, length)
    assert out[1, 0, :4].isnan().all() and out[1, 0, 4:].isfinite().all() and out[0].isfinite().all()


def test_attention_reads_strided_queries():
    B, Hq, Hkv, D, cap = 3, 8, 2, 128, 160
    cache = _cache(B, Hkv, cap, D, seed=7)
    rows = _randn(B, 2, (Hq + 2 * Hkv) * D, seed=8)
    q = rows[:, :, :Hq * D].view(B, 2, Hq, D)
    start = torch.randint(0, 20, (B, 2), device=DEV, generator=_gen(1))    # int64
    length = torch.randint(1, 140, (2, B), device=DEV, generator=_gen(2), dtype=torch.int32).t()
    expect = ops.int4_decode_attention(q.clone(), cache, start, length)
    _check_attention(expect, q, cache, start, length, D ** -0.5)
    assert torch.equal(ops.int4_decode_attention(q, cache, start, length), expect)
    assert torch.equal(ops.int4_decode_attention(q.transpose(2, 3).contiguous().transpose(2, 3), cache, start, length), expect)
    odd = torch.empty(q.numel() + 1, device=DEV, dtype=torch.bfloat16)[1:].view(q.shape).copy_(q)
    assert torch.equal(ops.int4_decode_attention(odd, cache, start, length), expect)
    same = ops.int4_decode_attention(q[:, :1].expand(B, 2, Hq, D), cache, start[:, :1].expand(B, 2), length[:, :1].expand(B, 2))
    assert torch.equal(same[:, 0], same[:, 1]) and torch.equal(same[:, 0], expect[:, 0])


def test_attention_past_32_bits():
    """A cache whose last head starts past 2^32 bytes of codes."""
    H, D, cap = 8, 128, 1 << 23
    cache = ops.int4_cache(1, H, cap, D, DEV)
    n = 5000
    part = _cache(1, H, 5008, D, seed=11)
    for whole, some in zip(cache, part):
        whole[:, :, cap - 5008:] = some
    q = _randn(1, 1, 16, D, seed=12)
    start = torch.tensor([[cap - n]], device=DEV, dtype=torch.int32)
    length = torch.tensor([[n]], device=DEV, dtype=torch.int32)
    out = ops.int4_decode_attention(q, cache, start, length)
    assert torch.equal(out, ops.int4_decode_attention(q, part, start - (cap - 5008), length))
    k, v = _randn(1, 3, H, D, seed=13), _randn(1, 3, H, D, seed=14)
    slots = torch.tensor([[cap - 1, cap, cap - 3]], device=DEV)
    ops.int4_cache_write(cache, k, v, slots)
    kr, _ = ops.int4_cache_read(cache, torch.tensor([cap - 2], device=DEV), 3)
    want = ref.int4_values(*ref.int4_quantize(k, 32))
    assert torch.equal(kr[0, :, 1], want[0, 0]) and (kr[0, :, 2] == 0).all()


def test_two_streams_and_two_graphs_at_once():
    """Calls in flight beside one another and replayed graphs share nothing; a replay sees new rows, slices and queries."""
    B, Hq, Hkv, D, cap = 2, 8, 2, 128, 3008
    caches = [_cache(B, Hkv, cap, D, seed=20 + i) for i in range(2)]
    qs = [_randn(B, 1, Hq, D, seed=30 + i) for i in range(2)]
    start = torch.zeros(B, 1, device=DEV, dtype=torch.int32)
    lens = [torch.tensor([[3000], [17]], device=DEV, dtype=torch.int32), torch.tensor([[900], [2500]], device=DEV, dtype=torch.int32)]
    w = ops.int4_quantize_weight(_randn(256, Hq * D, seed=40))
    rows = [_randn(B, 1, 2 * Hkv, D, seed=50 + i) for i in range(2)]
    slots = [n.clone() - 1 for n in lens]

    def step(i):
        ops.int4_cache_write(caches[i], rows[i][:, :, :Hkv], rows[i][:, :, Hkv:], slots[i])
        att = ops.int4_decode_attention(qs[i], caches[i], start, lens[i])
        return att, ops.int4_linear(att.view(B, Hq * D), w)
    alone = [step(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(step(i))
        torch.cuda.synchronize()
        for a, b in zip(got, alone):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(i))
        graphs.append(g)
    for _ in range(5):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, alone):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    lens[0].copy_(torch.tensor([[1], [2000]]))
    slots[0].copy_(lens[0] - 1)
    qs[0].copy_(_randn(B, 1, Hq, D, seed=60))
    rows[0].copy_(_randn(B, 1, 2 * Hkv, D, seed=61))
    graphs[0].replay()
    torch.cuda.synchronize()
    again = step(0)
    assert torch.equal(outs[0][0], again[0]) and torch.equal(outs[0][1], again[1])
    _check_attention(again[0], qs[0], caches[0], start, lens[0], D ** -0.5)


# ------------------------------------------------------------------------------------------------- products
def _check_linear(y, x, w):
    """Against 64 bits: the result is rounded to bf16; fp32 sums of exact products add FP32 of sum |x w| for each matrix instruction of a
    chain (K / 16 at most) and for each of the sums that meet at the end (64 at most)."""
    wd = ops.int4_dequantize_weight(w).double()
    K = wd.shape[1]
    x = x.reshape(-1, K).double()
    expect, mag = x @ wd.t(), x.abs() @ wd.abs().t()
    bound = HALF * expect.abs() + (K / 16 + 64) * FP32 * mag + 1e-30
    assert ((y.reshape(expect.shape).double() - expect).abs() <= bound).all()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("N,K", [(1, 128), (3, 256), (148, 384), (777, 1280), (2560, 9728), (6145, 640), (20001, 512)])
def test_linear(N, K, group):
    w = ops.int4_quantize_weight((_randn(N, K, seed=N) * 0.05).bfloat16(), group)
    for M in (1, 2, 7, 8, 9, 16, 17, 40):
        x = _randn(M, K, seed=M)
        _check_linear(ops.int4_linear(x, w), x, w)
    _lib.check_status()


@pytest.mark.parametrize("N,K", [(5, 32), (300, 96), (1000, 160), (64, 2080)])
def test_linear_with_a_last_segment_that_is_not_whole(N, K):
    w = ops.int4_quantize_weight(_randn(N, K, seed=N), 32)
    for M in (1, 8, 13):
        x = _randn(M, K, seed=M)
        _check_linear(ops.int4_linear(x, w), x, w)


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("F,K", [(1, 128), (5, 256), (150, 384), (4864, 256), (9728, 128), (333, 1152)])
def test_linear_swiglu(F, K, group):
    """Against 64 bits: gate and up are as `_check_linear` has them, rounded to bf16; silu has a slope of at most 1.1, and the result is
    rounded once more, with 2^-20 for the fp32 exponential, division and products."""
    w = ops.int4_quantize_weight((_randn(2 * F, K, seed=F) * 0.1).bfloat16(), group)
    wd = ops.int4_dequantize_weight(w).double()
    for M in (1, 8, 11, 16, 19):
        x = _randn(M, K, seed=M)
        y, mag = x.double() @ wd.t(), x.double().abs() @ wd.abs().t()
        err = HALF * y.abs() * 1.01 + (K / 16 + 64) * FP32 * mag
        gate, up, dg, du = y[:, :F], y[:, F:], err[:, :F], err[:, F:]
        expect = torch.nn.functional.silu(gate) * up
        bound = 1.1 * dg * (up.abs() + du) + torch.nn.functional.silu(gate).abs() * du + (HALF + 2.0 ** -20) * (expect.abs() + dg * up.abs()) * 1.01 + 1e-30
        assert ((ops.int4_linear_swiglu(x, w).double() - expect).abs() <= bound).all()
    _lib.check_status()


@pytest.mark.parametrize("N,K", [(5, 160), (777, 1280), (2500, 2304), (33001, 2080)])
def test_linear_in_blocks_and_with_values(N, K):
    """Rows on both sides of the rules: up to 32 in one launch, more in blocks of 32 or with the values written out, and the same bits each time."""
    w = ops.int4_quantize_weight((_randn(N, K, seed=N) * 0.05).bfloat16(), 32)
    for M in (9, 16, 17, 32, 33, 65, 80, 129):
        x = _randn(M, K + 8, seed=M)[:, :K]
        y = ops.int4_linear(x, w)
        _check_linear(y, x, w)
        assert torch.equal(y, ops.int4_linear(x, w))
    _lib.check_status()


def test_linear_rows_of_any_layout():
    N, K = 200, 256
    w = ops.int4_quantize_weight(_randn(N, K, seed=1))
    for x in (_randn(4, 3 * K, seed=2)[:, K:2 * K], _randn(K, 5, seed=3).t(), _randn(2, 3, K, seed=4), _randn(6 * K + 1, seed=5)[1:].view(6, K),
              _randn(1, K, seed=6).expand(7, K), _randn(1, K, seed=6).expand(30, K), _randn(K, seed=7)):
        y = ops.int4_linear(x, w)
        assert y.shape == (*x.shape[:-1], N)
        _check_linear(y, x, w)
    assert ops.int4_linear(_randn(0, K), w).shape == (0, N)
    w = ops.int4_quantize_weight(_randn(3000, 1536, seed=8))               # more than 16 rows of it go in one launch
    for x in (_randn(20, 2000, seed=2)[:, 64:1600], _randn(1536, 17, seed=3).t(), _randn(2, 3, 4, 1536, seed=4), _randn(1, 1536, seed=6).expand(30, 1536),
              _randn(24 * 768 + 1536, seed=9).as_strided((24, 1536), (768, 1))):
        y = ops.int4_linear(x, w)
        assert y.shape == (*x.shape[:-1], 3000)
        _check_linear(y, x, w)


def test_chains_of_clusters_on_two_streams_and_in_graphs():
    """Products whose CTAs share K and hold all tensor memory, one after the other (each reads what the one before wrote), between bf16
    products, beside the same on another stream, and replayed."""
    n = 2304                            # more than 2 ** 22 values: 24 rows go in one launch
    ws = [ops.int4_quantize_weight((_randn(n, n, seed=i) * 0.03).bfloat16()) for i in range(3)]
    plain = (_randn(n, n, seed=9) * 0.03).bfloat16()
    xs = [_randn(24, n, seed=20 + i) for i in range(2)]

    def chain(x):
        with torch.no_grad():
            for w in ws:
                x = ops.linear(ops.int4_linear(ops.int4_linear(x, w), w), plain)
            return x
    alone = [chain(x) for x in xs]
    torch.cuda.synchronize()
    one = ops.int4_linear(xs[0], ws[0])
    _check_linear(one, xs[0], ws[0])
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        got = []
        for x, s in zip(xs, streams):
            with torch.cuda.stream(s):
                got.append(chain(x))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, alone))
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(chain(x))
        graphs.append(g)
    for _ in range(5):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, alone))
    xs[0].copy_(_randn(24, n, seed=30))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], chain(xs[0]))
    _lib.check_status()


@pytest.mark.parametrize("group", [32, 64, 128])
def test_weights_are_the_plain_form_to_the_bit(group):
    w = _randn(101, 384, seed=group)
    w[3, 5], w[4, 200] = float("nan"), 3e38
    for x in (w, _randn(101, 800, seed=2)[:, 400:784], w.t().contiguous().t()):
        got = ops.int4_quantize_weight(x, group)
        codes, scale = ref.int4_quantize(x, group)
        assert torch.equal(got.codes, codes)
        _same(got.scale[:, :101].transpose(0, 1).float(), scale.float())
        assert (got.scale[:, 101:] == 0).all()
        _same(ops.int4_dequantize_weight(got).float(), ref.int4_values(codes, scale).float())


@pytest.mark.parametrize("M", [1, 3, 4, 5])
@pytest.mark.parametrize("N,K,group", [(6, 32, 32), (777 * 2, 160, 32), (6144, 2560, 64), (2560, 4096, 128), (39000, 256, 64), (40, 32768, 128)])
@pytest.mark.parametrize("glu", [False, True])
def test_norm_ahead_of_the_product(M, N, K, group, glu):
    """Against the product of the norm's own rounding in 64 bits: a value of the norm is off by one rounding to bf16 and 2^-20 of fp32 (a sum of K
    squares in parts, a root, two products), which the product sees as that share of its terms' magnitudes."""
    w = ops.int4_quantize_weight((_randn(N, K, seed=N) * 0.1).bfloat16(), group)
    wd = ops.int4_dequantize_weight(w).double()
    wide = _randn(M, K + 8, seed=1)
    norm_w = (1 + _randn(K, seed=2) * 0.2).bfloat16()
    for n in (None, M, M // 2):
        x, delta = wide[:, :K], None if n is None else _randn(n, K, seed=3)
        res, y = ops.int4_norm_linear(x, delta, norm_w, 1e-6, w, glu)
        expect = x.clone()
        if n is not None:
            expect[:n] = (x[:n].float() + delta.float()).bfloat16()
        assert torch.equal(res, expect)
        r = expect.double()
        h = r * (r.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * norm_w.double()
        p, mag = h @ wd.t(), h.abs() @ wd.abs().t()
        err = (HALF + 2.0 ** -20) * 1.01 * mag + HALF * p.abs() * 1.01 + (K / 16 + 64) * FP32 * mag * 1.01
        if not glu:
            assert ((y.double() - p).abs() <= err + 1e-30).all()
            continue
        F = N // 2
        gate, up, dg, du = p[:, :F], p[:, F:], err[:, :F], err[:, F:]
        z = torch.nn.functional.silu(gate) * up
        bound = 1.1 * dg * (up.abs() + du) + torch.nn.functional.silu(gate).abs() * du + (HALF + 2.0 ** -20) * (z.abs() + 1.1 * dg * up.abs()) * 1.01 + 1e-30
        assert ((y.double() - z).abs() <= bound).all()
    _lib.check_status()


def test_a_weight_without_rows():
    w = ops.int4_quantize_weight(_randn(0, 256))
    for M in (0, 1, 20, 40, 200):
        assert ops.int4_linear(_randn(M, 256), w).shape == (M, 0) and ops.int4_linear_swiglu(_randn(M, 256), w).shape == (M, 0)
    assert ops.int4_dequantize_weight(w).shape == (0, 256)


def test_refusals_on_the_device():
    cache, rows, none = _cache(2, 2, 32, 128, seed=1), _randn(2, 8 * 128), torch.zeros(2, device=DEV, dtype=torch.int32)
    for w in (torch.ones(128, device=DEV), torch.ones(64, device=DEV).bfloat16(), torch.ones(128).bfloat16(), _randn(256)[::2]):
        with pytest.raises(ValueError):
            ops.int4_qk_norm_rope_decode(rows, w, None, none, 4, 1e4, 1e-6, False, cache, none)
    with pytest.raises(ValueError):
        ops.int4_qk_norm_rope_decode(rows, None, None, none[:1], 4, 1e4, 1e-6, False, cache, none)
    w, x, one = ops.int4_quantize_weight(_randn(8, 64)), _randn(2, 64), torch.ones(64, device=DEV).bfloat16()
    for bad in ((x[:, :32], None, one), (x, _randn(3, 64), one), (x, _randn(2, 32), one), (x, None, one[:32]), (x, None, one.cpu())):
        with pytest.raises(ValueError):
            ops.int4_norm_linear(*bad, 1e-6, w)
    cache = _cache(1, 2, 32, 96, seed=1)
    q, one = _randn(1, 1, 4, 96), torch.ones(1, 1, device=DEV, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.int4_decode_attention(q, cache, one, one)                      # head dim 96
    cache = _cache(1, 2, 32, 64, seed=1)
    with pytest.raises(TypeError):
        ops.int4_decode_attention(_randn(1, 1, 4, 64).float(), cache, one, one)
    with pytest.raises(ValueError):
        ops.int4_decode_attention(_randn(1, 1, 4, 64), cache, one.cpu(), one)
    with pytest.raises(TypeError):
        ops.int4_cache_write(cache, torch.zeros(1, 1, 2, 64, device=DEV), torch.zeros(1, 1, 2, 64, device=DEV), one)
    with pytest.raises(TypeError):
        ops.int4_linear(torch.zeros(1, 128, device=DEV), ops.int4_quantize_weight(_randn(8, 128)))
    with pytest.raises(ValueError):
        ops.int4_linear(torch.zeros(1, 128), ops.int4_quantize_weight(_randn(8, 128)))
