"""The inference engine with its cache and its weights in four bits: against an engine whose ordinary cache holds the very values that the
quantised one stands for, and against one whose model has the values of the quantised weights."""
import copy

import pytest
import torch

from ksa_b200 import ops
from ksa_b200.config import get_preset
from ksa_b200.inference import Int4LayerCache, KsaInferenceEngine
from ksa_b200.inference import engine as engine_module
from ksa_b200.inference.engine import _Int4Layer
from ksa_b200.models import get_model_class
from ksa_b200.ops import reference as ref

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _model(device, chunk=16, window=2, n_sum=1):
    head = 128 if device == "cuda" else 64
    cfg = get_preset("qwen3-ksa-tiny").merge({
        "num_layers": 4, "summary_layer_freq": [1, 1, 0, 1], "embed_dim": 256, "intermediate_dim": 512, "vocab_size": 512, "head_dim": head,
        "num_heads": 4, "num_kv_heads": 2, "summary_chunk_size": chunk, "summary_token_num": n_sum, "summary_sliding_chunk_num": window})
    torch.manual_seed(0)
    m = get_model_class(cfg.model_class)(cfg)
    m.init_weights(seed=0)
    with torch.no_grad():
        for p in m.parameters():
            if p.dim() >= 2:
                p.mul_(2.0)
    return m.eval() if device == "cpu" else m.cuda().to(torch.bfloat16).eval()


def _round_trip(x):
    return ref.int4_values(*ref.int4_quantize(x, 32)).to(x.dtype)


def _slices(q, k, v, start, length, scale, counters=None):
    """Attention over an ordinary cache in the steps of the plain form of four bits: in fp32 a sum in another order would now and then
    put a key of the next step on the other side of the middle between two codes."""
    out = torch.zeros_like(q)
    for b in range(q.shape[0]):
        for t in range(q.shape[1]):
            lo, n = int(start[b, t]), int(length[b, t])
            if n > 0:
                kf, vf = (x[b, :, lo:lo + n].bfloat16().float() for x in (k, v))
                p = torch.softmax(q[b, t].view(kf.shape[0], -1, q.shape[3]) @ kf.transpose(1, 2) * scale, -1)
                out[b, t] = (p @ vf).reshape(q.shape[2:])
    return out


def _values_in_the_cache(monkeypatch, eng):
    """From here on every row that ``eng`` writes into its ordinary caches is what four bits would make of it."""
    if eng.layer_caches[0].k.device.type == "cpu":
        monkeypatch.setattr(engine_module, "_decode_attention", _slices)
    decode, append, move = ops.qk_norm_rope_decode, engine_module._cache_append, engine_module._cache_move

    def rounded(*a):
        if len(a) > 10 and a[10] is not None and any(a[10] is c.k for c in eng.layer_caches if hasattr(c, "k")):
            k_cache, v_cache, slots = a[10], a[11], a[12].reshape(-1).tolist()
            out = decode(*a)
            for b, s in enumerate(slots):
                if s >= 0:
                    k_cache[b, :, s], v_cache[b, :, s] = _round_trip(k_cache[b, :, s]), _round_trip(v_cache[b, :, s])
            return out
        return decode(*a)
    monkeypatch.setattr(ops, "qk_norm_rope_decode", rounded)
    monkeypatch.setattr(engine_module, "_cache_append", lambda k, v, *rest: append(_round_trip(k), _round_trip(v), *rest))
    for c in eng.layer_caches:
        c.k.copy_(_round_trip(c.k))
        c.v.copy_(_round_trip(c.v))


def _relative(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("chunk,window,n_sum,lengths", [(16, 2, 1, [37, 37, 37]), (16, 3, 2, [50, 16, 50]), (8, 1, 1, [5, 31, 64]), (16, 0, 1, [40, 40, 33])])
def test_cache_in_four_bits(monkeypatch, device, chunk, window, n_sum, lengths):
    """Prompts of unequal length (groups of sequences that are not neighbours), chunk ends of some or all sequences, growing caches."""
    model = _model(device, chunk, window, n_sum)
    B, new = len(lengths), 2 * chunk + 5
    torch.manual_seed(3)
    prompt = torch.randint(0, 500, (B, max(lengths)), device=device)
    plain = KsaInferenceEngine(model, max_len=256, batch=B, cuda_graph=False)
    eng = KsaInferenceEngine(model, max_len=max(lengths) + 4, batch=B, kv_cache="int4")
    assert all(isinstance(c, Int4LayerCache) for c in eng.layer_caches)
    a, b = plain.prefill(prompt, lengths=lengths), eng.prefill(prompt, lengths=lengths)
    assert torch.equal(a, b)                     # the prompt's own attention is unchanged
    _values_in_the_cache(monkeypatch, plain)
    for c, q in zip(plain.layer_caches, eng.layer_caches):      # what the prompt left is there, value by value
        k, v = ops.int4_cache_read(q.data, torch.zeros(B, dtype=torch.int32, device=device), q.data.capacity)
        n = min(k.shape[2], c.k.shape[2])
        spec = q.spec
        for i, l in enumerate(lengths):
            if spec is None:
                used = torch.arange(l)
            else:
                full = l // chunk
                used = torch.cat([torch.arange(spec.text0, spec.text0 + min(full, window) * chunk), torch.arange(spec.sum0, spec.sum0 + full * n_sum),
                                  spec.n_sum + chunk - 1 - torch.arange(l - full * chunk)])
            assert torch.equal(k[i][:, used].to(c.k.dtype), c.k[i][:, used]) and torch.equal(v[i][:, used].to(c.v.dtype), c.v[i][:, used])
    # fp32: the sums' order; bf16: the bound that two engines in bf16 are held to elsewhere
    bound = 2e-3 if device == "cpu" else 5e-2
    for step in range(new):
        nxt = a.argmax(-1)
        a, b = plain.decode_step(nxt), eng.decode_step(nxt)
        assert _relative(b, a) < bound, (step, _relative(b, a))
    assert eng.max_len > max(lengths) + 4 and eng.cache_bytes() < plain.cache_bytes()
    again = eng.prefill(prompt[:, :lengths[0]])  # a second request on the same engine
    assert torch.equal(again, plain.prefill(prompt[:, :lengths[0]]))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("B", [1, 3, 20])
def test_weights_in_four_bits(device, B):
    model = _model(device)
    values = copy.deepcopy(model)
    with torch.no_grad():
        for layer in values.layers:
            for lin in (layer.attn.wqkv, layer.attn.wqkv_summary, layer.attn.output_proj, layer.mlp.w13, layer.mlp.w2):
                if lin is not None:
                    lin.weight.copy_(ops.int4_dequantize_weight(ops.int4_quantize_weight(lin.weight, 32)))
    head = ops.int4_quantize_weight(model.lm_head_weight, 32)
    with torch.no_grad():
        values.lm_head_weight.copy_(ops.int4_dequantize_weight(head))
    torch.manual_seed(3)
    prompt = torch.randint(0, 500, (B, 30), device=device)
    plain = KsaInferenceEngine(values, max_len=128, batch=B)
    eng = KsaInferenceEngine(values, max_len=128, batch=B, weights="int4", weight_group=32)
    eng._int4, eng._int4_head = [_Int4Layer(layer, 32) for layer in model.layers], head      # of the weights that the values come from
    a, b = plain.prefill(prompt), eng.prefill(prompt)
    bound = 1e-4 if device == "cpu" else 5e-2
    for step in range(22):
        nxt = a.argmax(-1)
        a, b = plain.decode_step(nxt), eng.decode_step(nxt)
        assert _relative(b, a) < bound, (step, _relative(b, a))


@pytest.mark.parametrize("device", DEVICES)
def test_both_together_generate(device):
    """Graphs and eager steps of an engine with both give the same tokens; nothing of a model in four bits is far from the model."""
    model = _model(device)
    torch.manual_seed(5)
    prompt = torch.randint(0, 500, (2, 41), device=device)
    kw = dict(max_len=160, batch=2, kv_cache="int4", weights="int4")
    one = KsaInferenceEngine(model, **kw).generate(prompt, 40)
    two = KsaInferenceEngine(model, cuda_graph=False, **kw).generate(prompt, 40)
    assert torch.equal(one, two) and one.shape == (2, 81)


def test_refusals():
    model = _model("cpu")
    with pytest.raises(ValueError):
        KsaInferenceEngine(model, 64, 1, kv_cache="fp8")
    with pytest.raises(ValueError):
        KsaInferenceEngine(model, 64, 1, weights="int8")
    model.tp = object()
    with pytest.raises(ValueError):
        KsaInferenceEngine(model, 64, 1, weights="int4")


@pytest.mark.parametrize("device", DEVICES)
def test_moving_rows(device):
    cache = ops.int4_cache(3, 2, 64, 64, device)
    rows = torch.randn(3, 64, 2, 64, device=device).bfloat16()
    ops.int4_cache_write(cache, rows, rows.flip(1), torch.arange(64, device=device).repeat(3, 1))
    want = [t.clone() for t in cache]
    src, dst, on = torch.tensor([3, 40, 0]), torch.tensor([20, 61, 32]), torch.tensor([1, 1, 0])
    for t in want:
        t[0, :, 20:30] = t[0, :, 3:13].clone()
        t[1, :, 61:64] = t[1, :, 40:43].clone()              # the rest would lie past the cache
    ops.int4_cache_move(cache, src.to(device), dst.to(device), on.to(device), 10)
    assert all(torch.equal(a, b) for a, b in zip(cache, want))
    with pytest.raises(ValueError):
        ops.int4_cache_move(cache, src.to(device), dst.to(device), on[:2].to(device), 10)
