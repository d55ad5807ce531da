"""Decode steps of an engine with weights in four bits read nothing but the codes: ordinary steps and those that close a chunk, few and
more sequences, the output head included."""
import copy

import pytest
import torch

from ksa_b200 import ops
from ksa_b200.config import get_preset
from ksa_b200.inference import KsaInferenceEngine
from ksa_b200.inference.cache import cache_tensors
from ksa_b200.models import get_model_class

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _model(device, own_summary):
    cfg = get_preset("qwen3-ksa-tiny").merge({
        "num_layers": 4, "summary_layer_freq": [1, 1, 0, 1], "embed_dim": 256, "intermediate_dim": 512, "vocab_size": 512,
        "head_dim": 128 if device == "cuda" else 64, "num_heads": 4, "num_kv_heads": 2, "summary_chunk_size": 16, "summary_token_num": 1,
        "summary_sliding_chunk_num": 2, "summary_token_begin": 505, "summary_independent_parameters": own_summary})
    model = get_model_class(cfg.model_class)(cfg)
    model.init_weights(seed=0)
    with torch.no_grad():
        for p in model.parameters():
            if p.dim() >= 2:
                p.mul_(2.0)
    return model.eval() if device == "cpu" else model.cuda().to(torch.bfloat16).eval()


def _products(model):
    """The weights that an engine holds in four bits."""
    out = [model.lm_head_weight]
    for layer in model.layers:
        out += [lin.weight for lin in (layer.attn.wqkv, layer.attn.wqkv_summary, layer.attn.output_proj, layer.mlp.w13, layer.mlp.w2) if lin is not None]
    return out


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("B", [1, 4, 5, 20])
@pytest.mark.parametrize("own_summary", [False, True])
def test_steps_read_the_codes_alone(device, B, own_summary):
    """Against an ordinary engine on a model of the codes' values.  Both begin with what that engine's prompt has left, and the bf16 weights of the engine
    under test are not numbers once it is made."""
    model = _model(device, own_summary)
    assert model.output is not None and (model.layers[0].attn.wqkv_summary is not None) == own_summary
    values = copy.deepcopy(model)
    with torch.no_grad():
        for p in _products(values):
            p.copy_(ops.int4_dequantize_weight(ops.int4_quantize_weight(p.detach(), 32)))
    plain = KsaInferenceEngine(values, max_len=128, batch=B)
    eng = KsaInferenceEngine(model, max_len=128, batch=B, weights="int4", weight_group=32)
    torch.manual_seed(3)
    prompt = torch.randint(0, 500, (B, 30), device=device)
    logits = plain.prefill(prompt)
    eng.prefill(prompt)                         # its counters
    for to, was in zip(eng.layer_caches, plain.layer_caches):
        for a, b in zip(cache_tensors(to), cache_tensors(was)):
            a.copy_(b)
    with torch.no_grad():
        for p in _products(model):
            p.fill_(float("nan"))
    # fp32: the sums' order; bf16: the bound that two engines in bf16 are held to elsewhere
    bound = 1e-4 if device == "cpu" else 5e-2
    for step in range(22):                      # chunks end at 32 and 48
        token = logits.argmax(-1)
        logits, got = plain.decode_step(token), eng.decode_step(token)
        off = float((got.float() - logits.float()).norm() / logits.float().norm())
        assert off < bound, (step, off)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("head", [32, 96])
def test_head_dims_are_refused_when_the_engine_is_made(device, head):
    """A cache of such heads can be written; its attention (on a GPU) and its moves cannot, and the first step or closed chunk would say so."""
    cfg = get_preset("qwen3-ksa-tiny").merge({"num_layers": 2, "summary_layer_freq": [1, 0], "embed_dim": 64, "intermediate_dim": 128, "vocab_size": 512,
                                              "head_dim": head, "num_heads": 2, "num_kv_heads": 1, "summary_chunk_size": 8, "summary_token_begin": 505})
    model = get_model_class(cfg.model_class)(cfg).eval().to(device)
    with pytest.raises(ValueError):
        KsaInferenceEngine(model, 64, 1, kv_cache="int4")
