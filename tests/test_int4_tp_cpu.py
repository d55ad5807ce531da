"""The cache in four bits under tensor parallelism, on CPU ranks (gloo): every rank holds its heads' cache, and prompts, steps, closed chunks
and growing caches give what the unsharded engine with such a cache gives."""
import os
import socket

import numpy as np
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from ksa_b200.config import get_preset
from ksa_b200.models import get_model_class


def _free_port() -> int:
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _cfg():
    return get_preset("qwen3-ksa-tiny").merge({
        "num_layers": 3, "summary_layer_freq": [1, 0, 1], "embed_dim": 64, "intermediate_dim": 128, "vocab_size": 256,
        "head_dim": 64, "num_heads": 4, "num_kv_heads": 2, "summary_chunk_size": 8, "summary_sliding_chunk_num": 2,
        "summary_token_num": 1, "summary_token_begin": 200})


def _full_model(cfg):
    torch.manual_seed(0)
    model = get_model_class(cfg.model_class)(cfg)
    model.init_weights(seed=0)
    return model.float()


def _logits(model, tokens, heads):
    """Prompt and steps with given tokens; the cache has ``heads`` key heads."""
    from ksa_b200.inference import Int4LayerCache, KsaInferenceEngine
    eng = KsaInferenceEngine(model, max_len=24, batch=2, kv_cache="int4")
    assert all(isinstance(c, Int4LayerCache) and c.data.k.shape[1] == heads for c in eng.layer_caches)
    outs = [eng.prefill(tokens[:, :21])]
    outs += [eng.decode_step(tokens[:, t]) for t in range(21, 40)]
    assert eng.max_len > 24
    return torch.stack(outs)


def _worker(rank, world, port, out_q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        from ksa_b200.parallel.tp import TpContext, build_tp_model
        cfg = _cfg()
        tp = TpContext(dist.group.WORLD, cfg.embed_dim, max_rows=256)
        model = build_tp_model(_full_model(cfg).state_dict(), cfg, tp)
        out_q.put((rank, _logits(model, _tokens(), cfg.num_kv_heads // world).numpy()))
    finally:
        dist.destroy_process_group()


def _tokens():
    return torch.randint(0, 200, (2, 40), generator=torch.Generator().manual_seed(5))


def test_sharded_cache_in_four_bits_matches_the_whole_one():
    world = 2
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = _free_port()
    ps = [ctx.Process(target=_worker, args=(r, world, port, q)) for r in range(world)]
    for p in ps:
        p.start()
    got = dict(q.get(timeout=120) for _ in ps)
    for p in ps:
        p.join(60)
        assert p.exitcode == 0
    expect = _logits(_full_model(_cfg()), _tokens(), 2).numpy()
    for rank in range(world):
        assert got[rank].shape == expect.shape
        # fp32: the sums' order, and a key now and then on the other side of the middle between two codes
        assert np.linalg.norm(got[rank] - expect) < 2e-3 * np.linalg.norm(expect)
