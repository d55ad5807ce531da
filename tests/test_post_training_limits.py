"""Where a post-training step is refused or takes another path."""
from types import SimpleNamespace

import pytest
import torch

from ksa_b200.parallel import fsdp
from ksa_b200.training.engine import TrainEngine
from test_post_training import _batch, _model


def test_log_probs_of_a_shard_of_the_sequence_are_refused():
    """Under context parallelism a rank has parts of answers, and a loss of those is another loss."""
    model = _model("cpu")
    tokens, labels = _batch("cpu")
    model.cp = SimpleNamespace()
    with pytest.raises(ValueError, match="shard"):
        model(tokens, labels=labels, log_probs=True)


def test_log_probs_of_the_last_token_alone_are_refused():
    """Its logits would come back in their place."""
    model = _model("cpu")
    tokens, labels = _batch("cpu")
    with pytest.raises(ValueError, match="log_probs"):
        model(tokens, labels=labels, log_probs=True, last_token_only=True)


@pytest.mark.parametrize("clip_norm,comm,want", [(0.0, None, "fused"), (1.0, None, "collective"), (1.0, "collective", "collective"), (0.0, "collective", "collective")])
def test_clipping_by_the_norm_takes_the_back_end_that_has_it(clip_norm, comm, want, monkeypatch):
    """On the GPUs of one node, without a back end asked for."""
    class Reached(Exception):
        pass

    def stop(*args, **kw):
        raise Reached
    monkeypatch.setattr(TrainEngine, "__init__", stop)
    engine = fsdp.FsdpEngine.__new__(fsdp.FsdpEngine)
    with pytest.raises(Reached):
        engine.__init__(torch.nn.Linear(2, 2), device=torch.device("cuda"), world_size=2, rank=0, comm=comm, clip_norm=clip_norm)
    assert engine.comm == want
