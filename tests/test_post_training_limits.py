"""Where a post-training step is refused or takes another path."""
from types import SimpleNamespace

import pytest

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
