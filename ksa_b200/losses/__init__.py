from .ce import CrossEntropyLoss
from .distill import attention_cosine_loss, attention_mse_loss, kl_divergence_loss
from .chunked import ChunkedDistillLossComputer
from .post_training import PolicyLoss, PreferenceLoss

__all__ = ["CrossEntropyLoss", "attention_mse_loss", "attention_cosine_loss", "kl_divergence_loss",
           "ChunkedDistillLossComputer", "PolicyLoss", "PreferenceLoss"]
