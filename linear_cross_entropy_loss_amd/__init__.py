"""MI355X-native fused linear + cross-entropy loss (drop-in for ``linear_cross_entropy``), and what else is done at the output
layer of a language model: distillation from a teacher's top logits, the top logits of a row, sampling."""
from .ops import fwd_configs, bwd_configs, LinearCrossEntropyLoss, linear_cross_entropy, LinearXentImplementation
from .distillation import linear_distillation
from .selection import sample_logits, top_logits

__all__ = ["fwd_configs", "bwd_configs", "LinearCrossEntropyLoss", "linear_cross_entropy",
           "LinearXentImplementation", "linear_distillation", "sample_logits", "top_logits"]
