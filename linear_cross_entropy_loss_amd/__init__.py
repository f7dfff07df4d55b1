"""MI355X-native fused linear + cross-entropy loss (drop-in for ``linear_cross_entropy``), and what else is done at the output
layer of a language model: distillation from a teacher's top logits, the top logits of a row, sampling; the log-probabilities of given tokens
with their gradients, logits of 8-bit weights, clipping of gradients."""
from .ops import fwd_configs, bwd_configs, LinearCrossEntropyLoss, linear_cross_entropy, LinearXentImplementation
from .distillation import linear_distillation
from .selection import sample_logits, top_logits
from .token_logits import linear_token_logits
from .quantization import Quantized, quantize_rows, quantize_weight, quantized_logits
from .clipping import clip_gradients

__all__ = ["fwd_configs", "bwd_configs", "LinearCrossEntropyLoss", "linear_cross_entropy",
           "LinearXentImplementation", "linear_distillation", "sample_logits", "top_logits", "linear_token_logits", "Quantized",
           "quantize_rows", "quantize_weight", "quantized_logits", "clip_gradients"]
