from .activations import relu
from .layers import (AttentionMask, KeyValueCache, RotaryTable, TokenIds, attention, batchnorm, conv_nd, embedding, head_norm, layer_norm, max_pool,
                     rotate)
from .losses import distillation, log_probabilities

__all__ = ["AttentionMask", "KeyValueCache", "RotaryTable", "TokenIds", "attention", "batchnorm", "conv_nd", "distillation", "embedding", "head_norm",
           "layer_norm", "log_probabilities", "max_pool", "relu", "rotate"]
