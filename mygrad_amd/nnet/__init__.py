from .activations import relu
from .layers import AttentionMask, KeyValueCache, RotaryTable, attention, batchnorm, conv_nd, head_norm, max_pool, rotate

__all__ = ["AttentionMask", "KeyValueCache", "RotaryTable", "attention", "batchnorm", "conv_nd", "head_norm", "max_pool", "relu", "rotate"]
