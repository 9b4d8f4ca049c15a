from .attention import AttentionMask, KeyValueCache, attention
from .batchnorm import batchnorm
from .conv import conv_nd
from .head_norm import RotaryTable, head_norm, rotate
from .pooling import max_pool
from .utils import sliding_window_copy, sliding_window_view

__all__ = ["AttentionMask", "KeyValueCache", "RotaryTable", "attention", "batchnorm", "conv_nd", "head_norm", "max_pool", "rotate",
           "sliding_window_copy", "sliding_window_view"]
