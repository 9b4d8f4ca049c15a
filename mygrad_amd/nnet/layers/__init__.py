from .attention import AttentionMask, KeyValueCache, attention
from .batchnorm import batchnorm
from .conv import conv_nd
from .embedding import TokenIds, embedding
from .head_norm import RotaryTable, head_norm, rotate
from .layer_norm import layer_norm
from .pooling import max_pool
from .utils import sliding_window_copy, sliding_window_view

__all__ = ["AttentionMask", "KeyValueCache", "RotaryTable", "TokenIds", "attention", "batchnorm", "conv_nd", "embedding", "head_norm", "layer_norm",
           "max_pool", "rotate", "sliding_window_copy", "sliding_window_view"]
