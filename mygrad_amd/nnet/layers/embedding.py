"""Rows of a table by token on the MI355X, with the gradient of the table, and the tokens that it and the losses over a
vocabulary take.  The reference has no counterpart; the operation keeps its ``Operation`` contract
(``mygrad/operation_base.py:54-228``)."""

from math import prod
from numbers import Real
from typing import Optional

import numpy as np

from ... import _device, _hip
from ...operation_base import Operation
from ...tensor_base import Tensor

__all__ = ["TokenIds", "Embedding", "embedding"]

_DTYPES = (np.float16, np.float32, np.float64)


class TokenIds:
    """Tokens of a vocabulary, checked once and sent to the device once, for any number of calls.

    Parameters
    ----------
    ids : ArrayLike
        Whole numbers of any shape: places in a vocabulary, or -1 where there is no token (padding).

    >>> from mygrad_amd.nnet import TokenIds
    >>> TokenIds([[4, 0, 2], [1, -1, -1]])
    TokenIds(shape=(2, 3), below=5)
    """

    def __init__(self, ids):
        if isinstance(ids, Tensor):
            ids = ids.data
        arr = np.asarray(ids)
        if arr.size == 0 and arr.dtype == np.float64 and not isinstance(ids, np.ndarray):
            arr = arr.astype(np.int32)  # an empty list
        if arr.dtype.kind not in "iu":
            raise TypeError(f"tokens are whole numbers, got {arr.dtype}")
        if arr.size and (arr.min() < -1 or arr.max() >= 2**31 - 1):
            raise ValueError(f"tokens are places in a vocabulary, or -1 for none, got {arr.min()} to {arr.max()}")
        self._host = np.array(arr, dtype=np.int32, order="C")
        self._host.flags.writeable = False
        self._below = int(arr.max()) + 1 if arr.size else 0
        self._value = None

    @classmethod
    def _on_device(cls, value, below):
        """Tokens that a kernel wrote, all of them less than ``below``."""
        self = cls.__new__(cls)
        self._host, self._below, self._value = None, below, value
        return self

    # Read only: what they were checked for goes for all calls.
    @property
    def shape(self):
        return (self._value if self._host is None else self._host).shape

    @property
    def ndim(self):
        return len(self.shape)

    @property
    def size(self):
        return prod(self.shape)

    @property
    def below(self):
        """No token is as large as this."""
        return self._below

    @property
    def data(self):
        """The tokens as a NumPy array of int32, which is read only."""
        if self._host is None:
            host = self._value.host()
            host.flags.writeable = False
            self._host = host
        return self._host

    def reshape(self, *shape):
        """The same tokens in another shape."""
        if len(shape) == 1 and not isinstance(shape[0], (int, np.integer)):
            shape = tuple(shape[0])
        out = TokenIds.__new__(TokenIds)
        out._below = self._below
        out._host = None if self._host is None else self._host.reshape(shape)
        out._value = None if self._value is None else self._value.reshape(shape)
        return out

    def __array__(self, dtype=None, copy=None):
        return self.data.copy() if dtype is None else self.data.astype(dtype)

    def __len__(self):
        return self.shape[0]

    def __repr__(self):
        return f"TokenIds(shape={self.shape}, below={self.below})"

    def _buffer(self):
        if self._value is None:
            buf = _device.DeviceBuffer(max(self._host.nbytes, 16))
            if self._host.nbytes:
                buf.stage(self._host)
            self._value = _device.DeviceArray(buf, self._host.shape, np.int32)
        return self._value.buf


def as_tokens(ids, vocabulary):
    """``ids`` as :class:`TokenIds` that lie in a vocabulary of that size."""
    tokens = ids if isinstance(ids, TokenIds) else TokenIds(ids)
    if tokens.below > vocabulary:
        raise ValueError(f"tokens up to {tokens.below - 1} for a vocabulary of {vocabulary}")
    return tokens


class Embedding(Operation):
    """``weight:(vocabulary, dim)``."""

    takes_device_arrays = True

    def __call__(self, weight, *, tokens, scale):
        self.variables = (weight,)
        w = _device.value_of(weight)
        if w.ndim != 2:
            raise ValueError(f"`weight` must have the axes (vocabulary, dim), got shape {w.shape}")
        if w.dtype not in _DTYPES:
            raise TypeError(f"embedding runs on the GPU in float16, float32 or float64, got {w.dtype} (there is no CPU fallback)")
        if not isinstance(scale, Real) or not abs(scale) <= 1e30:
            raise ValueError(f"`scale` must be a number of at most 1e30 in size, got {scale}")
        self._tokens, self._scale = as_tokens(tokens, w.shape[0]), float(scale)
        shape = self._tokens.shape + w.shape[1:]
        if 0 in shape:
            return np.empty(shape, dtype=w.dtype)
        out, wb = _device.DeviceBuffer(prod(shape) * w.dtype.itemsize), _device.to_device(w)  # until the launch
        _hip.check(_hip.lib().mg_embedding_fwd(_hip.storage_code(w.dtype), self._tokens.size, *w.shape, self._scale, self._tokens._buffer().ptr,
                                               wb.ptr, out.ptr))
        y = _device.download(out, shape, w.dtype)
        _device.attach(y, out)
        return y

    def backward_var(self, grad, index, **kwargs):
        w = _device.value_of(self.variables[index])
        if grad.size == 0 or w.size == 0:
            return np.zeros(w.shape, dtype=w.dtype)
        if grad.shape != self._tokens.shape + w.shape[1:]:
            raise NotImplementedError(f"embedding backward for gradient of shape {grad.shape} (no CPU fallback)")
        out, gb = _device.DeviceBuffer(w.nbytes), _device.to_device(grad, w.dtype)
        _hip.check(_hip.lib().mg_embedding_bwd(_hip.storage_code(w.dtype), self._tokens.size, *w.shape, self._scale, self._tokens._buffer().ptr,
                                               gb.ptr, out.ptr))
        return _device.download(out, w.shape, w.dtype)


def embedding(weight, tokens, *, scale: float = 1.0, constant: Optional[bool] = None) -> Tensor:
    """Rows of ``weight:(vocabulary, dim)`` by token on the GPU, times ``scale``: ``(*tokens.shape, dim)``.

    ``weight`` is float16, float32 or float64.  ``tokens`` are whole numbers of any shape, less than ``vocabulary``; -1 stands for
    no token, whose row is zeros.  :class:`TokenIds` are checked and sent to the device once, any other array in each call.
    The gradient of ``weight`` is an array of its shape; the rows of a token that occurs more than once are added in float32
    (float64 for float64), and a result is rounded once.  The same call gives the same bits every time; in which order rows are added
    hangs on all tokens of the call.

    >>> import mygrad_amd as mg
    >>> from mygrad_amd.nnet import embedding
    >>> weight = mg.Tensor([[1.0, 2.0], [3.0, 4.0], [5.0, 6.0]])
    >>> y = embedding(weight, [2, 0, 2, -1])
    >>> y
    Tensor([[5., 6.],
            [1., 2.],
            [5., 6.],
            [0., 0.]])
    >>> y.backward()
    >>> weight.grad
    array([[1., 1.],
           [0., 0.],
           [2., 2.]])
    """
    return Tensor._op(Embedding, weight, op_kwargs=dict(tokens=tokens, scale=scale), constant=constant)
