"""Distillation from a teacher's likeliest tokens on the MI355X.  The reference has no counterpart; the operation keeps its
``Operation`` contract (``mygrad/operation_base.py:54-228``)."""

from math import prod
from numbers import Real
from typing import Optional

import numpy as np

from ... import _device, _graph, _hip
from ...operation_base import Operation
from ...tensor_base import Tensor
from ..layers.embedding import TokenIds, as_tokens
from .log_probabilities import result_type

__all__ = ["Distillation", "distillation"]

_DTYPES = (np.float16, np.float32, np.float64)
_MOST_TAUGHT = 256
_MOST_SHAPES = 64
_described = {}  # what was checked of calls of the same shapes


class Distillation(Operation):
    """``logits:(..., vocabulary)`` with ``teacher:(..., k)``, a constant."""

    takes_device_arrays = True

    def __call__(self, logits, teacher, *, tokens, temperature):
        self.variables = (logits, teacher)
        z, y = _device.value_of(logits), _device.value_of(teacher)
        if _graph.TRACK_GRAPH and not teacher.constant:
            raise ValueError("the teacher's logits have no gradient: they must be a constant")
        tokens = self._tokens = tokens if isinstance(tokens, TokenIds) else TokenIds(tokens)
        key = z.shape, z.dtype, y.shape, y.dtype, tokens.shape, temperature, type(temperature)
        found = _described.get(key)
        if found is None:
            found = self._describe(z, y, tokens, temperature)
            if len(_described) >= _MOST_SHAPES:
                _described.clear()
            _described[key] = found
        self._code, self._call, self._dtype, taught = found
        rows, vocabulary, count, _ = self._call
        as_tokens(tokens, vocabulary)
        lead, item = z.shape[:-1], self._dtype.itemsize
        self._empty = rows == 0
        if self._empty:
            return np.empty(lead, dtype=self._dtype)
        zb, yb = _device.to_device(z), _device.to_device(y, None if taught == y.dtype else taught)  # until the launch
        out = _device.DeviceBuffer(rows * item)
        # what the gradient needs of a row: three statistics and the shares of its tokens
        self._kept = None if logits.constant else _device.DeviceBuffer((3 + count) * rows * item)
        _hip.check(_hip.lib().mg_distillation_fwd(self._code, _hip.storage_code(taught), *self._call, zb.ptr, tokens._buffer().ptr,
                                                  yb.ptr, out.ptr, *self._both()))
        loss = _device.download(out, lead, self._dtype)
        _device.attach(loss, out)
        return loss

    def _both(self):
        """Where the statistics and the shares lie."""
        if self._kept is None:
            return None, None
        return self._kept.ptr, self._kept.ptr + 3 * self._call[0] * self._dtype.itemsize

    @staticmethod
    def _describe(z, y, tokens, temperature):
        """The checked arguments of the entry points, the type of the loss and the one that the teacher's logits are taken in."""
        if z.ndim < 1 or z.shape[-1] == 0:
            raise ValueError(f"`logits` must have the axes (..., vocabulary), got shape {z.shape}")
        if z.dtype not in _DTYPES or y.dtype not in _DTYPES:
            raise TypeError(f"distillation runs on the GPU in float16, float32 or float64, got {z.dtype} and {y.dtype} (there is no CPU fallback)")
        dtype = result_type(z.dtype)
        if y.dtype == np.float64 and dtype != np.float64:
            raise TypeError(f"a teacher in float64 for logits in {z.dtype}: its digits would be lost")
        if y.shape != tokens.shape or y.ndim < 1 or y.shape[:-1] != z.shape[:-1]:
            raise ValueError(f"tokens of shape {tokens.shape} and teacher's logits of shape {y.shape} for logits of shape {z.shape}")
        if not 1 <= y.shape[-1] <= _MOST_TAUGHT:
            raise ValueError(f"a row is taught by 1 to {_MOST_TAUGHT} tokens, got {y.shape[-1]}")
        if not isinstance(temperature, Real) or not 1e-30 <= temperature <= 1e30:
            raise ValueError(f"`temperature` must be a positive number (1e-30 to 1e30), got {temperature}")
        call = prod(z.shape[:-1]), z.shape[-1], y.shape[-1], float(temperature)
        return _hip.storage_code(z.dtype), call, dtype, y.dtype if y.dtype in (z.dtype, dtype) else dtype

    def backward_var(self, grad, index, **kwargs):
        z = _device.value_of(self.variables[0])
        if index != 0:
            raise NotImplementedError("the teacher's logits have no gradient")
        if self._empty:
            return np.zeros(z.shape, dtype=z.dtype)
        if grad.shape != z.shape[:-1]:
            raise NotImplementedError(f"distillation backward for gradient of shape {grad.shape} (no CPU fallback)")
        out, zb, gb = _device.DeviceBuffer(z.nbytes), _device.to_device(z), _device.to_device(grad, self._dtype)
        _hip.check(_hip.lib().mg_distillation_bwd(self._code, *self._call, zb.ptr, self._tokens._buffer().ptr, *self._both(),
                                                  gb.ptr, out.ptr))
        return _device.download(out, z.shape, z.dtype)


def distillation(logits, tokens, teacher, *, temperature: float = 1.0, constant: Optional[bool] = None) -> Tensor:
    """How far each row of ``logits:(..., vocabulary)`` is from a teacher that names its likeliest tokens, on the GPU::

        p = softmax(logits / temperature)        q = softmax(teacher / temperature)
        loss = sum(q * (log(q) - log(p[tokens])))

    Parameters
    ----------
    logits : ArrayLike, shape=(..., vocabulary)
        float16, float32 or float64; ``p`` is over the whole vocabulary.
    tokens : ArrayLike, shape=(..., k)
        The teacher's tokens for each row, at most 256 (whole numbers, or :class:`~mygrad_amd.nnet.TokenIds` such as
        :func:`~mygrad_amd.nnet.log_probabilities` gives); -1 where the teacher names fewer.
    teacher : ArrayLike, shape=(..., k)
        The teacher's logits (or log probabilities) of those tokens, a constant; ``q`` is over these alone.  float16 or float32, float64
        beside logits of float64.
    temperature : float
        Divides both sides' logits.  Neither the loss nor its gradient is multiplied by its square.
    constant : Optional[bool]
        If True, the returned tensor is a constant.

    Returns
    -------
    Tensor
        A loss for each row, float32 (float64 for float64 logits).  Without any of the teacher's tokens it is 0 and has no gradient.
        Against a row whose logits are all minus infinity it is infinite and has no gradient; infinity or NaN among a
        row's logits or the teacher's makes its results NaN.

    >>> import mygrad_amd as mg
    >>> from mygrad_amd.nnet import distillation
    >>> logits = mg.Tensor([[0.0, 1.0, 3.0, 2.0]])
    >>> loss = distillation(logits, [[2, 3]], [[1.0, 0.0]])
    >>> loss.data.round(3)
    array([0.127])
    >>> loss.backward()
    >>> logits.grad.round(3)
    array([[ 0.032,  0.087, -0.087, -0.032]])
    """
    return Tensor._op(Distillation, logits, teacher, op_kwargs=dict(tokens=tokens, temperature=temperature), constant=constant)
