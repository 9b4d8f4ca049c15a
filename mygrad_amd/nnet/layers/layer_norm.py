"""Layer norm on the MI355X.  The reference has no counterpart; the operation keeps its ``Operation`` contract
(``mygrad/operation_base.py:54-228``)."""

from math import prod
from typing import Optional

import numpy as np

from ... import _device, _hip
from ...operation_base import Operation
from ...tensor_base import Tensor

__all__ = ["LayerNorm", "layer_norm"]

_DTYPES = (np.float16, np.float32, np.float64)
_MOST_SHAPES = 64
_described = {}  # what was checked of calls of the same shapes


class LayerNorm(Operation):
    """``x:(..., dim)``, and ``weight:(dim,)`` and ``bias:(dim,)`` where there are any: ``given`` names them."""

    takes_device_arrays = True

    def __call__(self, x, *params, eps, given):
        self.variables = (x, *params)
        values = [_device.value_of(t) for t in self.variables]
        xd = values[0]
        key = tuple([(v.shape, v.dtype) for v in values]), given, eps
        found = _described.get(key)
        if found is None:
            found = self._describe(values, given, eps)
            if len(_described) >= _MOST_SHAPES:
                _described.clear()
            _described[key] = found
        self._call, self._places, self._sizes, item = found
        self._empty = self._call[1] * self._call[2] == 0
        self._backed = None
        if self._empty:
            return np.empty(xd.shape, dtype=xd.dtype)
        held = [_device.to_device(v) for v in values]  # until the launch
        # behind the result, for the gradient: two parts of the mean and 1 / sqrt for each row
        self._kept, behind = None, -(-self._sizes[0] // 16) * 16
        out = _device.DeviceBuffer(behind + 3 * self._call[1] * item)
        if not all([t.constant for t in self.variables]):
            self._kept = out.ptr + behind
            self._result = out
        xp, wp, bp = (None if n is None else held[n].ptr for n in self._places)
        _hip.check(_hip.lib().mg_layer_norm_fwd(*self._call, float(eps), xp, wp, bp, out.ptr, self._kept))
        y = _device.download(out, xd.shape, xd.dtype)
        _device.attach(y, out)
        return y

    @staticmethod
    def _describe(values, given, eps):
        """The checked arguments of the entry points, where x, weight and bias are among the variables, the variables' bytes, and those of a statistic."""
        x = values[0]
        if x.ndim < 1:
            raise ValueError(f"`x` must have the axes (..., dim), got shape {x.shape}")
        if x.dtype not in _DTYPES:
            raise TypeError(f"layer_norm runs on the GPU in float16, float32 or float64, got {x.dtype} (there is no CPU fallback)")
        dim = x.shape[-1]
        for name, value in zip(given, values[1:]):
            if value.shape != (dim,):
                raise ValueError(f"`{name}` must have shape ({dim},), got {value.shape}")
            if value.dtype != x.dtype:
                raise TypeError(f"layer_norm takes `{name}` in the dtype of `x` ({x.dtype}), got {value.dtype}")
        if not 0 <= eps < np.inf:
            raise ValueError(f"`eps` must be a non-negative number, got {eps}")
        places = 0, *(1 + given.index(name) if name in given else None for name in ("weight", "bias"))
        return (_hip.storage_code(x.dtype), prod(x.shape[:-1]), dim), places, [v.nbytes for v in values], 8 if x.dtype == np.float64 else 4

    def _run_backward(self, grad, want):
        values = [_device.value_of(t) for t in self.variables]
        x = values[0]
        if grad.shape != x.shape:
            raise NotImplementedError(f"layer_norm backward for gradient of shape {grad.shape} (no CPU fallback)")
        xb, gb = _device.to_device(x), _device.to_device(grad, x.dtype)
        wb = None if self._places[1] is None else _device.to_device(values[self._places[1]])
        out = {i: _device.DeviceBuffer(self._sizes[i]) for i in want}
        _hip.check(_hip.lib().mg_layer_norm_bwd(*self._call, xb.ptr, None if wb is None else wb.ptr, self._kept, gb.ptr,
                                                *(out[i].ptr if i in out else None for i in self._places)))
        return {i: _device.download(buf, values[i].shape, x.dtype) for i, buf in out.items()}

    def backward_var(self, grad, index, **kwargs):
        if self._empty:
            value = _device.value_of(self.variables[index])
            return np.zeros(value.shape, dtype=value.dtype)
        # backward() asks for each variable in turn with the same `grad`: the first request computes all that are wanted
        if self._backed is None or self._backed[0] is not grad or index not in self._backed[1]:
            want = {index} | {i for i, var in enumerate(self.variables) if not var.constant}
            self._backed = (grad, self._run_backward(grad, want))
        out = self._backed[1].pop(index)
        if not self._backed[1]:
            self._backed = None
        return out


def layer_norm(x, weight=None, bias=None, *, eps: float, constant: Optional[bool] = None) -> Tensor:
    """Norm each row of ``x:(..., dim)`` on the GPU::

        y = weight * (x - mean(x)) / sqrt(mean((x - mean(x)) ** 2) + eps) + bias

    ``weight`` and ``bias`` are ``(dim,)`` in the dtype of ``x`` (float16, float32 or float64), or None; ``eps`` is a
    non-negative number and has no default.  Sums are carried in float32 (float64 for float64), the gradients of
    ``weight`` and ``bias`` are joined in float64, and each result is rounded once.  A row whose squared deviations add up to more than
    float32 (float64) holds, 3e38, is scaled by 0.

    >>> import mygrad_amd as mg
    >>> from mygrad_amd.nnet import layer_norm
    >>> layer_norm(mg.Tensor([[1.0, 2.0, 3.0], [4.0, 4.0, 10.0]]), eps=0.0).data.round(3)
    array([[-1.225,  0.   ,  1.225],
           [-0.707, -0.707,  1.414]])
    """
    if eps is None:
        raise TypeError("`eps` must be a non-negative number")
    given = [(name, value) for name, value in (("weight", weight), ("bias", bias)) if value is not None]
    return Tensor._op(LayerNorm, x, *[value for _, value in given], op_kwargs=dict(eps=eps, given=tuple([name for name, _ in given])), constant=constant)
