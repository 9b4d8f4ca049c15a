"""A norm for each head and rotary positions in one pass on the MI355X, for the queries and keys of an attention.
The reference has no counterpart; the operation keeps its ``Operation`` contract (``mygrad/operation_base.py:54-228``)."""

from math import prod
from numbers import Integral
from typing import Optional

import numpy as np

from ... import _device, _hip
from ...operation_base import Operation
from ...tensor_base import Tensor

__all__ = ["head_norm", "rotate", "HeadNorm", "RotaryTable", "RotaryPositions"]

_DTYPES = (np.float16, np.float32, np.float64)
_MOST_SHAPES = 64  # that positions keep device copies and descriptors for; those in use are held by their users as well


class RotaryTable:
    """cos and sin of the angles that rotary positions turn pairs of values by, made once.

    Parameters
    ----------
    sections : int or sequence of ints
        Pairs of a head's values that each axis of positions turns: ``dim // 2`` for the one axis of a text,
        ``(16, 24, 24)``, say, for time, height and width.  What the pairs leave of a head stays as it is.
    length : int
        Positions lie in ``[0, length)``.
    base : float
        Pair ``m`` of the ``n`` of an axis turns by ``position * base ** (-m / n)``.
    interleaved : bool
        Pairs are values ``(2p, 2p + 1)``; otherwise ``(p, p + P)`` with ``P`` pairs in all.
    """

    def __init__(self, sections, length, *, base=10000.0, interleaved=False):
        sections = (sections,) if isinstance(sections, Integral) else tuple(sections)
        if not sections or len(sections) > 255 or not all(isinstance(n, Integral) and n >= 0 for n in sections) or not 1 <= sum(sections) <= 512:
            raise ValueError(f"`sections` are pairs for each axis, 1 to 512 in all, got {sections}")
        if not isinstance(length, Integral) or not 1 <= length < 1 << 30:
            raise ValueError(f"`length` must be a whole number of 1 or more, got {length}")
        if not base > 0 or not np.isfinite(base):
            raise ValueError(f"`base` must be a positive number, got {base}")
        if not isinstance(interleaved, (bool, np.bool_)):
            raise TypeError(f"`interleaved` must be a boolean value, got: {interleaved}")
        self._sections, self._length, self._interleaved = tuple(map(int, sections)), int(length), bool(interleaved)
        frequency = np.concatenate([float(base) ** (-np.arange(n) / n) if n else np.empty(0) for n in self.sections])
        angle = np.arange(self.length)[:, None] * frequency
        self._turns = np.stack((np.cos(angle), np.sin(angle)), -1)
        self._axis_of = np.repeat(np.arange(len(self.sections)), self.sections).astype(np.uint8)
        self._buffers = {}

    # Read only: the angles are made of them.
    @property
    def sections(self):
        return self._sections

    @property
    def length(self):
        return self._length

    @property
    def interleaved(self):
        return self._interleaved

    @property
    def pairs(self):
        """Of all axes."""
        return sum(self._sections)

    def _buffer(self, what):
        buf = self._buffers.get(what)
        if buf is None:
            arr = self._axis_of if what == "axis_of" else self._turns.astype(what)
            buf = self._buffers[what] = _device.from_host(np.ascontiguousarray(arr)).buf
        return buf

    def at(self, positions):
        """The table at the positions of some tokens, for any number of calls: ``positions`` are whole numbers of
        shape ``(..., axes)`` whose leading axes broadcast to those of the tokens, or ``(tokens,)`` for one axis."""
        return RotaryPositions(self, positions)


class RotaryPositions:
    """What :meth:`RotaryTable.at` gives."""

    def __init__(self, table, positions):
        arr = np.array(positions)
        whole = arr.shape == (len(table.sections),)  # one token's, or for one axis those of one token in a row of one
        if arr.dtype.kind not in "iu":
            raise TypeError(f"positions are whole numbers, got {arr.dtype}")
        axes = len(table.sections)
        if arr.ndim == 1 and axes == 1:
            arr = arr[:, None]
        if arr.ndim < 1 or arr.shape[-1] != axes:
            raise ValueError(f"positions must have shape (..., {axes}) for {axes} axes, got {arr.shape}")
        if arr.size and (arr.min() < 0 or arr.max() >= table.length):
            raise ValueError(f"positions must lie in [0, {table.length}), got {arr.min()} to {arr.max()}")
        self._table, self._positions, self._whole = table, arr.astype(np.int32), whole
        self._bound, self._described = {}, {}

    @property
    def table(self):
        return self._table

    def _check(self, lead):
        try:
            fits = lead == () and self._whole or np.broadcast_shapes(self._positions.shape[:-1], lead) == lead
        except ValueError:
            fits = False
        if not fits:
            raise ValueError(f"positions of shape {self._positions.shape} for tokens of shape {lead}")

    def _buffer(self, lead):
        buf = self._bound.get(lead)
        if buf is None:
            self._check(lead)
            if len(self._bound) >= _MOST_SHAPES:
                self._bound.clear()
            spread = self._positions if lead == () else np.broadcast_to(self._positions, lead + self._positions.shape[-1:])
            buf = self._bound[lead] = _device.from_host(np.ascontiguousarray(spread)).buf
        return buf


_described = {}  # descriptors of norms without positions


class HeadNorm(Operation):
    """``x:(..., heads, dim)`` with ``weight:(dim,)`` or ``(heads, dim)``; an empty ``weight`` stands for none."""

    takes_device_arrays = True

    def __call__(self, x, weight, *, eps, rotary):
        """``eps`` None: no norm."""
        self.variables = (x, weight)
        xd, wd = _device.value_of(x), _device.value_of(weight)
        if rotary is not None and not isinstance(rotary, RotaryPositions):
            raise TypeError(f"`rotary` must come from RotaryTable.at, got {type(rotary).__name__}")
        self._backed = None
        self._weighted = wd.size > 0
        described = _described if rotary is None else rotary._described
        key = xd.shape, xd.dtype, wd.shape, wd.dtype, eps
        found = described.get(key)
        if found is None:
            found = self._describe(xd, wd, eps, rotary)
            if xd.size == 0:
                return np.empty(xd.shape, dtype=xd.dtype)
            if len(described) >= _MOST_SHAPES:
                described.clear()
            described[key] = found
        self._desc, self._table, self._held = found
        xb = _device.to_device(xd)
        wb = _device.to_device(wd) if self._weighted else None
        out = _device.DeviceBuffer(xd.nbytes)
        _hip.check(_hip.lib().mg_head_norm_fwd(self._desc, xb.ptr, None if wb is None else wb.ptr, self._table, out.ptr))
        y = _device.download(out, xd.shape, xd.dtype)
        _device.attach(y, out)
        return y

    def _describe(self, x, w, eps, rotary):
        """The checked descriptor (nothing writes to it), the table's address, and what holds the memory of both."""
        if x.ndim < 2:
            raise ValueError(f"`x` must have the axes (..., heads, dim), got shape {x.shape}")
        if x.dtype not in _DTYPES:
            raise TypeError(f"head_norm runs on the GPU in float16, float32 or float64, got {x.dtype} (there is no CPU fallback)")
        lead, (heads, dim) = x.shape[:-2], x.shape[-2:]
        if not 1 <= dim <= 1024 or heads > 65535:
            raise ValueError(f"heads have 1 to 1024 values and number at most 65535, got {x.shape}")
        if self._weighted:
            if w.shape not in ((dim,), (heads, dim)):
                raise ValueError(f"`weight` must have shape ({dim},) or ({heads}, {dim}), got {w.shape}")
            if w.dtype != x.dtype:
                raise TypeError(f"head_norm takes `weight` in the dtype of `x` ({x.dtype}), got {w.dtype}")
        if eps is not None and not 0 <= eps < np.inf:
            raise ValueError(f"`eps` must be a non-negative number, got {eps}")
        table = None if rotary is None else rotary.table
        if table is not None:
            if 2 * table.pairs > dim:
                raise ValueError(f"{table.pairs} pairs do not fit in {dim} values")
            rotary._check(lead)
        if x.size == 0:
            return None
        desc = _hip.HeadNormDesc(_hip.storage_code(x.dtype), eps is not None, w.size // dim if self._weighted else 0, 0, 1, 0, prod(lead),
                                 heads, dim, 0, 0, 0.0 if eps is None else eps, None, None)
        if table is None:
            return desc, None, None
        desc.interleaved, desc.axes, desc.pairs, desc.table_rows = table.interleaved, len(table.sections), table.pairs, table.length
        held = rotary._buffer(lead), table._buffer("axis_of"), table._buffer("f8" if x.dtype == np.float64 else "f4")
        desc.positions, desc.axis_of = held[0].ptr, held[1].ptr
        return desc, held[2].ptr, held

    def _run_backward(self, grad, want):
        x, w = (_device.value_of(t) for t in self.variables)
        if grad.shape != x.shape:
            raise NotImplementedError(f"head_norm backward for gradient of shape {grad.shape} (no CPU fallback)")
        xb, gb = _device.to_device(x), _device.to_device(grad, x.dtype)
        wb = _device.to_device(w) if self._weighted else None
        out = {i: _device.DeviceBuffer(a.nbytes) for i, a in enumerate((x, w)) if i in want}
        _hip.check(_hip.lib().mg_head_norm_bwd(self._desc, xb.ptr, None if wb is None else wb.ptr, self._table, gb.ptr,
                                               *(out[i].ptr if i in out else None for i in range(2))))
        return {i: _device.download(buf, (x, w)[i].shape, x.dtype) for i, buf in out.items()}

    def backward_var(self, grad, index, **kwargs):
        value = _device.value_of(self.variables[index])
        if _device.value_of(self.variables[0]).size == 0 or value.size == 0:
            return np.zeros(value.shape, dtype=value.dtype)
        # backward() asks for each variable in turn with the same `grad`: the first request computes all that are wanted
        if self._backed is None or self._backed[0] is not grad or index not in self._backed[1]:
            want = {index} | {i for i, var in enumerate(self.variables) if not var.constant and (i == 0 or self._weighted)}
            self._backed = (grad, self._run_backward(grad, want))
        out = self._backed[1].pop(index)
        if not self._backed[1]:
            self._backed = None
        return out


def head_norm(x, weight=None, *, eps: float, rotary: Optional[RotaryPositions] = None, constant: Optional[bool] = None) -> Tensor:
    """Norm the values of each head of ``x:(..., heads, dim)`` on the GPU, and turn them by rotary positions::

        y = turn(weight * x / sqrt(mean(x ** 2) + eps))

    ``weight`` is ``(dim,)``, one for all heads, or ``(heads, dim)`` (so queries and keys of one projection take one call),
    in the dtype of ``x`` (float16, float32 or float64), or None; ``eps`` is a non-negative number and has no default;
    ``rotary`` comes from :meth:`RotaryTable.at`, None leaves the values where they are.  Sums and angles are carried in
    float32 (float64 for float64), the result is rounded once.

    >>> import mygrad_amd as mg
    >>> from mygrad_amd.nnet import RotaryTable, head_norm
    >>> table = RotaryTable(1, 8)
    >>> head_norm(mg.Tensor([[[3.0, 4.0]], [[3.0, 4.0]]]), eps=0.0, rotary=table.at([0, 1])).data.round(3)
    array([[[ 0.849,  1.131]],
           [[-0.493,  1.325]]])
    """
    if eps is None:
        raise TypeError("`eps` must be a non-negative number; without a norm use rotate()")
    if weight is None:
        weight = np.array([])
    elif 0 in np.shape(weight) and np.shape(weight) != np.shape(x)[-2:]:  # to the operation an empty one is none
        raise ValueError(f"`weight` of shape {np.shape(weight)} for heads of shape {np.shape(x)[-2:]}")
    return Tensor._op(HeadNorm, x, weight, op_kwargs=dict(eps=eps, rotary=rotary), constant=constant)


def rotate(x, rotary: RotaryPositions, *, constant: Optional[bool] = None) -> Tensor:
    """Turn the values of each head of ``x:(..., heads, dim)`` by rotary positions (:func:`head_norm` without the norm)."""
    if rotary is None:
        raise TypeError("`rotary` must come from RotaryTable.at, got None")
    return Tensor._op(HeadNorm, x, np.array([]), op_kwargs=dict(eps=None, rotary=rotary), constant=constant)
