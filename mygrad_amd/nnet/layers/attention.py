"""Attention on the MI355X: scores with a cap, a bias by distance and masks, its gradients, and a cache of keys
and values for a few new tokens at a time.  The reference has no counterpart; the operation keeps its ``Operation``
contract (``mygrad/operation_base.py:54-228``)."""

from typing import Optional

import numpy as np

from ... import _device, _graph, _hip
from ...operation_base import Operation
from ...tensor_base import Tensor

__all__ = ["attention", "Attention", "AttentionMask", "KeyValueCache"]

_DTYPES = (np.float16, np.float32, np.float64)
_MOST_TOKENS = 1 << 30
_MOST_SHAPES = 64  # that a mask keeps device copies and descriptors for; those in use are held by their users as well


def _integers(values, what, ndim):
    arr = np.array(values)
    if arr.dtype.kind not in "iu":
        raise TypeError(f"{what} are whole numbers, got {arr.dtype}")
    if arr.ndim not in ndim:
        raise ValueError(f"{what} have {' or '.join(map(str, ndim))} axes, got shape {arr.shape}")
    return arr


class AttentionMask:
    """Which keys each query sees.  Made once and used by any number of calls (the layers of a model, say): what it
    needs on the device is uploaded by the first of them.

    The last query stands at the last key: of ``n`` keys and ``t`` queries, query ``i`` is at ``i + n - t``.

    Parameters
    ----------
    causal : bool
        No query sees a key behind its own place.
    window : int, optional
        A query sees the ``window`` keys that end at its place (not causal: and as many that begin there).
    prefix : int or array of ints (batch,), optional
        Every query also sees the first ``prefix`` keys (of its document).  Only with ``causal``, not with ``window``.
    documents : array of ints (keys,) or (batch, keys), optional
        The document each token belongs to; a query sees its own document only.  A document is one run of tokens.
        Tokens of a negative number are padding: they see nothing and nothing sees them.
    lengths : int or array of ints (batch,), optional
        Keys in use; those behind them are not looked at, whatever they hold.
    """

    def __init__(self, causal=False, *, window=None, prefix=None, documents=None, lengths=None):
        if not isinstance(causal, (bool, np.bool_)):
            raise TypeError(f"`causal` must be a boolean value, got: {causal}")
        self._causal = bool(causal)
        self._window = 0
        if window is not None:
            if _integers(window, "keys in a window", (0,)) < 1:
                raise ValueError(f"a window holds one key or more, got {window}")
            self._window = min(int(window), _MOST_TOKENS)
        self._lengths = self._prefix = self._starts = self._ends = None
        if prefix is not None:
            if not self._causal or window is not None:
                raise ValueError("a prefix goes with a causal mask without a window")
            self._prefix = self._counts(prefix, "keys of a prefix")
        if lengths is not None:
            self._lengths = self._counts(lengths, "lengths")
            self._shortest, self._mean, self._longest = (int(f(self._lengths)) if self._lengths.size else 0 for f in (np.min, np.mean, np.max))
        if documents is not None:
            self._starts, self._ends = _runs(np.atleast_2d(_integers(documents, "numbers of documents", (1, 2))))
        self._bound, self._described = {}, {}

    @staticmethod
    def _counts(values, what):
        arr = _integers(values, what, (0, 1))
        if arr.size and (arr.min() < 0 or arr.max() >= _MOST_TOKENS):
            raise ValueError(f"{what} lie in [0, 2**30), got {arr.min()} to {arr.max()}")
        return arr.astype(np.int32)

    # Read only: descriptors that calls have made are not made again.
    @property
    def causal(self):
        return self._causal

    @property
    def window(self):
        """Keys of the window, 0 for none."""
        return self._window

    @property
    def lengths(self):
        """Keys in use of each sequence, or None."""
        return None if self._lengths is None else self._lengths.copy()

    def _check(self, batch, keys):
        for what, arr in (("lengths", self._lengths), ("prefix", self._prefix)):
            if arr is not None and arr.ndim and arr.shape != (batch,):
                raise ValueError(f"`{what}` must have shape ({batch},) for a batch of {batch}, got {arr.shape}")
        if self._lengths is not None and self._longest > keys:
            raise ValueError(f"a length of {self._longest} among {keys} keys")
        if self._starts is not None and (self._starts.shape[1] != keys or self._starts.shape[0] not in (1, batch)):
            raise ValueError(f"`documents` must have shape ({keys},) or ({batch}, {keys}), got {self._starts.shape}")

    def _bind(self, batch, keys):
        """Device buffers (lengths, prefix, starts, ends) for a batch of that many keys; whoever launches with them holds them."""
        held = self._bound.get((batch, keys))
        if held is None:
            self._check(batch, keys)
            if len(self._bound) >= _MOST_SHAPES:
                self._bound.clear()
            held = self._bound[batch, keys] = tuple(None if arr is None else _uploaded(np.broadcast_to(arr, shape)) for arr, shape in (
                (self._lengths, (batch,)), (self._prefix, (batch,)), (self._starts, (batch, keys)), (self._ends, (batch, keys))))
        return held


def _uploaded(arr):
    return _device.from_host(np.ascontiguousarray(arr)).buf


def _runs(ids):
    """First and one-behind-last place of the run that each place of ``ids``:(batch, keys) lies in; 0, 0 for padding."""
    batch, keys = ids.shape
    if keys >= _MOST_TOKENS:
        raise ValueError(f"2**30 keys or more: {keys}")
    place = np.arange(keys, dtype=np.int32)
    begins = np.ones(ids.shape, dtype=bool)
    begins[:, 1:] = ids[:, 1:] != ids[:, :-1]
    starts = np.maximum.accumulate(np.where(begins, place, 0), axis=1)
    last = np.ones(ids.shape, dtype=bool)
    last[:, :-1] = begins[:, 1:]
    ends = np.minimum.accumulate(np.where(last, place + 1, keys)[:, ::-1], axis=1)[:, ::-1]
    for row, first in zip(ids, begins):
        named = row[first & (row >= 0)]
        if np.unique(named).size != named.size:
            raise ValueError("a document is one run of tokens: a number comes back behind another one")
    padding = ids < 0
    return (np.where(padding, 0, a).astype(np.int32) for a in (starts, ends))


_LARGEST = 1e30  # of scale and cap in single precision, and one over it the smallest cap: their quotients and products stay numbers there


def _check_scores(scale, cap, dim, dtype):
    scale = dim ** -0.5 if scale is None else float(scale)
    if not np.isfinite(scale):
        raise ValueError(f"`scale` must be finite, got {scale}")
    cap = 0.0 if cap is None else float(cap)
    if cap < 0 or not np.isfinite(cap):
        raise ValueError(f"`cap` must be a positive number or None, got {cap}")
    if dtype != np.float64 and (abs(scale) > _LARGEST or cap > _LARGEST or 0 < cap < 1 / _LARGEST):
        raise ValueError(f"scores in single precision take a `scale` of at most {_LARGEST:g} and a `cap` of {1 / _LARGEST:g} to {_LARGEST:g}, "
                         f"got {scale} and {cap or None}")
    return scale, cap


def _slopes_on_device(slopes, heads, dtype):
    if slopes is None:
        return None
    if isinstance(slopes, Tensor):
        if _graph.TRACK_GRAPH and not slopes.constant:
            raise ValueError("`slopes` have no gradient: pass a constant tensor or an array")
        slopes = slopes._value
    elif not isinstance(slopes, np.ndarray):
        slopes = np.asarray(slopes)
    if slopes.shape != (heads,):
        raise ValueError(f"`slopes` must have shape ({heads},), one for each query head, got {slopes.shape}")
    if slopes.dtype.kind != "f":
        raise TypeError(f"`slopes` are floating-point numbers, got {slopes.dtype}")
    return _device.to_device(slopes, np.float64 if dtype == np.float64 else np.float32)


_UNMASKED = AttentionMask()


def _describe(q, k, v, scale, cap, slopes, mask):
    """The descriptor, checked once for each mask and set of shapes and types (nothing writes to it), and the buffers that it points to,
    which have to outlive it."""
    if mask is None:
        mask = _UNMASKED
    elif not isinstance(mask, AttentionMask):
        raise TypeError(f"`mask` must be an AttentionMask, got {type(mask).__name__}")
    sloped = _slopes_on_device(slopes, q.shape[2], q.dtype) if slopes is not None and q.ndim == 4 else None
    key = q.shape, k.shape, v.shape, q.dtype, k.dtype, v.dtype, scale, cap
    found = mask._described.get(key)
    if found is None:
        _check_operands(q, k, v)
        scale, cap = _check_scores(scale, cap, q.shape[3], q.dtype)
        (batch, queries, heads, dim), (keys, kv_heads) = q.shape, k.shape[1:3]
        mask._check(batch, keys)
        if not q.size:
            return None, None  # nothing to compute, nothing to upload
        buffers = mask._bind(batch, keys)
        longest, mean = (0, 0) if mask._lengths is None else (max(mask._longest, 1), mask._mean)
        desc = _hip.AttentionDesc(_hip.storage_code(q.dtype), mask._causal, batch, queries, keys, heads, kv_heads, dim, mask._window, scale, cap, longest, mean,
                                  *(None if b is None else b.ptr for b in buffers), None)
        if len(mask._described) >= _MOST_SHAPES:
            mask._described.clear()
        found = mask._described[key] = desc, buffers
    if sloped is None:
        return found
    desc = _hip.AttentionDesc.from_buffer_copy(found[0])
    desc.slopes = sloped.ptr
    return desc, (found[1], sloped)


def _check_operands(q, k, v):
    for name, arr in (("q", q), ("k", k), ("v", v)):
        if arr.ndim != 4:
            raise ValueError(f"`{name}` must have the axes (batch, tokens, heads, dim), got shape {arr.shape}")
        if arr.dtype not in _DTYPES:
            raise TypeError(f"attention runs on the GPU in float16, float32 or float64, got {arr.dtype} (there is no CPU fallback)")
        if arr.dtype != q.dtype:
            raise TypeError(f"attention takes q, k and v in one dtype, got {q.dtype}, {k.dtype} and {v.dtype}")
    if k.shape != v.shape:
        raise ValueError(f"k and v must have one shape, got {k.shape} and {v.shape}")
    if q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError(f"q and k must agree in batch and head dimension, got {q.shape} and {k.shape}")
    if q.shape[2] == 0 or k.shape[2] == 0 or q.shape[2] % k.shape[2]:
        raise ValueError(f"the query heads must be a multiple of the key heads, got {q.shape[2]} and {k.shape[2]}")
    if not 1 <= q.shape[3] <= 256:
        raise ValueError(f"the head dimension must be 1 to 256, got {q.shape[3]}")


class Attention(Operation):
    """``q:(batch, queries, heads, dim)`` over ``k, v:(batch, keys, key heads, dim)``."""

    takes_device_arrays = True

    def __call__(self, q, k, v, *, scale=None, cap=None, slopes=None, mask=None):
        self.variables = (q, k, v)
        qd, kd, vd = (_device.value_of(t) for t in (q, k, v))
        self._backed = None
        self._desc, self._held = _describe(qd, kd, vd, scale, cap, slopes, mask)
        if self._desc is None:
            return np.zeros(qd.shape, dtype=qd.dtype)
        qb, kb, vb = (_device.to_device(a) for a in (qd, kd, vd))
        self._out = _device.DeviceBuffer(qd.nbytes)
        self._lse = self._rest = None
        if _graph.TRACK_GRAPH and not (q.constant and k.constant and v.constant):
            wide = 8 if qd.dtype == np.float64 else 4
            self._lse = _device.DeviceBuffer(qd.size // qd.shape[3] * wide)
            if qd.dtype == np.float16:
                self._rest = _device.DeviceBuffer(qd.nbytes)
        rest, lse = (None if b is None else b.ptr for b in (self._rest, self._lse))
        _hip.check(_hip.lib().mg_attention_fwd(self._desc, qb.ptr, kb.ptr, vb.ptr, self._out.ptr, rest, lse))
        out = _device.download(self._out, qd.shape, qd.dtype)
        _device.attach(out, self._out)
        return out

    def _run_backward(self, grad, want):
        arrays = [_device.value_of(t) for t in self.variables]
        q = arrays[0]
        if grad.shape != q.shape:
            raise NotImplementedError(f"attention backward for gradient of shape {grad.shape} (no CPU fallback)")
        if self._lse is None:
            raise RuntimeError("attention kept nothing for a gradient: the graph was not tracked, or q, k and v were constants")
        held = [_device.to_device(a) for a in arrays]
        gb = _device.to_device(grad, q.dtype)
        indices = ({0} if 0 in want else set()) | ({1, 2} if want & {1, 2} else set())
        out = {i: _device.DeviceBuffer(max(arrays[i].nbytes, 16)) for i in indices}
        _hip.check(_hip.lib().mg_attention_bwd(self._desc, *(b.ptr for b in held), self._out.ptr,
                                               None if self._rest is None else self._rest.ptr, self._lse.ptr, gb.ptr,
                                               *(out[i].ptr if i in out else None for i in range(3))))
        return {i: _device.download(out[i], arrays[i].shape, q.dtype) for i in want}

    def backward_var(self, grad, index, **kwargs):
        value = _device.value_of(self.variables[index])
        if _device.value_of(self.variables[0]).size == 0 or value.size == 0:
            return np.zeros(value.shape, dtype=value.dtype)
        # backward() asks for each variable in turn with the same `grad`: the first request computes all that are wanted
        if self._backed is None or self._backed[0] is not grad or index not in self._backed[1]:
            want = {index} | {i for i, var in enumerate(self.variables) if not var.constant}
            self._backed = (grad, self._run_backward(grad, want))
        out = self._backed[1].pop(index)
        if not self._backed[1]:
            self._backed = None
        return out


def attention(q, k, v, *, scale=None, cap=None, slopes=None, mask=None, constant: Optional[bool] = None) -> Tensor:
    """Softmax attention on the GPU::

        scores = scale * q @ k.T;  scores = cap * tanh(scores / cap);  scores -= slopes * |place of query - place of key|
        out = softmax(scores over the keys that `mask` lets a query see) @ v

    ``q:(batch, queries, heads, dim)`` and ``k, v:(batch, keys, key heads, dim)`` in float16, float32 or float64, all
    three alike; ``heads`` is a multiple of ``key heads`` and query head ``h`` reads key head ``h // (heads / key heads)``;
    ``dim`` is at most 256.  These are the axes that ``einsum("btc,chd->bthd", x, w)`` gives.  Sums are carried in float32
    (float64 for float64), the result is rounded once.  A query that sees no key gets zeros and passes no gradient on.
    What a query does not see does not touch its result, infinities and NaN included.

    ``scale`` is ``dim ** -0.5`` unless given; ``cap`` and ``slopes`` (one for each query head, a constant) are left out
    unless given (slopes in float32, float64 for float64); ``mask`` is an :class:`AttentionMask`, none for all keys.

    >>> import numpy as np
    >>> from mygrad_amd.nnet import AttentionMask, attention
    >>> x = np.ones((1, 3, 1, 2))
    >>> attention(x, x, np.arange(6.).reshape(1, 3, 1, 2), mask=AttentionMask(causal=True)).data[0, :, 0]
    array([[0., 1.],
           [1., 2.],
           [2., 3.]])
    """
    return Tensor._op(Attention, q, k, v, op_kwargs=dict(scale=scale, cap=cap, slopes=slopes, mask=mask), constant=constant)


class KeyValueCache:
    """Keys and values of the tokens that a model has seen, on the device, for attention of a few new tokens at a time.

    A step of generation makes one mask, ``AttentionMask(causal=True, lengths=n)`` with the lengths that count the new
    tokens, and each layer's cache takes it twice::

        cache.write(k, v, mask)          # the new tokens go to the places that end at their sequence's length
        out = cache.attend(q, mask=mask)

    Nothing here is recorded in a graph.  A cache starts out with zeros; what lies behind a length is never looked at."""

    def __init__(self, batch, capacity, heads, dim, dtype=np.float32):
        dtype = np.dtype(dtype)
        if dtype not in _DTYPES:
            raise TypeError(f"a cache holds float16, float32 or float64 values, got {dtype}")
        shape = tuple(int(_integers(n, "extents of a cache", (0,))) for n in (batch, capacity, heads, dim))
        if min(shape) < 1 or shape[1] >= _MOST_TOKENS or shape[3] > 256:
            raise ValueError(f"a cache needs a batch, a capacity, heads and a dimension (at most 256) of one or more, got {shape}")
        self._shape, self._dtype = shape, dtype
        nbytes = int(np.prod(shape, dtype=np.int64)) * dtype.itemsize
        self._keys, self._values = _device.DeviceBuffer(nbytes), _device.DeviceBuffer(nbytes)
        for buf in (self._keys, self._values):
            _hip.check(_hip.lib().mg_memset_zero(buf.ptr, nbytes))

    @property
    def shape(self):
        """Batch, capacity, heads and dimension."""
        return self._shape

    @property
    def dtype(self):
        return self._dtype

    @property
    def keys(self):
        """``(batch, capacity, heads, dim)``, on the device; ``.host()`` copies what it holds now."""
        return _device.DeviceArray(self._keys, self._shape, self._dtype)

    @property
    def values(self):
        """Like :attr:`keys`."""
        return _device.DeviceArray(self._values, self._shape, self._dtype)

    def _operand(self, x, name):
        value = _device.value_of(x) if isinstance(x, Tensor) else x if isinstance(x, _device.DeviceArray) else np.asarray(x)
        if value.ndim != 4 or value.shape[0] != self._shape[0] or value.shape[3] != self._shape[3]:
            raise ValueError(f"`{name}` must have shape ({self._shape[0]}, tokens, heads, {self._shape[3]}), got {value.shape}")
        if value.dtype != self._dtype:
            raise TypeError(f"a cache of {self._dtype} takes `{name}` in that dtype, got {value.dtype}")
        return value

    @staticmethod
    def _masked(mask):
        if not isinstance(mask, AttentionMask):
            raise TypeError(f"`mask` must be an AttentionMask, got {type(mask).__name__}")
        if mask._lengths is None:
            raise ValueError("a cache needs the sequences' lengths: AttentionMask(..., lengths=...)")
        return mask

    def write(self, k, v, mask):
        """Puts the tokens of ``k, v:(batch, tokens, heads, dim)`` at the places that end at ``mask.lengths``."""
        kd, vd = self._operand(k, "k"), self._operand(v, "v")
        batch, capacity, heads, dim = self._shape
        if kd.shape != vd.shape or kd.shape[2] != heads:
            raise ValueError(f"k and v must both have {heads} heads and as many tokens, got {kd.shape} and {vd.shape}")
        tokens = kd.shape[1]
        lengths = self._masked(mask)._bind(batch, capacity)[0]
        if mask._shortest < tokens:
            raise ValueError(f"{tokens} tokens do not fit in a length of {mask._shortest}: lengths count the new tokens")
        if tokens == 0:
            return
        kb, vb = _device.to_device(kd), _device.to_device(vd)
        _hip.check(_hip.lib().mg_cache_write(_hip.storage_code(self._dtype), batch, tokens, capacity, heads * dim, lengths.ptr, kb.ptr, vb.ptr,
                                             self._keys.ptr, self._values.ptr))

    def attend(self, q, *, mask, scale=None, cap=None, slopes=None):
        """:func:`attention` of ``q:(batch, queries, query heads, dim)`` over what the cache holds up to ``mask.lengths``; a constant."""
        qd, mask = self._operand(q, "q"), self._masked(mask)
        keys = self.keys
        desc, held = _describe(qd, keys, keys, scale, cap, slopes, mask)
        if desc is None:
            return Tensor(np.zeros(qd.shape, dtype=qd.dtype), constant=True, copy=False)
        qb, out = _device.to_device(qd), _device.DeviceBuffer(qd.nbytes)
        _hip.check(_hip.lib().mg_attention_fwd(desc, qb.ptr, self._keys.ptr, self._values.ptr, out.ptr, None, None))
        return Tensor(_device.DeviceArray(out, qd.shape, qd.dtype), constant=True, copy=False)
