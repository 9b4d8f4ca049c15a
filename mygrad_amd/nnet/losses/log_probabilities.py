"""Log probabilities of tokens on the MI355X, with entropies and the likeliest alternatives.  Where the reference has losses of
a batch of classes (``mygrad/nnet/losses/softmax_crossentropy.py``), this gives each token's own value; the operation keeps its
``Operation`` contract (``mygrad/operation_base.py:54-228``)."""

from math import prod
from numbers import Integral
from typing import Optional

import numpy as np

from ... import _device, _hip
from ...operation_base import Operation
from ...tensor_base import Tensor
from ..layers.embedding import TokenIds, as_tokens

__all__ = ["LogProbabilities", "log_probabilities"]

_DTYPES = (np.float16, np.float32, np.float64)
_MOST_TOP = 128


def result_type(dtype):
    """What values of a row come in: those of float16 logits are not rounded to its eleven bits."""
    return np.dtype(np.float64 if dtype == np.float64 else np.float32)


class _Plan:
    """The checked arguments of calls of one kind, and their launch."""

    def __init__(self, z, lead, entropy, top):
        """``lead``: the shape of the tokens, None without them."""
        if z.ndim < 1:
            raise ValueError(f"`logits` must have the axes (..., vocabulary), got shape {z.shape}")
        if z.dtype not in _DTYPES:
            raise TypeError(f"log_probabilities runs on the GPU in float16, float32 or float64, got {z.dtype} (there is no CPU fallback)")
        if z.shape[-1] == 0:
            raise ValueError("there are no tokens in the vocabulary")
        if not isinstance(entropy, (bool, np.bool_)):
            raise TypeError(f"`entropy` must be a boolean value, got: {entropy}")
        if not isinstance(top, Integral) or isinstance(top, (bool, np.bool_)) or not 0 <= top <= min(_MOST_TOP, z.shape[-1]):
            raise ValueError(f"`top` must be a whole number up to {_MOST_TOP} and to the vocabulary of {z.shape[-1]}, got {top}")
        if lead is None and not entropy and not top:
            raise TypeError("log_probabilities without tokens, entropies or alternatives has nothing to compute")
        if lead is not None and lead != z.shape[:-1]:
            raise ValueError(f"tokens of shape {lead} for logits of shape {z.shape}")
        self.lead, self.rows, self.vocabulary = z.shape[:-1], prod(z.shape[:-1]), z.shape[-1]
        self.tokens, self.entropy, self.top, self.empty = lead is not None, bool(entropy), int(top), z.size == 0
        self.code, self.dtype = _hip.storage_code(z.dtype), result_type(z.dtype)
        self.shape = (2, *self.lead) if entropy and self.tokens else self.lead  # of what has a gradient
        self.nbytes = prod(self.shape) * self.dtype.itemsize
        self.kept_bytes = 3 * self.rows * self.dtype.itemsize
        self.alternatives = (*self.lead, self.top)

    def planes(self, ptr):
        """Where log probabilities and entropies (or their gradients) lie."""
        if not self.tokens:
            return None, ptr
        return ptr, ptr + self.nbytes // 2 if self.entropy else None

    def no_alternatives(self):
        return np.empty(self.alternatives, dtype=self.dtype), np.empty(self.alternatives, dtype=np.int32)

    def run(self, z, ids, keep):
        """The memory of the values that have a gradient (and, if it is to follow, of what it needs behind them), and the likeliest tokens."""
        out = _device.DeviceBuffer(self.nbytes + (self.kept_bytes if keep else 0)) if self.tokens or self.entropy else None
        kept = out.ptr + self.nbytes if keep else None  # behind the result
        top = ()
        if self.top:
            count = self.rows * self.top
            top = (_device.DeviceArray(_device.DeviceBuffer(count * self.dtype.itemsize), self.alternatives, self.dtype),
                   _device.DeviceArray(_device.DeviceBuffer(count * 4), self.alternatives, np.int32))
        zb = _device.to_device(z)  # until the launch
        _hip.check(_hip.lib().mg_log_probabilities_fwd(self.code, self.rows, self.vocabulary, self.top, ids, zb.ptr,
                                                       *((None, None) if out is None else self.planes(out.ptr)), kept,
                                                       *((top[0].buf.ptr, top[1].buf.ptr) if top else (None, None))))
        return out, top


_plans = {}
_MOST_PLANS = 64


def _plan(z, tokens, entropy, top):
    """The plan of a call, whose tokens fit its vocabulary."""
    key = z.shape, z.dtype, None if tokens is None else tokens.shape, entropy, top, type(entropy), type(top)
    plan = _plans.get(key)
    if plan is None:
        plan = _Plan(z, key[2], entropy, top)
        if len(_plans) >= _MOST_PLANS:
            _plans.clear()
        _plans[key] = plan
    if tokens is not None:
        as_tokens(tokens, plan.vocabulary)
    return plan


class LogProbabilities(Operation):
    """``logits:(..., vocabulary)``."""

    takes_device_arrays = True

    def __call__(self, logits, *, tokens, entropy, top, alternatives):
        """``tokens``: TokenIds or None; ``alternatives``: a list that receives the likeliest tokens and their log probabilities."""
        self.variables = (logits,)
        z = _device.value_of(logits)
        plan = self._plan = _plan(z, tokens, entropy, top)
        self._tokens = tokens
        if plan.empty:
            alternatives += plan.no_alternatives()
            return np.empty(plan.shape, dtype=plan.dtype)
        out, found = plan.run(z, None if tokens is None else tokens._buffer().ptr, not logits.constant)
        self._kept = None if logits.constant else out
        alternatives += found
        y = _device.download(out, plan.shape, plan.dtype)
        _device.attach(y, out)
        return y

    def backward_var(self, grad, index, **kwargs):
        plan, z = self._plan, _device.value_of(self.variables[index])
        if plan.empty:
            return np.zeros(z.shape, dtype=z.dtype)
        if grad.shape != plan.shape:
            raise NotImplementedError(f"log_probabilities backward for gradient of shape {grad.shape} (no CPU fallback)")
        zb, gb = _device.to_device(z), _device.to_device(grad, plan.dtype)
        out = _device.DeviceBuffer(z.nbytes)
        ids = None if self._tokens is None else self._tokens._buffer().ptr
        _hip.check(_hip.lib().mg_log_probabilities_bwd(plan.code, plan.rows, plan.vocabulary, ids, zb.ptr, self._kept.ptr + plan.nbytes,
                                                       *plan.planes(gb.ptr), out.ptr))
        return _device.download(out, z.shape, z.dtype)


def log_probabilities(logits, tokens=None, *, entropy: bool = False, top: int = 0, constant: Optional[bool] = None):
    """What ``logits:(..., vocabulary)`` say of their tokens, in one pass over them on the GPU::

        log_probability = log(softmax(logits))[token]
        entropy = -sum(softmax(logits) * log(softmax(logits)))

    Parameters
    ----------
    logits : ArrayLike, shape=(..., vocabulary)
        float16, float32 or float64.  Minus infinity rules a token out.
    tokens : Optional[ArrayLike], shape=(...)
        Whole numbers below ``vocabulary``, or :class:`~mygrad_amd.nnet.TokenIds`.  -1 stands for no token: its log
        probability is 0 and has no gradient, whatever the logits hold.
    entropy : bool
        Whether the entropies are wanted, too.
    top : int
        How many of the likeliest tokens are wanted (at most 128).
    constant : Optional[bool]
        If True, the returned tensor is a constant.

    Returns
    -------
    Tensor
        The log probabilities, of the logits' leading shape; with ``entropy`` of shape ``(2, ...)``, the log probabilities
        and the entropies, and without tokens the entropies alone.  They are float32 (float64 for float64 logits) and have a
        gradient.  A row whose logits are all minus infinity has log probabilities of minus infinity, an entropy of 0 and
        gradients of zero; infinity or NaN among its logits makes a row's results NaN.

    With ``top``, a tuple of that (None without tokens and entropies) and of the likeliest alternatives: their log probabilities
    ``(..., top)``, a constant, in falling order, and their :class:`~mygrad_amd.nnet.TokenIds`, the lowest one first among equals.

    >>> import mygrad_amd as mg
    >>> from mygrad_amd.nnet import log_probabilities
    >>> logits = mg.Tensor([[0.0, 1.0, 3.0, 2.0], [0.0, 0.0, 0.0, 0.0]])
    >>> log_probabilities(logits, [2, 1]).data.round(3)
    array([-0.44 , -1.386])
    >>> scores, likeliest, which = log_probabilities(logits, [2, 1], entropy=True, top=2)
    >>> scores.data.round(3)
    array([[-0.44 , -1.386],
           [ 0.948,  1.386]])
    >>> which.data
    array([[2, 3],
           [0, 1]], dtype=int32)
    """
    alternatives = []
    if tokens is not None and not isinstance(tokens, TokenIds):
        tokens = TokenIds(tokens)
    if tokens is not None or entropy or not top:
        out = Tensor._op(LogProbabilities, logits, op_kwargs=dict(tokens=tokens, entropy=entropy, top=top, alternatives=alternatives), constant=constant)
        if not top:
            return out
    else:  # nothing that has a gradient
        if constant is not None and not isinstance(constant, bool):
            raise TypeError(f"`constant` must be a boolean value, got: {constant}")
        z = _device.value_of(logits if isinstance(logits, Tensor) else Tensor(logits, constant=True, copy=False))
        plan, out = _plan(z, None, entropy, top), None
        alternatives += plan.no_alternatives() if plan.empty else plan.run(z, None, False)[1]
    likeliest, which = alternatives
    which = TokenIds._on_device(which, np.shape(logits)[-1]) if isinstance(which, _device.DeviceArray) else TokenIds(which)
    return out, Tensor(likeliest, constant=True, copy=False), which
