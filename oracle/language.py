"""A language model's ends and the norm between its blocks in 64 bits and more (what NumPy has: 80 on x86, so that float64 has
something to be held to), from their formulas (tests only)."""

import numpy as np

WIDE = np.longdouble


def layer_norm(x, w=None, b=None, eps=0.0, g=None):
    """y, and with ``g`` dx, dw, db; rows are the last axis."""
    x = np.asarray(x, WIDE)
    w = np.ones(x.shape[-1]) if w is None else np.asarray(w, WIDE)
    middle = x - x.mean(-1, keepdims=True)
    r = 1 / np.sqrt((middle**2).mean(-1, keepdims=True) + eps)
    n = middle * r
    y = n * w + (0 if b is None else np.asarray(b, WIDE))
    if g is None:
        return y
    g = np.asarray(g, WIDE)
    u = g * w
    dx = r * (u - u.mean(-1, keepdims=True) - n * (u * n).mean(-1, keepdims=True))
    rows = tuple(range(x.ndim - 1))
    return y, dx, (g * n).sum(rows), g.sum(rows)


def embedding(weight, ids, scale=1.0, g=None):
    """y, and with ``g`` the gradient of ``weight``."""
    weight, ids = np.asarray(weight, WIDE), np.asarray(ids)
    y = np.where((ids >= 0)[..., None], weight[np.maximum(ids, 0)] if weight.shape[0] else 0.0, 0.0) * scale
    if g is None:
        return y
    dw = np.zeros_like(weight)
    for token, row in zip(ids.ravel(), np.asarray(g, WIDE).reshape(ids.size, -1)):
        if token >= 0:
            dw[token] += row * scale
    return y, dw


def softmax_row(z, per=1.0):
    """t = (z - max) * per, p = softmax and log s (minus infinity for a row that is ruled out throughout, whose p are zeros)."""
    z = np.asarray(z, WIDE)
    m = z.max(-1, keepdims=True)
    t = (z - np.where(m == -np.inf, 0, m)) * per
    e = np.exp(t)
    s = e.sum(-1, keepdims=True)
    with np.errstate(divide="ignore"):
        return t, e / np.where(s == 0, 1, s), np.log(s)


def log_probabilities(z, ids=None, g=None, h=None):
    """Log probabilities and entropies of rows ``z:(rows, V)``, and the gradient of z by ``g`` of the one and ``h`` of the other."""
    t, p, log_s = softmax_row(z)
    bounded = np.where(p > 0, t, 0)
    a = (p * bounded).sum(-1, keepdims=True)
    nothing = np.isneginf(log_s[:, 0])
    ids = np.full(len(t), -1) if ids is None else np.asarray(ids)
    at = np.arange(len(t)), np.maximum(ids, 0)
    with np.errstate(invalid="ignore"):
        scores = np.where(ids < 0, 0, np.where(nothing, -np.inf, t[at] - log_s[:, 0]))
        entropy = np.where(nothing, 0, log_s[:, 0] - a[:, 0])
    dz = np.zeros_like(t)
    if g is not None:
        g = np.where(ids < 0, 0, np.asarray(g, WIDE))[:, None]
        dz -= p * g
        dz[at] += g[:, 0]
    if h is not None:
        dz -= p * (bounded - a) * np.asarray(h, WIDE)[:, None]
    dz[nothing] = 0
    return scores, entropy, dz


def likeliest(z, count):
    """Places of the largest values of each row, the lowest first among equals."""
    return np.argsort(-np.asarray(z, WIDE), axis=-1, kind="stable")[..., :count]


def distillation(z, ids, teacher, temperature=1.0, g=None):
    """A loss for each row, and with ``g`` the gradient of ``z``."""
    ids, per = np.asarray(ids), 1 / temperature
    t, p, log_s = softmax_row(z, per)
    u, q, log_total = softmax_row(np.where(ids < 0, -np.inf, np.asarray(teacher, WIDE)), per)
    nothing = np.isneginf(log_s)
    taught = np.take_along_axis(t, np.maximum(ids, 0), 1)
    with np.errstate(invalid="ignore"):
        log_p = np.where(nothing, -np.inf, taught - log_s)
        terms = np.where(q > 0, q * (u - log_total - log_p), 0)
    loss = terms.sum(-1)
    if g is None:
        return loss
    dz = p * (q.sum(-1, keepdims=True) > 0)
    for k in range(ids.shape[1]):
        dz[np.arange(len(ids)), np.maximum(ids[:, k], 0)] -= q[:, k]
    dz *= np.asarray(g, WIDE)[:, None] * per
    dz[nothing[:, 0]] = 0
    return loss, dz
