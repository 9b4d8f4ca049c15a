"""Attention, its gradient and the norm of heads with rotary positions in 64 bits, from their formulas (tests only).

Shapes as in the package: q:(B, TQ, HQ, D), k and v:(B, TK, HK, D)."""

import numpy as np


def visible(B, TQ, TK, causal=False, window=None, prefix=None, documents=None, lengths=None):
    """seen[b, i, j], pair by pair as the mask's description has it."""
    seen = np.zeros((B, TQ, TK), dtype=bool)
    each = lambda v, b: v if np.ndim(v) == 0 else v[b]
    for b in range(B):
        n = TK if lengths is None else int(each(lengths, b))
        ids = None if documents is None else np.broadcast_to(documents, (B, TK))[b]
        for i in range(TQ):
            place = i + n - TQ
            if ids is not None and (not 0 <= place < n or ids[place] < 0):
                continue
            first = 0 if ids is None else int(np.flatnonzero(ids == ids[place])[0])
            for j in range(n):
                if ids is not None and ids[j] != ids[place]:
                    continue
                ok = not causal or j <= place
                if window is not None:
                    ok = ok and j > place - window and (causal or j < place + window)
                if prefix is not None:
                    ok = ok or j < first + int(each(prefix, b))
                seen[b, i, j] = ok
    return seen


def _scores(q, k, scale, cap, slopes, lengths):
    B, TQ, HQ, D = q.shape
    TK, HK = k.shape[1:3]
    k = np.repeat(k, HQ // HK, axis=2)
    s = np.einsum("bihd,bjhd->bhij", q, k) * scale
    bent = None
    if cap:
        bent = np.tanh(s / cap)
        s = cap * bent
    if slopes is not None:
        n = np.broadcast_to(TK if lengths is None else np.asarray(lengths), (B,))
        place = np.arange(TQ)[None] + n[:, None] - TQ
        s = s - np.asarray(slopes, dtype=np.float64)[None, :, None, None] * np.abs(place[:, None, :, None] - np.arange(TK))
    return s, bent


def forward(q, k, v, seen, *, scale=None, cap=None, slopes=None, lengths=None):
    """out, the weights P:(B, HQ, TQ, TK) and the scores behind the cap and the bias; products of what is not seen are left out
    whatever it holds."""
    q, k, v = (np.asarray(a, dtype=np.float64) for a in (q, k, v))
    group = q.shape[2] // k.shape[2]
    scale = q.shape[3] ** -0.5 if scale is None else scale
    with np.errstate(all="ignore"):
        s, bent = _scores(q, k, scale, cap, slopes, lengths)
    s = np.where(seen[:, None], s, -np.inf)
    top = s.max(-1, initial=-np.inf, keepdims=True)
    e = np.where(seen[:, None], np.exp(s - np.where(top == -np.inf, 0, top)), 0.0)
    total = e.sum(-1, keepdims=True)
    p = e / np.where(total > 0, total, 1)
    vr = np.repeat(v, group, axis=2)
    if np.isfinite(v).all():
        out = np.einsum("bhij,bjhd->bihd", p, vr)
    else:
        out = np.zeros(q.shape)
        for b, i, j in zip(*np.nonzero(seen)):
            out[b, i] += p[b, :, i, j, None] * vr[b, j]
    return out, p, (s, bent)


def backward(q, k, v, g, seen, *, scale=None, cap=None, slopes=None, lengths=None):
    """dq, dk, dv."""
    q, k, v, g = (np.asarray(a, dtype=np.float64) for a in (q, k, v, g))
    B, TK, HK, D = k.shape
    group = q.shape[2] // HK
    scale = D ** -0.5 if scale is None else scale
    out, p, (_, bent) = forward(q, k, v, seen, scale=scale, cap=cap, slopes=slopes, lengths=lengths)
    kr, vr = (np.repeat(a, group, axis=2) for a in (k, v))
    dp = np.einsum("bihd,bjhd->bhij", g, vr)
    ds = p * (dp - np.einsum("bihd,bihd->bhi", g, out)[..., None])
    if bent is not None:
        ds = ds * (1 - bent * bent)
    ds *= scale
    shared = lambda a: a.reshape(B, TK, HK, group, D).sum(3)
    return (np.einsum("bhij,bjhd->bihd", ds, kr), shared(np.einsum("bhij,bihd->bjhd", ds, q)), shared(np.einsum("bhij,bihd->bjhd", p, g)))


def angles(sections, positions, base=10000.0):
    """Angles of all pairs at positions:(..., axes)."""
    return np.concatenate([np.asarray(positions, dtype=np.float64)[..., a, None] * float(base) ** (-np.arange(n) / max(n, 1))
                           for a, n in enumerate(sections)], -1)


def _turn(z, angle, interleaved):
    """angle:(..., 1, pairs) against z:(..., heads, D)."""
    pairs = angle.shape[-1]
    first, second = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else (slice(0, pairs), slice(pairs, 2 * pairs))
    out = z.copy()
    turned = (z[..., first] + 1j * z[..., second]) * np.exp(1j * angle)
    out[..., first], out[..., second] = turned.real, turned.imag
    return out


def head_norm(x, w, eps, angle=None, interleaved=False):
    """``eps`` None: no norm; ``w`` None: no weight; ``angle``:(..., pairs) or None."""
    x = np.asarray(x, dtype=np.float64)
    z = x if eps is None else x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    z = z if w is None else z * np.asarray(w, dtype=np.float64)
    return z if angle is None else _turn(z, angle[..., None, :], interleaved)


def head_norm_backward(x, w, eps, g, angle=None, interleaved=False):
    """dx, dw (None without a weight)."""
    x, u = np.asarray(x, dtype=np.float64), np.asarray(g, dtype=np.float64)
    if angle is not None:
        u = _turn(u, -angle[..., None, :], interleaved)
    r = 1.0 if eps is None else 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    dw = None
    if w is not None:
        w = np.asarray(w, dtype=np.float64)
        over = tuple(range(x.ndim - w.ndim))
        dw = (u * x * r).sum(over)
        u = u * w
    return (u if eps is None else r * (u - x * r * r * (u * x).mean(-1, keepdims=True))), dw
