"""How far attention and its gradients may be from their formulas, element by element (tests only).

u is the unit of the sums (2^-24, 2^-53 for float64), r that of the type of the results (2^-11 for float16, else u), w what the operands of
the second products keep: float16 multiplies weights and gradients of scores in two parts of it (2^-22), the other types as they are.
With |q_i| and the like for norms of rows, and each sum of n terms off by n u of the terms' magnitudes:

    x = scale q.k            (D + 8) u scale |q_i| |k_j|
    s                        (1 - t^2) of that behind a cap (t the tangent), 8 u of the largest value on its way, and in float16 2^-19
                             of the tangent's own
    P                        of itself: that of s, their mean over the row, (n + 32) u and w; and in float16 2^-31, below which it has no parts
    out                      sum P |v| of those, and r
    dP                       (D + 8) u |g_i| |v_j|
    D_i = g_i . out_i        (D + 8) u |g_i| |out_i|, and sum |g| of out's before it is rounded (float16 keeps 22 bits of it)
    dS = P (dP - D) (1 - t^2) scale
                             its factors' errors times the others, w of itself, and in float16 2^-31 of the head's largest
    dq, dk, dv               the sums of those over keys, or queries and heads, and r
"""

import numpy as np

from oracle import attention as ora

UNIT = {np.float16: (2.0**-24, 2.0**-11), np.float32: (2.0**-24, 2.0**-24), np.float64: (2.0**-53, 2.0**-53)}
SMALLEST = {np.float16: 2.0**-24, np.float32: 2.0**-126, np.float64: 2.0**-1022}


def _norms(a):
    return np.sqrt((a * a).sum(-1))


def formulas_and_bars(dtype, q, k, v, g, seen, *, scale=None, cap=None, slopes=None, lengths=None):
    """[(value, bar)] of out, dq, dk and dv in 64 bits."""
    u, r = UNIT[dtype]
    half = dtype == np.float16
    w = 2.0**-22 if half else 0.0
    how = dict(scale=scale, cap=cap, slopes=slopes, lengths=lengths)
    out, p, (s, bent) = ora.forward(q, k, v, seen, **how)
    grads = ora.backward(q, k, v, g, seen, **how)
    scale = q.shape[3] ** -0.5 if scale is None else abs(scale)
    q, k, v, g = (np.asarray(a, dtype=np.float64) for a in (q, k, v, g))
    (B, TQ, HQ, D), (TK, HK) = q.shape, k.shape[1:3]
    group = HQ // HK
    kr, vr = (np.repeat(a, group, axis=2) for a in (k, v))
    by_head = lambda a: a.transpose(0, 2, 1)  # (B, T, H) norms as (B, H, T)
    nq, nk, nv, ng, no = (by_head(_norms(a)) for a in (q, kr, vr, g, out))

    plain = scale * nq[..., None] * nk[:, :, None]
    of_x = (D + 8) * u * plain
    through, of_through = 1.0, 4 * u
    of_s = of_x
    if cap:
        through = 1 - bent * bent
        of_t = through * of_x / cap + (of_x / cap) ** 2 + 4 * u + (2.0**-19 * np.abs(bent) + 2.0**-22 if half else 0)
        of_s, of_through = cap * of_t, 2 * np.abs(bent) * of_t + of_t**2 + 4 * u
    far = np.where(seen[:, None], np.abs(np.where(seen[:, None], s, 0.0)), 0.0)
    of_s = of_s + 8 * u * (plain + (cap or 0.0) + far * (1 if slopes is None else 2))
    of_p = p * (of_s + (p * of_s).sum(-1, keepdims=True) + (TK + 32) * u + w) + (2.0**-31 * (p > 0) if half else 0.0)
    before = np.einsum("bhij,bjhd->bihd", of_p, np.abs(vr))
    bars = [before + 1.01 * r * (np.abs(out) + before) + SMALLEST[dtype]]

    dp = np.einsum("bihd,bjhd->bhij", g, vr)
    delta = np.einsum("bihd,bihd->bhi", g, out)[..., None]
    of_dp = (D + 8) * u * ng[..., None] * nv[:, :, None]
    kept = before + (2.0**-21 if half else 2 * u) * np.abs(out)
    of_delta = (D + 8) * u * (ng * no)[..., None] + np.einsum("bihd,bihd->bhi", np.abs(g), kept)[..., None]
    apart = np.abs(dp - delta)
    ds = p * apart * through * scale
    of_ds = scale * (of_p * apart * through + p * (of_dp + of_delta + 2 * u * (np.abs(dp) + np.abs(delta))) * through + p * apart * of_through) + w * ds
    if half:
        of_ds = of_ds + 2.0**-31 * ds.max((2, 3), initial=0.0, keepdims=True) * (p > 0)
    shared = lambda a: a.reshape(B, TK, HK, group, D).sum(3)
    ends = lambda a, value: a + 1.01 * r * (np.abs(value) + a) + SMALLEST[dtype]
    bars.append(ends(np.einsum("bhij,bjhd->bihd", of_ds + (TK + 8) * u * ds, np.abs(kr)), grads[0]))
    bars.append(ends(shared(np.einsum("bhij,bihd->bjhd", of_ds + (TQ * group + 8) * u * ds, np.abs(q))), grads[1]))
    bars.append(ends(shared(np.einsum("bhij,bihd->bjhd", of_p + (TQ * group + 8) * u * p, np.abs(g))), grads[2]))
    return list(zip((out, *grads), bars))
