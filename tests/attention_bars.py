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


def over_keys(w, x):
    """sum_j w:(B, H, TQ, TK) x:(B, TK, H, D), as (B, TQ, H, D)."""
    return (w @ x.transpose(0, 2, 1, 3)).transpose(0, 2, 1, 3)


def over_queries(w, x):
    """sum_i w x:(B, TQ, H, D), as (B, TK, H, D)."""
    return (w.transpose(0, 1, 3, 2) @ x.transpose(0, 2, 1, 3)).transpose(0, 2, 1, 3)


class Formulas:
    """out, dq, dk, dv and what they are made of, in 64 bits."""

    def __init__(self, q, k, v, g, seen, *, scale=None, cap=None, slopes=None, lengths=None):
        self.seen, self.cap, self.biased = seen, cap, slopes is not None
        out, self.p, (self.s, bent) = ora.forward(q, k, v, seen, scale=scale, cap=cap, slopes=slopes, lengths=lengths)
        self.q, k, v, self.g = (np.asarray(a, dtype=np.float64) for a in (q, k, v, g))
        self.shape = k.shape
        self.group = q.shape[2] // k.shape[2]
        self.k, self.v = (np.repeat(a, self.group, axis=2) for a in (k, v))
        self.scale = q.shape[3] ** -0.5 if scale is None else scale
        self.bent = 0.0 if bent is None else bent
        self.through = 1 - self.bent * self.bent
        self.dp = self.g.transpose(0, 2, 1, 3) @ self.v.transpose(0, 2, 3, 1)
        self.delta = (self.g * out).sum(-1).transpose(0, 2, 1)[..., None]
        self.ds = self.p * (self.dp - self.delta) * self.through * self.scale
        self.results = [out, over_keys(self.ds, self.k), self.shared(over_queries(self.ds, self.q)), self.shared(over_queries(self.p, self.g))]

    def by_head(self, a):
        """dk or dv of each query head, as (B, TK, HK, group, D)."""
        B, TK, HK, D = self.shape
        return a.reshape(B, TK, HK, self.group, D)

    def shared(self, a):
        return self.by_head(a).sum(3)


def bars_of(dtype, f):
    """Largest differences to be expected of `f.results`."""
    u, r = UNIT[dtype]
    half = dtype == np.float16
    w = 2.0**-22 if half else 0.0
    (TQ, _, D), TK = f.q.shape[1:], f.shape[1]
    terms = TQ * f.group
    out, dq, dk, dv = f.results
    scale = abs(f.scale)
    nq, nk, nv, ng, no = (_norms(a).transpose(0, 2, 1) for a in (f.q, f.k, f.v, f.g, out))

    plain = scale * nq[..., None] * nk[:, :, None]
    of_s, of_through = (D + 8) * u * plain, 4 * u
    if f.cap:
        of_t = f.through * of_s / f.cap + (of_s / f.cap) ** 2 + 4 * u + (2.0**-19 * np.abs(f.bent) + 2.0**-22 if half else 0)
        of_s, of_through = f.cap * of_t, 2 * np.abs(f.bent) * of_t + of_t**2 + 4 * u
    far = np.abs(np.where(f.seen[:, None], f.s, 0.0))
    of_s = of_s + 8 * u * (plain + (f.cap or 0.0) + far * (2 if f.biased else 1))
    of_p = f.p * (of_s + (f.p * of_s).sum(-1, keepdims=True) + (TK + 32) * u + w) + (2.0**-31 * (f.p > 0) if half else 0.0)
    before = over_keys(of_p, np.abs(f.v))  # out's rounding

    of_dp = (D + 8) * u * ng[..., None] * nv[:, :, None]
    kept = before + (2.0**-21 if half else 2 * u) * np.abs(out)
    of_delta = (D + 8) * u * (ng * no)[..., None] + (np.abs(f.g) * kept).sum(-1).transpose(0, 2, 1)[..., None]
    apart = np.abs(f.dp - f.delta)
    ds = np.abs(f.ds)
    of_ds = scale * (of_p * apart * f.through + f.p * (of_dp + of_delta + 2 * u * (np.abs(f.dp) + np.abs(f.delta))) * f.through
                     + f.p * apart * of_through) + w * ds
    if half:
        of_ds = of_ds + 2.0**-31 * ds.max((2, 3), initial=0.0, keepdims=True) * (f.p > 0)
    ends = lambda a, value: a + 1.01 * r * (np.abs(value) + a) + SMALLEST[dtype]
    return [ends(before, out), ends(over_keys(of_ds + (TK + 8) * u * ds, np.abs(f.k)), dq),
            ends(f.shared(over_queries(of_ds + (terms + 8) * u * ds, np.abs(f.q))), dk),
            ends(f.shared(over_queries(of_p + (terms + 8) * u * f.p, np.abs(f.g))), dv)]


def formulas_and_bars(dtype, q, k, v, g, seen, **how):
    """[(value, bar)] of out, dq, dk and dv."""
    f = Formulas(q, k, v, g, seen, **how)
    return list(zip(f.results, bars_of(dtype, f)))


def _case(dtype, B, TQ, TK, HQ, HK, D, mask=None, cap=None, bias=False, scale=None, grad_scale=1.0):
    return dict(dtype=dtype, shape=(B, TQ, TK, HQ, HK, D), mask=mask or {}, cap=cap, bias=bias, scale=scale, grad_scale=grad_scale)


_DOCUMENTS = np.repeat([4, 0, -1, 2], [60, 1, 19, 70])

# Each way to compute the three passes: rows, 32 columns a block with keys split or not, 128 queries a block; dk and dv in one piece and in cuts.
CASES = [
    *(_case(dtype, *shape, **how) for dtype in (np.float16, np.float32) for shape, how in (
        ((2, 90, 90, 4, 2, 64), dict(cap=0.05, scale=3.0)), ((2, 90, 90, 4, 2, 64), dict(cap=3.0, bias=True, scale=0.4, mask=dict(causal=True, prefix=40))),
        ((1, 3, 5003, 2, 1, 64), dict(mask=dict(causal=True))), ((2, 130, 257, 2, 1, 128), dict()), ((1, 9, 900, 2, 2, 252), dict()),
        ((1, 300, 300, 2, 2, 256), dict()), ((5, 150, 150, 14, 2, 36), dict()), ((9, 150, 150, 16, 4, 64), dict(mask=dict(causal=True))),
        ((9, 150, 150, 16, 16, 96), dict(mask=dict(documents=_DOCUMENTS), cap=4.0)), ((9, 130, 160, 16, 2, 128), dict(mask=dict(causal=True, window=50))),
        ((9, 150, 150, 16, 8, 72), dict(mask=dict(causal=True, documents=_DOCUMENTS), bias=True)), ((1, 700, 700, 4, 1, 80), dict(mask=dict(causal=True))),
        ((3, 33, 70, 6, 2, 34), dict(mask=dict(lengths=[70, 20, 0]))), ((1, 300, 300, 2, 2, 64), dict(mask=dict(causal=True), grad_scale=1e-4)))),
    _case(np.float64, 2, 90, 90, 4, 2, 20, cap=3.0, bias=True, mask=dict(causal=True, prefix=40)), _case(np.float64, 2, 65, 130, 3, 1, 72),
]


_MASKS = [dict(), dict(causal=True), dict(causal=True, window=37), dict(window=20), dict(causal=True, window=1), dict(causal=True, prefix=50),
          dict(causal=True, prefix=[0, 111]), dict(lengths=[130, 0]), dict(causal=True, lengths=[33, 97]), dict(documents=_DOCUMENTS[:130]),
          dict(causal=True, documents=np.stack([_DOCUMENTS[:130], _DOCUMENTS[20:]])), dict(causal=True, window=16, documents=_DOCUMENTS[:130]),
          dict(causal=True, prefix=20, documents=_DOCUMENTS[:130]), dict(causal=True, lengths=[100, 64], documents=_DOCUMENTS[:130])]
# Each mask in 32 columns a block, and in 128 queries a block.
CASES += [_case(dtype, 2, 130, 130, *heads, 32, mask=mask) for dtype in (np.float16, np.float32) for mask in _MASKS for heads in ((2, 1), (66, 22))]


def name_of(case):
    shape, rest = "x".join(map(str, case["shape"])), [k for k in ("cap", "bias", "scale") if case[k]] + list(case["mask"])
    rest += [str(v) for k, v in case["mask"].items() if k == "window"]
    return "-".join([np.dtype(case["dtype"]).name, shape, *rest, *(["small"] if case["grad_scale"] != 1 else [])])


def operands(case):
    """q, k, v, grad; which keys each query sees; the rest of the arguments, lengths among them."""
    B, TQ, TK, HQ, HK, D = case["shape"]
    rng = np.random.default_rng(list(case["shape"]))
    q, k, v, g = (rng.standard_normal(shape) for shape in ((B, TQ, HQ, D), (B, TK, HK, D), (B, TK, HK, D), (B, TQ, HQ, D)))
    slopes = (2.0 ** -np.arange(1, HQ + 1)).astype(np.float32) if case["bias"] else None
    arrays = [a.astype(case["dtype"]) for a in (q, k, v, g * case["grad_scale"])]
    return arrays, ora.visible(B, TQ, TK, **case["mask"]), dict(scale=case["scale"], cap=case["cap"], slopes=slopes, lengths=case["mask"].get("lengths"))
