"""What is timed of attention and its neighbours: ``head_norm`` (a norm for each head with rotary positions in the same
pass), ``attention`` (scores with a cap, a bias by distance, masks) and ``KeyValueCache`` (a few tokens against a long cache).

Where ``own`` is true a pass makes the package's calls on tensors that live on the device, and hands results back as torch
tensors over the same memory; where it is false it is the same arithmetic in elementary torch operations in 32 bits."""

import math

import numpy as np
import torch

own = False

_TORCH = {"f16": torch.float16, "f32": torch.float32}
_BYTES = {"f16": 2, "f32": 4}
_EPS = 1e-6
_BASE = 10000.0


# ----------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # a training step of a small model on short sequences: launches and the host side count
        _attention("attention-small-f32", "f32", 2, 77, 77, 4, 4, 32, mask="causal"),
        # the bulk of a language model's training: causal, shared key heads, capped scores
        _attention("attention-causal-f16", "f16", 4, 2048, 2048, 16, 4, 128, mask="causal", cap=50.0),
        # long sequences that are packed from documents; the largest pass
        _attention("attention-documents-f16", "f16", 1, 8192, 8192, 16, 16, 128, mask="documents", parts=5),
        # single precision with a bias by distance behind a prefix that every token sees (a captioned image)
        _attention("attention-prefix-f32", "f32", 4, 1024, 1024, 8, 8, 64, mask="prefix", parts=256, bias=True),
        # image tokens that look at a ragged number of others; a head dimension that fills no tile
        _attention("attention-cross-ragged-f16", "f16", 3, 1531, 997, 12, 12, 72),
        # queries of a language model of middle size: one axis of positions
        _norm("norm-text-f16", "f16", 4, (4096,), 32, 128),
        # video patches: time, height and width in single precision; a last axis that is odd
        _norm("norm-video-f32", "f32", 2, (8, 27, 33), 16, 72),
        # one new token of each request in a batch: nothing but latency
        _norm("norm-token-f16", "f16", 8, (1,), 8, 64, train=False),
        # one request, a short history: latency
        _cache("cache-small-f16", "f16", 1, 1, 512, 300, 8, 2, 64),
        # a full batch with histories of mixed lengths: bandwidth
        _cache("cache-batch-f16", "f16", 32, 1, 8192, 8000, 32, 8, 128),
        # one request with a long history: the work has to be split along it
        _cache("cache-long-f16", "f16", 1, 1, 131072, 131001, 32, 8, 128, cap=30.0),
        # several drafted tokens at once in single precision, with a bias by distance
        _cache("cache-drafted-f32", "f32", 6, 5, 2048, 1999, 12, 4, 96, bias=True),
    ]


def _attention(name, dtype, b, t, keys, heads, kv_heads, dim, mask="none", parts=0, cap=0.0, bias=False):
    """``parts``: keys of the prefix, number of documents, or keys in the window."""
    return {"name": name, "kind": "attention", "dtype": dtype, "b": b, "t": t, "keys": keys, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "mask": mask, "parts": parts, "cap": cap, "bias": bias}


def _norm(name, dtype, b, grid, heads, dim, train=True):
    case = {"name": name, "kind": "norm", "dtype": dtype, "b": b, "heads": heads, "dim": dim, "axes": len(grid), "train": train}
    return dict(case, **{"grid%d" % a: n for a, n in enumerate(grid)})


def _cache(name, dtype, b, t, capacity, length, heads, kv_heads, dim, cap=0.0, bias=False):
    """Histories are ``length // 2`` to ``length`` tokens long, the ``t`` new ones among them."""
    return {"name": name, "kind": "cache", "dtype": dtype, "b": b, "t": t, "capacity": capacity, "length": length, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "cap": cap, "bias": bias}


def _spread(rng, low, high):
    """A whole number whose logarithm is spread evenly; no length of 3072."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return n - 1 if n == 3072 else n


def draw(rng):
    kind = rng.choice(("attention", "attention", "norm", "cache"))
    dtype, dim = rng.choice(("f16", "f16", "f32")), rng.choice((32, 64, 64, 72, 80, 96, 128, 128))
    kv_heads, group = rng.choice((1, 2, 3, 4, 8)), rng.choice((1, 1, 2, 3, 4, 8))
    heads = kv_heads * group
    if kind == "norm":
        axes = rng.choice((1, 1, 2, 3))
        heads = min(heads, 32)
        t = _spread(rng, 1, 16384)
        if axes == 1:
            grid = (t,)
        elif axes == 2:
            grid = (max(1, int(t ** 0.5)), max(1, int(t ** 0.5)) + rng.randrange(3))
        else:
            side = max(1, int(t ** (1 / 3)))
            grid = (side + rng.randrange(2), side, side + rng.randrange(3))
        b = max(1, min(rng.choice((1, 2, 4, 8)), (1 << 26) // (math.prod(grid) * heads * dim)))
        case = _norm("", dtype, b, grid, heads, dim, train=rng.random() < 0.75)
    elif kind == "cache":
        length = _spread(rng, 1, 131072)
        heads, kv_heads = min(heads, 32), min(kv_heads, 32)
        if heads % kv_heads:
            heads = kv_heads
        b = max(1, min(_spread(rng, 1, 48), (1 << 27) // (length * kv_heads * dim)))
        t = min(rng.choice((1, 1, 1, 2, 3, 5, 8)), max(1, length // 2))
        capacity = length + rng.randrange(1, 200)
        capacity += capacity == 3072
        case = _cache("", dtype, b, t, capacity, length, heads, kv_heads, dim, rng.choice((0.0, 0.0, 30.0)), rng.random() < 0.3)
    else:
        t = _spread(rng, 1, 8192 if dtype == "f16" else 2800)
        mask = rng.choice(("none", "causal", "causal", "prefix", "documents", "window"))
        keys = t if mask != "none" or rng.random() < 0.5 else _spread(rng, 1, 4096 if dtype == "f16" else 2000)
        room = (1 << 29) if dtype == "f16" else (1 << 25)
        while heads > 1 and heads * t * keys > room:
            heads, kv_heads = max(1, heads // 2), 1
        b = max(1, min(rng.choice((1, 2, 3, 4)), room // (heads * t * keys)))
        parts = {"prefix": max(1, t // 5), "documents": max(1, min(9, t // 100)), "window": max(1, t // 4)}.get(mask, 0)
        case = _attention("", dtype, b, t, keys, heads, kv_heads, dim, mask, parts, rng.choice((0.0, 0.0, 50.0)), rng.random() < 0.3)
    del case["name"]
    return case


# ------------------------------------------------------------------------------- what a program has in hand
class _Host:
    """Seeded values in host memory, where a program's data come from."""

    def __init__(self, case, seed):
        self._rng = torch.Generator(device="cuda").manual_seed(seed)
        self.order = np.random.default_rng(seed)
        self._dtype = _TORCH[case["dtype"]]

    def normal(self, shape, scale=1.0, middle=0.0):
        return torch.randn(shape, generator=self._rng, device="cuda").mul_(scale).add_(middle).to(self._dtype).cpu().numpy()


def _grid(case):
    return [case["grid%d" % a] for a in range(case["axes"])]


def _sections(case):
    """Pairs of a head's values that each axis of positions turns: all of them for one axis, even parts for two, and for three a
    quarter for the time and the rest in even parts (what that leaves over stays as it is)."""
    pairs = case["dim"] // 2
    return {1: (pairs,), 2: (pairs // 2,) * 2, 3: (pairs // 4,) + ((pairs - pairs // 4) // 2,) * 2}[case["axes"]]


def _document_ids(case, order):
    """Documents of one to three shares of the sequence, in an order of their own."""
    n, t = case["parts"], case["t"]
    share = [1 + k % 3 for k in range(n)]
    ends = [t * sum(share[:k + 1]) // sum(share) for k in range(n)]
    sizes = np.diff([0] + ends)
    return np.stack([np.repeat(np.arange(n), order.permutation(sizes)) for _ in range(case["b"])]).astype(np.int32)


def _history(case, order=None):
    """The requests' lengths, the new tokens among them."""
    low, high, b = max(case["t"], case["length"] // 2), case["length"], case["b"]
    lengths = np.array([high - (high - low) * k // max(1, b - 1) for k in range(b)], dtype=np.int32)
    return lengths if order is None else order.permutation(lengths)


def _slopes(heads):
    """Slopes of a bias by distance, a geometric series."""
    return (2.0 ** (-8.0 * (np.arange(heads) + 1) / heads)).astype(np.float32)


def _program_data(case, seed):
    """Host arrays by name."""
    host, kind, d = _Host(case, seed), case["kind"], {}
    b, heads, dim = case["b"], case["heads"], case["dim"]
    if kind == "norm":
        grid, axes = _grid(case), case["axes"]
        t = math.prod(grid)
        d["x"], d["g"] = host.normal((b, t, heads, dim), 1.5), host.normal((b, t, heads, dim))
        d["w"] = host.normal((dim,), 0.2, 1.0)
        where = np.stack(np.meshgrid(*(np.arange(n) for n in grid), indexing="ij"), -1).reshape(1, t, axes)
        d["positions"] = (where + host.order.integers(0, 300, (b, 1, axes))).astype(np.int32)
        return d
    kv_heads = case["kv_heads"]
    if kind == "attention":
        t, keys = case["t"], case["keys"]
        d["q"], d["k"] = host.normal((b, t, heads, dim), 1.3), host.normal((b, keys, kv_heads, dim), 1.3)
        d["v"], d["g"] = host.normal((b, keys, kv_heads, dim)), host.normal((b, t, heads, dim))
        if case["mask"] == "documents":
            d["documents"] = _document_ids(case, host.order)
    else:
        t, capacity = case["t"], case["capacity"]
        d["q"], d["k"], d["v"] = host.normal((b, t, heads, dim), 1.3), host.normal((b, t, kv_heads, dim), 1.3), host.normal((b, t, kv_heads, dim))
        d["old_k"], d["old_v"] = host.normal((b, capacity, kv_heads, dim), 1.3), host.normal((b, capacity, kv_heads, dim))
        d["lengths"] = _history(case, host.order)
    if case["bias"]:
        d["slopes"] = _slopes(heads)
    return d


def _angles(case, rows):
    """cos and sin of the angle of each pair at each position up to ``rows``, and the axis each pair goes by."""
    sections = _sections(case)
    frequency = np.concatenate([_BASE ** (-np.arange(n) / n) for n in sections])
    axis = np.repeat(np.arange(len(sections)), sections)
    angle = np.arange(rows)[:, None] * frequency[None]
    return np.cos(angle), np.sin(angle), axis


def _rows(case):
    return 300 + max(_grid(case))


def prepare(case, seed):
    data, kind = _program_data(case, seed), case["kind"]
    state = {"case": case}
    if not own:
        state.update({name: torch.from_numpy(value).cuda() for name, value in data.items()})
        if kind == "norm":
            cos, sin, axis = _angles(case, _rows(case))
            state["cos"], state["sin"] = (torch.from_numpy(v.astype(np.float32)).cuda() for v in (cos, sin))
            state["axis"] = torch.from_numpy(axis).cuda()
        return state

    import mygrad_amd as mg
    from mygrad_amd import nnet

    learnt = ("x", "w") if kind == "norm" else ("q", "k", "v") if kind == "attention" else ()
    state.update({name: mg.device_tensor(value, constant=name not in learnt) for name, value in data.items() if value.dtype.kind == "f"})
    if kind == "norm":
        state["rotary"] = nnet.RotaryTable(_sections(case), _rows(case), base=_BASE).at(data["positions"])
    elif kind == "attention":
        mask, parts = case["mask"], case["parts"]
        more = {"prefix": {"prefix": parts}, "documents": {"documents": data.get("documents")}, "window": {"window": parts}}.get(mask, {})
        state["mask"] = nnet.AttentionMask(causal=mask != "none", **more)
    else:
        state["cache"] = nnet.KeyValueCache(case["b"], case["capacity"], case["kv_heads"], case["dim"], dtype=data["k"].dtype)
        whole = nnet.AttentionMask(lengths=np.full(case["b"], case["capacity"]))
        state["cache"].write(state.pop("old_k"), state.pop("old_v"), whole)
        state["mask"] = nnet.AttentionMask(causal=True, lengths=data["lengths"])
    return state


# ---------------------------------------------------------------------------------------- the package's calls
class _OnDevice:
    """A result's device memory, described to torch; keeps the memory alive."""

    def __init__(self, array):
        self._array = array
        self.__cuda_array_interface__ = {"shape": array.shape, "typestr": array.dtype.str, "data": (array.buf.ptr, False), "version": 2}


def _whole(array):
    return torch.as_tensor(_OnDevice(array), device="cuda")


def _run_own(state):
    from mygrad_amd import nnet

    case, kind = state["case"], state["case"]["kind"]
    if kind == "norm":
        x, w = state["x"], state["w"]
        out = nnet.head_norm(x, w, eps=_EPS, rotary=state["rotary"])
        if not case["train"]:
            return [_whole(out._value)]
        out.backward(state["g"])
        return [_whole(a) for a in (out._value, x._grad, w._grad)]
    scores = {"cap": case["cap"] or None, "slopes": state.get("slopes"), "mask": state["mask"]}
    q, k, v = state["q"], state["k"], state["v"]
    if kind == "attention":
        out = nnet.attention(q, k, v, **scores)
        out.backward(state["g"])
        return [_whole(a) for a in (out._value, q._grad, k._grad, v._grad)]
    cache = state["cache"]
    cache.write(k, v, state["mask"])
    out = cache.attend(q, **scores)
    return [_whole(a) for a in (out._value, cache.keys, cache.values)]


# ------------------------------------------------------------------------------ the same, operation by operation
def _visible(case, state):
    """Which keys each query sees, as (batch or 1, 1, 1, queries, keys); None for all of them."""
    mask = case.get("mask", "cache")
    if mask == "none":
        return None
    at = torch.arange(case["t"], device="cuda")
    if mask == "cache":
        lengths = state["lengths"].long()[:, None, None]
        return (torch.arange(case["capacity"], device="cuda") <= at[:, None] + lengths - case["t"])[:, None, None]
    keys = torch.arange(case["keys"], device="cuda")
    seen = keys <= at[:, None]
    if mask == "prefix":
        seen = seen | (keys < case["parts"])
    elif mask == "window":
        seen = seen & (keys > at[:, None] - case["parts"])
    elif mask == "documents":
        ids = state["documents"]
        return (seen & (ids[:, :, None] == ids[:, None, :]))[:, None, None]
    return seen[None, None, None]


def _by_head(x, kv_heads):
    """(batch, tokens, heads, dim) as (batch, key heads, heads that share one, tokens, dim) in 32 bits."""
    b, t, heads, dim = x.shape
    return x.float().permute(0, 2, 1, 3).reshape(b, kv_heads, heads // kv_heads, t, dim)


def _by_token(x, like):
    b, kv_heads, group, t, dim = x.shape
    return x.reshape(b, kv_heads * group, t, dim).permute(0, 2, 1, 3).contiguous().to(like.dtype)


def _distances(case, state):
    at = torch.arange(case["t"], device="cuda")
    if case["kind"] == "cache":
        keys = torch.arange(case["capacity"], device="cuda")
        where = at[:, None] + state["lengths"].long()[:, None, None] - case["t"]
        return (where - keys).abs().float()[:, None, None]
    keys = torch.arange(case["keys"], device="cuda")
    return (at[:, None] + (case["keys"] - case["t"]) - keys).abs().float()[None, None, None]


def _softmax_of_scores(case, state, q, k):
    """The weights and, for the gradient, what the cap lets through."""
    s = (q @ k.transpose(-1, -2)) * case["dim"] ** -0.5
    through = None
    if case["cap"]:
        bent = torch.tanh(s / case["cap"])
        s, through = bent * case["cap"], 1.0 - bent * bent
    if case["bias"]:
        slopes = state["slopes"].reshape(1, k.shape[1], -1, 1, 1)
        s = s - slopes * _distances(case, state)
    seen = _visible(case, state)
    if seen is not None:
        s = torch.where(seen, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, 1.0), through


def _run_plain(state):
    case, kind = state["case"], state["case"]["kind"]
    if kind == "norm":
        x, w = state["x"].float(), state["w"].float()
        pairs = sum(_sections(case))
        rows = state["positions"].long()[:, :, state["axis"]]  # (batch, tokens, pairs)
        column = torch.arange(pairs, device="cuda")
        cos, sin = state["cos"][rows, column][:, :, None], state["sin"][rows, column][:, :, None]
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
        z = x * r * w
        first, second = z[..., :pairs], z[..., pairs:2 * pairs]
        y = torch.cat((first * cos - second * sin, second * cos + first * sin, z[..., 2 * pairs:]), -1).to(state["x"].dtype)
        if not case["train"]:
            return [y]
        g = state["g"].float()
        first, second = g[..., :pairs], g[..., pairs:2 * pairs]
        u = torch.cat((first * cos + second * sin, second * cos - first * sin, g[..., 2 * pairs:]), -1)
        dw = (u * x * r).sum((0, 1, 2))
        u = u * w
        dx = r * (u - x * (r * r * (u * x).mean(-1, keepdim=True)))
        return [y, dx.to(y.dtype), dw.to(y.dtype)]
    kv_heads = case["kv_heads"]
    if kind == "cache":
        keys, values = state["old_k"], state["old_v"]
        new = (state["lengths"].long()[:, None] - case["t"]) + torch.arange(case["t"], device="cuda")
        request = torch.arange(case["b"], device="cuda")[:, None]
        keys[request, new], values[request, new] = state["k"], state["v"]
        p, _ = _softmax_of_scores(case, state, _by_head(state["q"], kv_heads), _by_head(keys, kv_heads))
        return [_by_token(p @ _by_head(values, kv_heads), state["q"]), keys, values]
    q, k, v, g = (_by_head(state[name], kv_heads) for name in "qkvg")
    p, through = _softmax_of_scores(case, state, q, k)
    out = p @ v
    dv = (p.transpose(-1, -2) @ g).sum(2, keepdim=True)
    ds = p * (g @ v.transpose(-1, -2) - (g * out).sum(-1, keepdim=True))
    if through is not None:
        ds = ds * through
    ds = ds * case["dim"] ** -0.5
    dk = (ds.transpose(-1, -2) @ q).sum(2, keepdim=True)
    return [_by_token(out, state["q"]), _by_token(ds @ k, state["q"]), _by_token(dk, state["k"]), _by_token(dv, state["v"])]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# -------------------------------------------------------------------------------- the definitions in 64 bits
def _norm64(case, x, w, positions):
    """Each pair as a complex number that is turned by its angle."""
    angle, start = [], 0
    for a, n in enumerate(_sections(case)):
        frequency = _BASE ** (-torch.arange(n, device="cuda", dtype=torch.float64) / n)
        angle.append(positions[:, :, a, None].double() * frequency)
        start += n
    angle = torch.cat(angle, -1)[:, :, None]
    z = x / ((x ** 2).mean(-1, keepdim=True) + _EPS).sqrt() * w
    turned = torch.complex(z[..., :start], z[..., start:2 * start]) * torch.polar(torch.ones_like(angle), angle)
    return torch.cat((turned.real, turned.imag, z[..., 2 * start:]), -1)


def _attend64(case, q, k, v, slope, first, ids):
    """One head of one sequence: q:(queries, dim); ``first``: the place of the first query; ``ids``: documents or None."""
    place = torch.arange(q.shape[0], device="cuda")[:, None] + first
    key = torch.arange(k.shape[0], device="cuda")[None]
    s = q @ k.T / math.sqrt(case["dim"])
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    if slope is not None:
        s = s - slope * (place - key).abs()
    mask = case.get("mask", "causal")
    if mask != "none":
        hidden = key > place
        if mask == "prefix":
            hidden = hidden & (key >= case["parts"])
        elif mask == "window":
            hidden = hidden | (place - key >= case["parts"])
        elif mask == "documents":
            hidden = hidden | (ids[:, None] != ids[None])
        s = s.masked_fill(hidden, -math.inf)
    return torch.softmax(s, -1) @ v


def exact(case, seed):
    """The cache that comes back beside a result is a copy of inputs: it has no value of its own here."""
    data, kind = _program_data(case, seed), case["kind"]
    held = {name: torch.from_numpy(value).cuda() for name, value in data.items()}
    if kind == "norm":
        x, w = (held[name].double().requires_grad_(case["train"]) for name in "xw")
        y = _norm64(case, x, w, held["positions"])
        return [y.detach(), *torch.autograd.grad(y, (x, w), held["g"].double())] if case["train"] else [y]
    group = case["heads"] // case["kv_heads"]
    out = torch.empty(held["q"].shape, dtype=torch.float64, device="cuda")
    grads = [torch.zeros(held[name].shape, dtype=torch.float64, device="cuda") for name in "qkv"]
    for n in range(case["b"]):
        for h in range(case["heads"]):
            slope = float(data["slopes"][h]) if case["bias"] else None
            q = held["q"][n, :, h].double()
            if kind == "cache":
                length = int(data["lengths"][n])
                k, v = (torch.cat((held["old_" + name][n, :length - case["t"], h // group], held[name][n, :, h // group])).double() for name in "kv")
                out[n, :, h] = _attend64(case, q, k, v, slope, length - case["t"], None)
                continue
            leaves = [q.requires_grad_()] + [held[name][n, :, h // group].double().requires_grad_() for name in "kv"]
            first = case["keys"] - case["t"]
            o = _attend64(case, *leaves, slope, first, held["documents"][n] if case["mask"] == "documents" else None)
            out[n, :, h] = o.detach()
            for total, part, head in zip(grads, torch.autograd.grad(o, leaves, held["g"][n, :, h].double()), (h, h // group, h // group)):
                total[n, :, head] += part
    return [out, None, None] if kind == "cache" else [out, *grads]


# ------------------------------------------------------------------------------- what a pass cannot do without
def _pairs_seen(case):
    """Pairs of a query and a key that it sees, for one head of the whole batch."""
    b, t, mask, parts = case["b"], case["t"], case["mask"], case["parts"]
    if mask == "none":
        return b * t * case["keys"]
    if mask == "documents":
        share = [1 + k % 3 for k in range(parts)]
        sizes = np.diff([0] + [t * sum(share[:k + 1]) // sum(share) for k in range(parts)])
        return b * int(sum(n * (n + 1) // 2 for n in sizes))
    rows = np.arange(1, t + 1)
    return b * int((np.minimum(rows, parts) if mask == "window" else np.maximum(rows, parts if mask == "prefix" else 0)).sum())


def work(case):
    """Operands read once and results written once; forward two products for each pair that is seen, backward five."""
    size, b, heads, dim = _BYTES[case["dtype"]], case["b"], case["heads"], case["dim"]
    if case["kind"] == "norm":
        t = math.prod(_grid(case))
        values = b * t * heads * dim
        tables = b * t * sum(_sections(case)) * 8
        return {"bytes": float(values * size * (5 if case["train"] else 2) + tables), "flops": float(values * (24 if case["train"] else 8))}
    if case["kind"] == "cache":
        seen = int(_history(case).sum())
        values = 2 * seen * case["kv_heads"] * dim + 2 * b * case["t"] * (heads + case["kv_heads"]) * dim
        return {"bytes": float(values * size), "flops": 4.0 * seen * case["t"] * heads * dim}
    ends = 2 * b * (2 * case["t"] * heads + 2 * case["keys"] * case["kv_heads"]) * dim
    return {"bytes": float(ends * size), "flops": 14.0 * _pairs_seen(case) * heads * dim}
