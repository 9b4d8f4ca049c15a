"""What is timed of the operators at a language model's two ends and between its blocks: ``embedding`` (rows of a table by token,
with the gradient of the whole table), ``layer_norm``, ``log_probabilities`` (of given tokens, with entropies and the likeliest
alternatives) and ``distillation`` (from a teacher's likeliest tokens).

Where ``own`` is true a pass makes the package's calls on tensors that live on the device, and hands results back as torch
tensors over the same memory; where it is false it is the same arithmetic in elementary torch operations, in 32 bits (64 for
float64)."""

import math

import numpy as np
import torch

own = False

_TORCH = {"f16": torch.float16, "f32": torch.float32, "f64": torch.float64}
_WIDE = {"f16": torch.float32, "f32": torch.float32, "f64": torch.float64}  # sums are carried in, and what losses come back in
_BYTES = {"f16": 2, "f32": 4, "f64": 8}
_EPS = 1e-5


# ----------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one new token of each request in a small batch: nothing but latency
        _norm("norm-token-f16", "f16", 8, 768, train=False),
        # the bulk of a language model's training
        _norm("norm-train-f16", "f16", 16384, 4096),
        # single precision, rows of a length that no vector divides
        _norm("norm-ragged-f32", "f32", 9973, 1531),
        # the next token of each request of a batch
        _embedding("embedding-token-f16", "f16", 32, 50001, 1024, train=False),
        # a training step on text, whose tokens are mostly a few
        _embedding("embedding-train-f16", "f16", 16384, 50000, 2048, scale=math.sqrt(2048.0)),
        # a short padded batch in single precision; rows that are no whole vectors
        _embedding("embedding-padded-f32", "f32", 1999, 32003, 771, padded=True),
        # what a server answers with: the token's log probability, entropy and the likeliest alternatives
        _scores("scores-serve-f16", "f16", 8, 50001, entropy=True, top=8, train=False),
        # a language model's loss and its gradient; the largest pass
        _scores("scores-train-f16", "f16", 4096, 50000),
        # a policy's loss: entropies have a gradient too, some tokens of the vocabulary are ruled out, rows are padded
        _scores("scores-policy-f32", "f32", 1021, 32003, entropy=True, top=5, masked=True, padded=True),
        # a few rows in single precision over a long vocabulary: the work has to be split along it
        _distillation("distill-few-f32", "f32", 12, 131101, 20),
        # training of a small model by a large one's answers
        _distillation("distill-train-f16", "f16", 4096, 32000, 64, temperature=2.0),
        # double precision, for checks by differences; teachers' lists of different lengths
        _distillation("distill-ragged-f64", "f64", 257, 4099, 33, padded=True),
    ]


def _norm(name, dtype, rows, dim, train=True):
    return {"name": name, "kind": "norm", "dtype": dtype, "rows": rows, "dim": dim, "train": train}


def _embedding(name, dtype, rows, vocabulary, dim, scale=1.0, padded=False, train=True):
    return {"name": name, "kind": "embedding", "dtype": dtype, "rows": rows, "vocabulary": vocabulary, "dim": dim, "scale": scale,
            "padded": padded, "train": train}


def _scores(name, dtype, rows, vocabulary, entropy=False, top=0, masked=False, padded=False, train=True):
    """``masked``: a part of the vocabulary has logits of minus infinity."""
    return {"name": name, "kind": "scores", "dtype": dtype, "rows": rows, "vocabulary": vocabulary, "entropy": entropy, "top": top,
            "masked": masked, "padded": padded, "train": train}


def _distillation(name, dtype, rows, vocabulary, top, temperature=1.0, padded=False, train=True):
    return {"name": name, "kind": "distillation", "dtype": dtype, "rows": rows, "vocabulary": vocabulary, "top": top,
            "temperature": temperature, "padded": padded, "train": train}


def _spread(rng, low, high):
    """A whole number whose logarithm is spread evenly."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("norm", "embedding", "scores", "distillation"))
    dtype, train = rng.choice(("f16", "f16", "f16", "f32", "f32", "f64")), rng.random() < 0.8
    # as much work as the largest listed case at most: what a wider type moves more it has fewer values of
    values = (1 << 26) * 2 // _BYTES[dtype]
    if kind == "norm":
        dim = _spread(rng, 16, 16384)
        dim -= dim % 8 if rng.random() < 0.5 else 0
        rows = min(_spread(rng, 1, 65536), values // dim)
        case = _norm("", dtype, rows, dim, train)
    elif kind == "embedding":
        dim = _spread(rng, 16, 8192)
        dim -= dim % 8 if rng.random() < 0.5 else 0
        vocabulary = max(2, min(_spread(rng, 200, 200000), values // dim))
        rows = min(_spread(rng, 1, 65536), max(1, values // 2 // dim))
        case = _embedding("", dtype, rows, vocabulary, dim, rng.choice((1.0, math.sqrt(dim), 0.25)), rng.random() < 0.3, train)
    elif kind == "scores":
        vocabulary, top = _spread(rng, 40, 160000), rng.choice((0, 0, 0, 1, 5, 20))
        rows = max(1, min(_spread(rng, 1, 8192), values // (8 if top else 1) // vocabulary))
        case = _scores("", dtype, rows, vocabulary, rng.random() < 0.5, top, rng.random() < 0.3, rng.random() < 0.3, train)
    else:
        vocabulary, top = _spread(rng, 150, 160000), _spread(rng, 1, 128)
        rows = max(1, min(_spread(rng, 1, 8192), values // vocabulary))
        case = _distillation("", dtype, rows, vocabulary, top, rng.choice((1.0, 1.0, 2.0, 0.5)), rng.random() < 0.3, train)
    del case["name"]
    return case


# ------------------------------------------------------------------------------- what a program has in hand
class _Seeded:
    """Seeded values on the device and, for what decides how much there is to do, in host memory."""

    def __init__(self, case, seed):
        self._rng = torch.Generator(device="cuda").manual_seed(seed)
        self.order = np.random.default_rng(seed)
        self._case = case

    def normal(self, shape, scale=1.0, middle=0.0, dtype=None):
        """In pieces: values are made in single precision."""
        out = torch.empty(shape, dtype=_TORCH[self._case["dtype"]] if dtype is None else dtype, device="cuda")
        flat = out.view(-1)
        for at in range(0, flat.numel(), 1 << 26):
            part = flat[at:at + (1 << 26)]
            part.copy_(torch.randn(part.shape, generator=self._rng, device="cuda").mul_(scale).add_(middle))
        return out

    def words(self, count, vocabulary):
        """Tokens of a text: the n-th most frequent one has about 1 / n of the most frequent one's share; ids are in no order."""
        rank = np.exp(self.order.random(count) * math.log(vocabulary)).astype(np.int64) - 1
        return self.order.permutation(vocabulary)[np.clip(rank, 0, vocabulary - 1)].astype(np.int32)


def _data(case, seed):
    """By name: what floats are, on the device; whole numbers as int32 host arrays."""
    made, kind, rows, d = _Seeded(case, seed), case["kind"], case["rows"], {}
    wide = _WIDE[case["dtype"]]
    if kind == "norm":
        dim = case["dim"]
        d["x"], d["g"] = made.normal((rows, dim), 1.5, 0.4), made.normal((rows, dim))
        d["w"], d["b"] = made.normal((dim,), 0.2, 1.0), made.normal((dim,), 0.2)
        return d
    vocabulary = case["vocabulary"]
    if kind == "embedding":
        d["table"], d["g"] = made.normal((vocabulary, case["dim"]), 0.05), made.normal((rows, case["dim"]))
        d["ids"] = made.words(rows, vocabulary)
        if case["padded"]:
            d["ids"][made.order.random(rows) < 0.2] = -1
        return d
    logits = made.normal((rows, vocabulary), 2.0)
    if kind == "scores":
        d["ids"] = made.words(rows, vocabulary)
        if case["masked"]:  # of any four neighbours one is out, and it is never the one that came
            out = torch.arange(vocabulary, device="cuda") % 4 == 3
            logits.masked_fill_(out, -math.inf)
            d["ids"] -= d["ids"] % 4 == 3
        # the model knows something: the token that came is likelier than others
        rows_at = torch.arange(rows, device="cuda")
        logits[rows_at, torch.from_numpy(d["ids"]).cuda().long()] += 6.0
        if case["padded"]:
            d["ids"][made.order.random(rows) < 0.2] = -1
        planes = (2, rows) if case["entropy"] else (rows,)
        d["g"] = made.normal(planes, 0.3, -1.0, wide)
    else:
        top = case["top"]
        # different tokens for each row: a stride through the vocabulary
        first, step = made.order.integers(0, vocabulary, (rows, 1)), made.order.integers(1, max(2, vocabulary // top), (rows, 1))
        d["ids"] = ((first + step * np.arange(top)) % vocabulary).astype(np.int32)
        at = torch.from_numpy(d["ids"]).cuda().long()
        logits.scatter_add_(1, at, made.normal((rows, top), 1.0, 3.0))
        d["teacher"] = made.normal((rows, top), 1.5, 4.0).sort(1, descending=True).values
        if case["padded"]:
            d["ids"][np.arange(top) >= made.order.integers(1, top + 1, (rows, 1))] = -1
        d["g"] = made.normal((rows,), 0.3, 1.0, wide)
    d["logits"] = logits
    return d


def prepare(case, seed):
    data = _data(case, seed)
    state = {"case": case}
    if not own:
        state.update({name: torch.from_numpy(value).cuda() if isinstance(value, np.ndarray) else value for name, value in data.items()})
        return state

    import mygrad_amd as mg
    from mygrad_amd import nnet

    learnt = {"norm": "xwb", "embedding": ("table",)}.get(case["kind"], ("logits",)) if case["train"] else ()
    for name, value in data.items():
        if isinstance(value, np.ndarray):
            state[name] = nnet.TokenIds(value)
        else:
            state[name] = mg.device_tensor(value.cpu().numpy(), constant=name not in learnt)
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
    more = []
    if kind == "norm":
        learnt = [state["x"], state["w"], state["b"]]
        out = nnet.layer_norm(*learnt, eps=_EPS)
    elif kind == "embedding":
        learnt = [state["table"]]
        out = nnet.embedding(state["table"], state["ids"], scale=case["scale"])
    elif kind == "scores":
        learnt = [state["logits"]]
        out = nnet.log_probabilities(state["logits"], state["ids"], entropy=case["entropy"], top=case["top"])
        if case["top"]:
            out, likeliest, which = out
            more = [_whole(likeliest._value), _whole(which._value)]
    else:
        learnt = [state["logits"]]
        out = nnet.distillation(state["logits"], state["ids"], state["teacher"], temperature=case["temperature"])
    result = [_whole(out._value), *more]
    if case["train"]:
        out.backward(state["g"])
        result += [_whole(t._grad) for t in learnt]
    return result


# ------------------------------------------------------------------------------ the same, operation by operation
def _norm_plain(case, state):
    x, w, b, g = (state[name].to(_WIDE[case["dtype"]]) for name in "xwbg")
    middle = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((middle * middle).mean(-1, keepdim=True) + _EPS)
    n = middle * r
    out = [n * w + b]
    if case["train"]:
        u = g * w
        dx = r * (u - u.mean(-1, keepdim=True) - n * (u * n).mean(-1, keepdim=True))
        out += [dx, (g * n).sum(0), g.sum(0)]
    return [v.to(state["x"].dtype) for v in out]


def _embedding_plain(case, state):
    table, g = state["table"], state["g"]
    wide, ids = _WIDE[case["dtype"]], state["ids"].long()
    there, at = (ids >= 0)[:, None], ids.clamp(min=0)
    out = [torch.where(there, table[at].to(wide) * case["scale"], 0.0)]
    if case["train"]:
        out.append(torch.zeros(table.shape, dtype=wide, device="cuda").index_add_(0, at, torch.where(there, g.to(wide) * case["scale"], 0.0)))
    return [v.to(table.dtype) for v in out]


def _ordered(z):
    """Whole numbers in the order of floats of 32 bits, and of no other."""
    bits = (z + 0.0).view(torch.int32).long()
    return torch.where(bits < 0, -(bits & 0x7fffffff), bits)


def _likeliest(z, count):
    """Places of the largest values, the lowest one first among equals."""
    if z.dtype == torch.float64:
        return torch.sort(z, -1, descending=True, stable=True).indices[:, :count]
    places = z.shape[-1] - 1 - torch.arange(z.shape[-1], device="cuda")
    return z.shape[-1] - 1 - (torch.topk((_ordered(z) << 32) + places, count, -1).values & 0xffffffff)


def _scores_plain(case, state):
    logits, g = state["logits"], state["g"]
    z, ids = logits.to(_WIDE[case["dtype"]]), state["ids"].long()
    there, at = ids >= 0, ids.clamp(min=0)[:, None]
    t = z - z.amax(-1, keepdim=True)
    e = torch.exp(t)
    s = e.sum(-1, keepdim=True)
    scores = [torch.where(there, (t.gather(1, at) - torch.log(s))[:, 0], 0.0)]
    if case["entropy"]:
        bounded = torch.where(e > 0, t, 0.0)
        middle = (e * bounded).sum(-1, keepdim=True) / s
        scores.append((torch.log(s) - middle)[:, 0])
    out = [torch.stack(scores) if case["entropy"] else scores[0]]
    if case["top"]:
        which = _likeliest(z, case["top"])
        out += [t.gather(1, which) - torch.log(s), which.int()]
    if case["train"]:
        own_g = torch.where(there, g[0] if case["entropy"] else g, 0.0)[:, None]
        e /= s
        dz = e * (-own_g)
        if case["entropy"]:
            dz -= e * (bounded - middle) * g[1][:, None]
        out.append(dz.scatter_add_(1, at, own_g).to(logits.dtype))
    return out


def _distillation_plain(case, state):
    logits, teacher, g = state["logits"], state["teacher"], state["g"]
    wide, ids, c = _WIDE[case["dtype"]], state["ids"].long(), 1.0 / case["temperature"]
    there, at = ids >= 0, ids.clamp(min=0)
    z = logits.to(wide)
    t = (z - z.amax(-1, keepdim=True)) * c
    e = torch.exp(t)
    s = e.sum(-1, keepdim=True)
    y = torch.where(there, teacher.to(wide), -math.inf)
    y = (y - y.amax(-1, keepdim=True)) * c
    f = torch.exp(y)
    total = f.sum(-1, keepdim=True)
    q = f / total
    terms = q * ((y - torch.log(total)) - (t.gather(1, at) - torch.log(s)))
    out = [torch.where(there, terms, 0.0).sum(-1)]
    if case["train"]:
        g = g[:, None] * c
        out.append((e / s * g).scatter_add_(1, at, -q * g).to(logits.dtype))
    return out


def _run_plain(state):
    plain = {"norm": _norm_plain, "embedding": _embedding_plain, "scores": _scores_plain, "distillation": _distillation_plain}
    return plain[state["case"]["kind"]](state["case"], state)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# -------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    """Which tokens are the likeliest is no computed number: it has no value of its own here."""
    d, kind = _data(case, seed), case["kind"]
    ids = torch.from_numpy(d["ids"]).cuda().long() if "ids" in d else None
    if kind == "norm":
        x, w, b = (d[name].double().requires_grad_(case["train"]) for name in "xwb")
        deviation = x - x.sum(1, keepdim=True) / case["dim"]
        y = deviation / (deviation.square().sum(1, keepdim=True) / case["dim"] + _EPS).sqrt() * w + b
        return [y.detach(), *torch.autograd.grad(y, (x, w, b), d["g"].double())] if case["train"] else [y]
    if kind == "embedding":
        # a token's row is picked by a product with a row that has a one at its place; tokens that are none have no row
        padded = torch.cat((d["table"].double(), torch.zeros(1, case["dim"], dtype=torch.float64, device="cuda")))
        out = [padded[ids] * case["scale"]]
        if case["train"]:
            order = torch.argsort(ids, stable=True)
            held, counts = torch.unique_consecutive(ids[order], return_counts=True)
            sums = torch.zeros(case["vocabulary"] + 1, case["dim"], dtype=torch.float64, device="cuda")
            owner = torch.repeat_interleave(held, counts)
            sums.index_add_(0, torch.where(owner < 0, case["vocabulary"], owner), d["g"][order].double())
            out.append(sums[:-1] * case["scale"])
        return out
    rows, parts = case["rows"], {}
    block = max(1, (1 << 26) // case["vocabulary"])
    for at in range(0, rows, block):
        these = slice(at, min(rows, at + block))
        z, tokens = d["logits"][these].double().requires_grad_(case["train"]), ids[these]
        if kind == "scores":
            lp = z - torch.logsumexp(z, 1, keepdim=True)
            each = torch.arange(len(tokens), device="cuda")
            result = [torch.where(tokens < 0, 0.0, lp[each, tokens.clamp(min=0)])]
            if case["entropy"]:
                result.append(-(lp.exp() * torch.where(lp == -math.inf, 0.0, lp)).sum(1))
            result = torch.stack(result)
            g = d["g"].double().reshape(-1, rows)[:, these]
            found = {"scores": result.detach()}
            if case["top"]:
                found["top"] = torch.sort(lp.detach(), 1, descending=True).values[:, :case["top"]]
        else:
            lp = torch.log_softmax(z / case["temperature"], 1)
            teacher = torch.where(tokens < 0, -math.inf, d["teacher"][these].double() / case["temperature"])
            q = torch.softmax(teacher, 1)
            result = torch.where(tokens < 0, 0.0, q * (torch.log_softmax(teacher, 1) - lp.gather(1, tokens.clamp(min=0)))).sum(1)
            g = d["g"].double()[these]
            found = {"scores": result.detach()}
        if case["train"]:
            found["dz"] = torch.autograd.grad(result, z, g)[0]
        for name, value in found.items():
            parts.setdefault(name, []).append(value)
    scores = torch.cat(parts["scores"], -1)
    out = [scores if case.get("entropy") or kind == "distillation" else scores[0]]
    if case["top"] and kind == "scores":
        out += [torch.cat(parts["top"]), None]
    return out + [torch.cat(parts["dz"])] if case["train"] else out


# ------------------------------------------------------------------------------- what a pass cannot do without
def _different(count, vocabulary):
    """How many different tokens a text of ``count`` has, on average (by the shares that its words are drawn with)."""
    place = np.arange(1, vocabulary + 1)
    share = np.log1p(1.0 / place) / math.log(vocabulary + 1)
    return float(-np.expm1(count * np.log1p(-np.minimum(share, 1 - 1e-12))).sum())


def work(case):
    """Operands read once and results written once.  Of a table a pass needs the rows that its tokens name; its gradient is written
    whole.  Tokens that are none have nothing to read."""
    size, wide, rows, train = _BYTES[case["dtype"]], max(4, _BYTES[case["dtype"]]), case["rows"], case["train"]
    if case["kind"] == "norm":
        dim = case["dim"]
        values = (4 if train else 2) * rows * dim + (4 if train else 2) * dim
        return {"bytes": float(values * size), "flops": float((20 if train else 8) * rows * dim)}
    if case["kind"] == "embedding":
        dim, vocabulary = case["dim"], case["vocabulary"]
        there = rows * (0.8 if case["padded"] else 1.0)
        values = (_different(there, vocabulary) + rows) * dim + ((there + vocabulary) * dim if train else 0)
        return {"bytes": float(values * size + 4 * rows), "flops": float((2 if train else 1) * there * dim)}
    values, each = rows * case["vocabulary"], 4 + (4 if train else 0)
    if case["kind"] == "scores":
        small = rows * (4 + wide * (2 if case["entropy"] else 1) * (2 if train else 1) + (4 + wide) * case["top"])
        each += (3 + (3 if train else 0)) if case["entropy"] else 0
    else:
        small = rows * (case["top"] * (4 + size) + wide * (2 if train else 1))
    return {"bytes": float(values * size * (2 if train else 1) + small), "flops": float(each * values)}
