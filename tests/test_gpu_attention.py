"""Attention on the GPU against its formulas in 64 bits.

Bars are bounds on the rounding, worked out from the operands of each test: u is the unit of the sums (2^-24, 2^-53 for float64), r
that of the type results and weights are rounded to on the way (2^-11 for float16, else u).  A score s = scale q.k is off by at most
(D + 8) u scale |q||k| and, behind cap and bias, by 8 u of the largest value on its way; a weight by twice that and by
(n + 32) u + r of itself; then every result is a weighted sum.  dS = P (dP - D) (1 - t^2) scale adds the errors of the two products
(D + 8) u |g||v|, of the stored result in D (r |g||out|) and of t."""

import numpy as np
import pytest

import mygrad_amd as mg
from mygrad_amd.nnet import AttentionMask, KeyValueCache, attention
from oracle import attention as ora

pytestmark = pytest.mark.gpu

UNIT = {np.float16: (2.0**-24, 2.0**-11), np.float32: (2.0**-24, 2.0**-24), np.float64: (2.0**-53, 2.0**-53)}
SMALLEST = {np.float16: 2.0**-24, np.float32: 2.0**-126, np.float64: 2.0**-1022}


@pytest.fixture(scope="module", autouse=True)
def device():
    if not mg.is_available():
        pytest.fail("libmygrad_hip.so / gfx950 device not available: the GPU tests need both")


def norms(a):
    return np.sqrt((np.asarray(a, dtype=np.float64) ** 2).sum(-1))


def _bounds(dtype, q, k, v, g, p, s, bent, out, grads, scale, cap):
    """Largest differences to be expected of out, dq, dk, dv, as arrays that broadcast against them."""
    u, r = UNIT[dtype]
    D, group = q.shape[3], q.shape[2] // k.shape[2]
    most = lambda a: norms(a).max(initial=0.0)
    seen = s[np.isfinite(s)]
    largest = max(np.abs(seen).max(initial=0.0), cap or 0.0, scale * most(q) * most(k))
    score = (D + 8) * u * scale * most(q) * most(k) + 8 * u * largest
    weight = 2 * score + (k.shape[1] + 32) * u + r
    size = np.abs(np.asarray(v, dtype=np.float64)).max(initial=0.0)
    smallest = SMALLEST[dtype]
    store = lambda a: 2 * r * np.abs(a) + smallest
    bars = [weight * size + store(out)]
    if grads is not None:
        inner = most(g) * most(v)  # |dP|, and |D|, at most
        through = 4 * u + (2 * score / cap if cap else 0.0)
        each = (weight * 2 * inner + 2 * (D + 8) * u * inner + r * inner + through * 2 * inner + r * 2 * inner) * scale
        columns = p.sum(2)  # (B, HQ, TK): weights a key gets in all
        B, TK, HK = k.shape[:3]
        columns = columns.reshape(B, HK, group, TK).sum(2).transpose(0, 2, 1)[..., None]
        rows = q.shape[1] * group * 2.0**-40  # what weights next to nothing may add
        bars += [each * np.abs(np.asarray(k, np.float64)).max(initial=0.0) + store(grads[0]),
                 each * (columns + rows) * np.abs(np.asarray(q, np.float64)).max() + store(grads[1]),
                 weight * (columns + rows) * np.abs(np.asarray(g, np.float64)).max() + store(grads[2])]
    return bars


def _check(dtype, B, TQ, TK, HQ, HK, D, *, cap=None, bias=False, scale=None, grad_scale=1.0, seed=0, **mask):
    rng = np.random.default_rng([seed, B, TQ, TK, HQ, HK, D])
    make = lambda *shape: rng.standard_normal(shape).astype(dtype)
    q, k, v, g = make(B, TQ, HQ, D), make(B, TK, HK, D), make(B, TK, HK, D), (rng.standard_normal((B, TQ, HQ, D)) * grad_scale).astype(dtype)
    slopes = (2.0 ** -np.arange(1, HQ + 1)).astype(np.float32) if bias else None
    how = dict(scale=scale, cap=cap, slopes=slopes)
    tensors = [mg.device_tensor(a) for a in (q, k, v)]
    out = attention(*tensors, **how, mask=AttentionMask(**mask) if mask else None)
    out.backward(mg.device_tensor(g, constant=True))
    got = [out.data] + [t.grad for t in tensors]
    seen = ora.visible(B, TQ, TK, **mask)
    how["lengths"] = mask.get("lengths")
    want, p, (s, bent) = ora.forward(q, k, v, seen, **how)
    grads = ora.backward(q, k, v, g, seen, **how)
    bars = _bounds(dtype, q, k, v, g, p, s, bent, want, grads, D**-0.5 if scale is None else scale, cap)
    for name, have, exact, bar in zip(("out", "dq", "dk", "dv"), got, (want, *grads), bars):
        assert have.dtype == dtype and have.shape == exact.shape
        over = np.abs(have.astype(np.float64) - exact) - bar
        assert np.isfinite(have).all() and (over <= 0).all(), (name, over.max(), np.unravel_index(over.argmax(), over.shape))
    # a row that sees nothing is zeros, and exactly so
    rows = ~seen.any(-1)
    assert not got[0][rows].any() and not got[1][rows].any()
    assert not got[2][~seen.any(1)].any() and not got[3][~seen.any(1)].any()
    # inference keeps nothing for a gradient and gives the same
    with mg.no_autodiff:
        again = attention(*tensors, scale=scale, cap=cap, slopes=slopes, mask=AttentionMask(**mask) if mask else None)
    over = np.abs(again.data.astype(np.float64) - want) - bars[0]
    assert (over <= 0).all()


DTYPES = [np.float16, np.float32, np.float64]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("TQ,TK,D", [(1, 1, 1), (1, 65, 32), (5, 3, 20), (64, 64, 64), (65, 63, 72), (127, 129, 96), (130, 257, 128), (33, 70, 80),
                                     (70, 33, 40), (40, 66, 192), (66, 40, 256), (31, 31, 7)])
def test_lengths_and_head_dimensions(dtype, TQ, TK, D):
    _check(dtype, 2, TQ, TK, 2, 1, D)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("TQ,TK,D", [(3, 70, 4), (40, 300, 36), (130, 90, 100), (200, 200, 132), (70, 140, 160), (9, 900, 252), (300, 300, 256), (50, 50, 34)])
def test_head_dimensions_that_fill_no_tile(dtype, TQ, TK, D):
    _check(dtype, 1, TQ, TK, 2, 2, D)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("TQ,TK,HQ,HK,D,mask", [
    (900, 900, 8, 1, 64, dict(causal=True)), (700, 700, 6, 2, 128, dict(causal=True, prefix=200)), (1000, 300, 2, 1, 32, dict()),
    (60, 1500, 2, 1, 64, dict()), (100, 800, 4, 2, 96, dict(causal=True)), (640, 640, 4, 1, 256, dict(causal=True, window=100)),
    (500, 500, 4, 1, 80, dict(documents=np.repeat([3, 1, 2, 0], [250, 3, 90, 157])))])
def test_few_heads_over_long_rows(dtype, TQ, TK, HQ, HK, D, mask):
    """Work is split along the keys, or the queries of one key, where there are few blocks of it."""
    _check(dtype, 1, TQ, TK, HQ, HK, D, **mask)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("mask,B,HQ,HK,D", [
    ("causal", 9, 16, 4, 64), ("both-ways", 8, 12, 4, 100), ("prefix", 9, 16, 2, 128), ("documents", 9, 16, 16, 32),
    ("documents-window", 7, 10, 5, 72), ("documents-prefix", 9, 16, 8, 160), ("documents-lengths", 9, 16, 4, 128), ("none", 5, 14, 2, 36)])
def test_many_heads(dtype, mask, B, HQ, HK, D):
    """Enough blocks of 128 queries for half the compute units, and more."""
    how = {**MASKS, "none": {}}[mask]
    if mask == "documents-lengths":
        how = {**how, "lengths": [150 - 9 * b for b in range(B)]}
    _check(dtype, B, 150, 150, HQ, HK, D, cap=4.0 if mask in ("prefix", "documents") else None, bias=mask == "both-ways", **how)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("B", [8, 9])
@pytest.mark.parametrize("bad", [np.nan, np.inf, "lowest"])
def test_many_heads_beside_documents_of_no_numbers(dtype, B, bad):
    bad = np.finfo(dtype).min if bad == "lowest" else bad
    rng = np.random.default_rng(B)
    T, H, D = 140, 16, 64
    ops = [rng.standard_normal((B, T, H, D)).astype(dtype) for _ in range(4)]
    documents = np.repeat([0, 1, 2], [50, 40, 50])
    results = []
    for spoil in (False, True):
        if spoil:
            ops = [a.copy() for a in ops]
            for a in ops:
                a[:, 50:90] = bad
        tensors = [mg.device_tensor(a) for a in ops]
        out = attention(*tensors[:3], mask=AttentionMask(causal=True, documents=documents))
        out.backward(tensors[3])
        results.append([out.data] + [t.grad for t in tensors[:3]])
    rows = documents != 1
    for clean, dirty in zip(*results):
        assert np.isfinite(dirty[:, rows]).all()
        assert np.allclose(dirty[:, rows], clean[:, rows], rtol=4 * UNIT[dtype][1], atol=max(64 * UNIT[dtype][1], 1024 * UNIT[dtype][0]))


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_mask_for_several_shapes(dtype):
    rng = np.random.default_rng(41)
    mask = AttentionMask(causal=True, lengths=[40, 3])
    for TQ, TK, HQ, HK, D in ((8, 50, 2, 1, 32), (50, 40, 4, 2, 64), (8, 50, 2, 1, 32)):
        q, k, v = (rng.standard_normal(shape).astype(dtype) for shape in ((2, TQ, HQ, D), (2, TK, HK, D), (2, TK, HK, D)))
        seen = ora.visible(2, TQ, TK, causal=True, lengths=[40, 3])
        want, p, (s, bent) = ora.forward(q, k, v, seen, lengths=[40, 3])
        bar = _bounds(dtype, q, k, v, None, p, s, bent, want, None, D**-0.5, None)[0]
        assert (np.abs(attention(q, k, v, mask=mask).data.astype(np.float64) - want) <= bar).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("HQ,HK", [(1, 1), (3, 3), (6, 2), (8, 1)])
def test_heads_that_share_keys(dtype, HQ, HK):
    _check(dtype, 3, 70, 70, HQ, HK, 64, causal=True)


MASKS = {
    "causal": dict(causal=True),
    "window": dict(causal=True, window=37),
    "both-ways": dict(window=20),
    "one": dict(causal=True, window=1),
    "prefix": dict(causal=True, prefix=50),
    "prefixes": dict(causal=True, prefix=[0, 131]),
    "lengths": dict(lengths=[150, 0]),
    "causal-lengths": dict(causal=True, lengths=[33, 97]),
    "documents": dict(documents=np.repeat([4, 0, 9, 2], [40, 1, 59, 50])),
    "causal-documents": dict(causal=True, documents=np.stack([np.repeat([0, 1, 2], [64, 64, 22]), np.repeat([5, -1, 3], [10, 40, 100])])),
    "documents-window": dict(causal=True, window=16, documents=np.repeat([0, 1], [65, 85])),
    "documents-prefix": dict(causal=True, prefix=20, documents=np.repeat([0, -7, 1], [70, 5, 75])),
    "documents-lengths": dict(causal=True, lengths=[100, 64], documents=np.repeat([0, 1, 2], [70, 40, 40])),
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mask", MASKS)
def test_masks(dtype, mask):
    _check(dtype, 2, 150, 150, 2, 1, 32, **MASKS[mask])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("TQ,TK,mask", [(9, 150, "causal"), (150, 9, "causal"), (20, 150, "window"), (1, 150, "causal-lengths"), (7, 150, "prefixes"),
                                        (130, 150, "causal-documents"), (64, 150, "lengths"), (200, 150, "both-ways")])
def test_masks_with_other_numbers_of_queries_than_keys(dtype, TQ, TK, mask):
    _check(dtype, 2, TQ, TK, 4, 2, 64, **MASKS[mask])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mask", [dict(), dict(causal=True), dict(causal=True, prefix=40)])
@pytest.mark.parametrize("cap,bias,scale", [(5.0, False, None), (None, True, None), (3.0, True, 0.4), (0.05, False, 3.0)])
def test_cap_bias_and_scale(dtype, mask, cap, bias, scale):
    _check(dtype, 2, 90, 90, 4, 2, 64, cap=cap, bias=bias, scale=scale, **mask)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("grad_scale", [1e-4, 300.0])
def test_gradients_of_any_size(dtype, grad_scale):
    """A small loss in float16: weights and gradients of scores lie far below what float16 resolves."""
    if dtype == np.float16 and grad_scale > 1:
        grad_scale = 30.0  # what dk sums to is representable
    _check(dtype, 1, 300, 300, 2, 2, 64, causal=True, grad_scale=grad_scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_rows(dtype):
    _check(dtype, 1, 3, 5003, 2, 1, 64, causal=True)
    _check(dtype, 1, 700, 1100, 1, 1, 128, causal=True, window=300)


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_same_bits_every_time(dtype):
    rng = np.random.default_rng(5)
    q, k, v, g = (mg.device_tensor(rng.standard_normal((2, 200, h, 64)).astype(dtype)) for h in (4, 2, 2, 4))
    runs = []
    for _ in range(3):
        out = attention(q, k, v, cap=10.0, mask=AttentionMask(causal=True))
        out.backward(g)
        runs.append([out.data.copy()] + [t.grad.copy() for t in (q, k, v)])
    for run in runs[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(runs[0], run))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, "lowest"])
@pytest.mark.parametrize("D", [64, 192])
def test_what_a_query_does_not_see_does_not_touch_it(dtype, bad, D):
    """Values in masked places: behind the lengths, in other documents of the same tiles, and in the future."""
    bad = np.finfo(dtype).min if bad == "lowest" else bad
    rng = np.random.default_rng(8)
    B, T, H = 2, 140, 2
    q, k, v, g = (rng.standard_normal((B, T, H, D)).astype(dtype) for _ in range(4))
    for mask, keys, queries in (
        (dict(lengths=[90, 0]), (slice(None), slice(90, None)), None),
        (dict(causal=True, documents=np.repeat([0, 1, 2], [50, 40, 50])), (slice(None), slice(50, 90)), (slice(None), slice(50, 90))),
        (dict(causal=True), (slice(None), slice(135, None)), (slice(None), slice(135, None))),
    ):
        spoilt = [a.copy() for a in (q, k, v, g)]
        spoilt[1][keys] = bad
        spoilt[2][keys] = bad
        if queries is not None:  # what stands at the same places: other rows' gradients stay clean
            spoilt[0][queries] = bad
            spoilt[3][queries] = bad
        results = []
        for ops in ((q, k, v, g), spoilt):
            tensors = [mg.device_tensor(a) for a in ops]
            out = attention(*tensors[:3], mask=AttentionMask(**mask))
            out.backward(tensors[3])
            results.append([out.data] + [t.grad for t in tensors[:3]])
        seen = ora.visible(B, T, T, **mask)
        rows = np.ones((B, T), dtype=bool)
        if queries is not None:
            rows[queries] = False
        columns = np.ones((B, T), dtype=bool)
        columns[keys] = False
        if mask == dict(causal=True):
            columns[:] = False  # the last queries see every key
        clean, dirty = results
        for n, where in ((0, rows), (1, rows), (2, columns), (3, columns)):
            assert np.isfinite(dirty[n][where]).all(), n
            assert np.allclose(dirty[n][where], clean[n][where], rtol=4 * UNIT[dtype][1], atol=max(64 * UNIT[dtype][1], 1024 * UNIT[dtype][0]))
        assert not dirty[0][~seen.any(-1)].any()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("T,D", [(700, 36), (600, 128), (20, 64), (20, 100)])
def test_documents_of_no_numbers_beside_others_where_work_is_split(dtype, T, D):
    rng = np.random.default_rng([T, D])
    HQ, HK = 4, 1
    q, k, v, g = (rng.standard_normal((1, T, H, D)).astype(dtype) for H in (HQ, HK, HK, HQ))
    middle = slice(T // 3, T // 2)
    documents = np.zeros(T, dtype=np.int64)
    documents[middle], documents[T // 2:] = 1, 2
    results = []
    for spoil in (False, True):
        ops = [a.copy() for a in (q, k, v, g)]
        if spoil:
            for a in ops:
                a[:, middle] = np.nan
        tensors = [mg.device_tensor(a) for a in ops]
        out = attention(*tensors[:3], mask=AttentionMask(causal=True, documents=documents))
        out.backward(tensors[3])
        results.append([out.data] + [t.grad for t in tensors[:3]])
    rows = documents != 1
    for clean, dirty in zip(*results):
        assert np.isnan(dirty[0, ~rows]).any() and np.isfinite(dirty[0, rows]).all()
        assert np.allclose(dirty[0, rows], clean[0, rows], rtol=4 * UNIT[dtype][1], atol=max(64 * UNIT[dtype][1], 1024 * UNIT[dtype][0]))


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_and_nan_in_sight(dtype):
    rng = np.random.default_rng(9)
    q, k, v = (rng.standard_normal((1, 80, 1, 64)).astype(dtype) for _ in range(3))
    v[0, 40, 0, 3] = np.nan
    v[0, 50, 0, 5] = np.inf
    out = attention(q, k, v, mask=AttentionMask(causal=True)).data[0, :, 0]
    assert np.isfinite(out[:40]).all()
    assert np.isnan(out[40:, 3]).all() and np.isfinite(np.delete(out[40:], [3, 5], axis=1)).all()
    assert np.isfinite(out[:50, 5]).all() and np.isposinf(out[50:, 5]).all()


def test_gradients_reach_only_what_wants_them():
    rng = np.random.default_rng(1)
    q, k, v = (rng.standard_normal((1, 20, 2, 16)) for _ in range(3))
    g = rng.standard_normal(q.shape)
    seen = ora.visible(1, 20, 20)
    want = ora.backward(q, k, v, g, seen)
    for wanted in ((0,), (1,), (2,), (0, 2)):
        tensors = [mg.tensor(a, constant=n not in wanted) for n, a in enumerate((q, k, v))]
        attention(*tensors).backward(g)
        for n, t in enumerate(tensors):
            assert (t.grad is None) == (n not in wanted)
            if n in wanted:
                assert np.allclose(t.grad, want[n], rtol=0, atol=1e-12)
    x = mg.tensor(q)  # one tensor in three places gets the sum
    attention(x, x, x).backward(g)
    assert np.allclose(x.grad, sum(ora.backward(q, q, q, g, seen)), rtol=0, atol=1e-12)
    assert attention(q, k, v).constant


def test_differences():
    """The gradient against differences of the operation's own results."""
    rng = np.random.default_rng(2)
    q, k, v, g = rng.standard_normal((1, 9, 4, 8)), rng.standard_normal((1, 11, 2, 8)), rng.standard_normal((1, 11, 2, 8)), rng.standard_normal((1, 9, 4, 8))
    how = dict(cap=2.0, slopes=np.array([0.5, 0.25, 0.1, 0.0]), mask=AttentionMask(causal=True, prefix=4))
    tensors = [mg.tensor(a) for a in (q, k, v)]
    attention(*tensors, **how).backward(g)
    f = lambda *ops: float((attention(*ops, **how).data * g).sum())
    for n in range(3):
        for index in rng.permutation((q, k, v)[n].size)[:6]:
            up, down = [a.copy() for a in (q, k, v)], [a.copy() for a in (q, k, v)]
            up[n].flat[index] += 1e-6
            down[n].flat[index] -= 1e-6
            assert abs((f(*up) - f(*down)) / 2e-6 - tensors[n].grad.flat[index]) < 1e-7


# ------------------------------------------------------------------------------------------------- the cache
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("HQ,HK,D,T", [(4, 1, 64, 1), (8, 8, 128, 1), (6, 2, 72, 3), (16, 1, 96, 5), (2, 1, 7, 2), (32, 4, 128, 8), (2, 2, 200, 1)])
@pytest.mark.parametrize("more", [dict(), dict(cap=4.0), dict(bias=True)])
def test_a_cache_gives_what_attention_over_its_tokens_gives(dtype, HQ, HK, D, T, more):
    rng = np.random.default_rng([HQ, HK, D, T])
    lengths = np.array([T, 300, 64, 65, 129])
    B, capacity = lengths.size, 310
    make = lambda *shape: rng.standard_normal(shape).astype(dtype)
    keys, values, q = make(B, capacity, HK, D), make(B, capacity, HK, D), make(B, T, HQ, D)
    cache = KeyValueCache(B, capacity, HK, D, dtype=dtype)
    assert not cache.keys.host().any() and not cache.values.host().any()
    old = lengths - T
    for n in range(0, int(old.max()), 100):  # the histories, in pieces; places behind a length hold what no one may look at
        piece = slice(n, min(n + 100, int(old.max())))
        cache.write(keys[:, piece], values[:, piece], AttentionMask(lengths=piece.stop))
    junk = np.full((B, capacity, HK, D), np.nan, dtype=dtype)
    for b, n in enumerate(old):
        junk[b, :n] = keys[b, :n]
    cache.write(junk, junk, AttentionMask(lengths=capacity))
    junk_v = junk.copy()
    for b, n in enumerate(old):
        junk_v[b, :n] = values[b, :n]
    cache.write(junk, junk_v, AttentionMask(lengths=capacity))
    new_k, new_v = make(B, T, HK, D), make(B, T, HK, D)
    mask = AttentionMask(causal=True, lengths=lengths)
    cache.write(mg.tensor(new_k), mg.device_tensor(new_v), mask)
    for b, n in enumerate(old):
        keys[b, n:n + T], values[b, n:n + T] = new_k[b], new_v[b]
        assert np.array_equal(cache.keys.host()[b, :n + T], keys[b, :n + T]) and np.array_equal(cache.values.host()[b, :n + T], values[b, :n + T])
    slopes = (2.0 ** -np.arange(1, HQ + 1)).astype(np.float32) if more.get("bias") else None
    how = dict(cap=more.get("cap"), slopes=slopes)
    out = cache.attend(q, mask=mask, **how)
    assert out.constant and out.dtype == dtype
    seen = ora.visible(B, T, capacity, causal=True, lengths=lengths)
    clean_k, clean_v = (np.where(np.arange(capacity)[None, :, None, None] < lengths[:, None, None, None], a, 0).astype(dtype) for a in (keys, values))
    want, p, (s, bent) = ora.forward(q, clean_k, clean_v, seen, lengths=lengths, **how)
    bar = _bounds(dtype, q, clean_k, clean_v, None, p, s, bent, want, None, D**-0.5, more.get("cap"))[0]
    over = np.abs(out.data.astype(np.float64) - want) - bar
    assert (over <= 0).all(), over.max()


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_long_history_among_short_ones(dtype):
    rng = np.random.default_rng(77)
    lengths, capacity = np.array([1, 20011, 0, 4097]), 20011
    B, HQ, HK, D = 4, 8, 2, 64
    make = lambda *shape: rng.standard_normal(shape).astype(dtype)
    keys, values, q = make(B, capacity, HK, D), make(B, capacity, HK, D), make(B, 1, HQ, D)
    cache = KeyValueCache(B, capacity, HK, D, dtype=dtype)
    cache.write(keys, values, AttentionMask(lengths=capacity))
    how = dict(mask=AttentionMask(causal=True, lengths=lengths))
    out = cache.attend(q, **how).data
    assert np.array_equal(out, cache.attend(q, **how).data)
    for b, n in enumerate(lengths):
        if n == 0:
            assert not out[b].any()
            continue
        k, v = keys[b:b + 1, :n], values[b:b + 1, :n]
        seen = np.ones((1, 1, n), dtype=bool)
        want, p, (s, bent) = ora.forward(q[b:b + 1], k, v, seen)
        bar = _bounds(dtype, q[b:b + 1], k, v, None, p, s, bent, want, None, D**-0.5, None)[0]
        assert (np.abs(out[b:b + 1].astype(np.float64) - want) <= bar).all()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("HK,D", [(1, 128), (1, 7)])
def test_offsets_beyond_32_bits(dtype, HK, D):
    """The last tokens of a cache with more than 2^32 bytes and, at 128 values a head, 2^31 values."""
    rng = np.random.default_rng(D)
    capacity = (1 << 24) + 77 if D == 128 else (1 << 32) // (D * np.dtype(dtype).itemsize) + 1000
    seen_tokens, T = 300, 2
    cache = KeyValueCache(1, capacity, HK, D, dtype=dtype)
    make = lambda *shape: rng.standard_normal(shape).astype(dtype)
    k, v, q = make(1, seen_tokens, HK, D), make(1, seen_tokens, HK, D), make(1, T, 2 * HK, D)
    cache.write(k, v, AttentionMask(causal=True, lengths=[capacity]))
    out = cache.attend(q, mask=AttentionMask(causal=True, window=seen_tokens - T, lengths=[capacity])).data
    seen = ora.visible(1, T, seen_tokens, causal=True, window=seen_tokens - T)
    want, p, (s, bent) = ora.forward(q, k, v, seen)
    bar = _bounds(dtype, q, k, v, None, p, s, bent, want, None, D**-0.5, None)[0]
    assert (np.abs(out.astype(np.float64) - want) <= bar).all()


def test_cache_refusals():
    cache = KeyValueCache(2, 10, 2, 16, dtype=np.float32)
    x = np.ones((2, 3, 2, 16), dtype=np.float32)
    for bad in (
        lambda: cache.write(x, x, AttentionMask(causal=True)),  # no lengths
        lambda: cache.write(x, x, AttentionMask(lengths=11)),
        lambda: cache.write(x, x, AttentionMask(lengths=[2, 5])),  # three tokens do not end at two
        lambda: cache.write(x, x[:, :2], AttentionMask(lengths=5)),
        lambda: cache.write(x[:1], x[:1], AttentionMask(lengths=5)),
        lambda: cache.write(x[:, :, :1], x[:, :, :1], AttentionMask(lengths=5)),
        lambda: cache.attend(x[:, :, :1], mask=AttentionMask(lengths=5)),
        lambda: cache.attend(x, mask=AttentionMask()),
        lambda: cache.attend(x[..., :8], mask=AttentionMask(lengths=5)),
        lambda: cache.attend(x, mask=AttentionMask(lengths=5), cap=-2.0),
    ):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: cache.write(x.astype(np.float64), x, AttentionMask(lengths=5)), lambda: cache.attend(x, mask=None)):
        with pytest.raises(TypeError):
            bad()
    assert not cache.keys.host().any()


def test_entry_points_refuse_bad_descriptors():
    from mygrad_amd import _device, _hip

    lib, buf = _hip.lib(), _device.DeviceBuffer(1 << 16)
    good = dict(dtype=0, causal=1, B=1, TQ=4, TK=4, HQ=2, HK=1, D=16, window=0, scale=0.25, cap=0.0)
    for status, change in ((-2, dict(dtype=3)), (-1, dict(HK=0)), (-1, dict(HQ=3, HK=2)), (-1, dict(TQ=-1)), (-2, dict(D=257)), (-2, dict(TK=1 << 30)),
                           (-2, dict(B=1 << 20, TQ=1 << 20)), (-1, dict(window=-1)), (-1, dict(scale=float("nan"))), (-1, dict(cap=-1.0)),
                           (-1, dict(starts=buf.ptr)), (-1, dict(window=2, prefix=buf.ptr))):
        desc = _hip.AttentionDesc(**{**good, **change})
        assert lib.mg_attention_fwd(desc, *[buf.ptr] * 6) == status, change
        assert lib.mg_attention_bwd(desc, *[buf.ptr] * 10) == status, change
    desc = _hip.AttentionDesc(**good)
    assert lib.mg_attention_fwd(desc, None, *[buf.ptr] * 5) == -1
    assert lib.mg_attention_fwd(None, *[buf.ptr] * 6) == -1
    assert lib.mg_attention_bwd(desc, *[buf.ptr] * 9, None) == -1  # dk without dv
    assert lib.mg_cache_write(5, 1, 1, 1, 1, *[buf.ptr] * 5) == -2
    assert lib.mg_cache_write(0, 1, -1, 1, 1, *[buf.ptr] * 5) == -1
    assert lib.mg_cache_write(0, 1, 1, 1, 1, None, *[buf.ptr] * 4) == -1
