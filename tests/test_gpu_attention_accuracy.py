"""How near attention and its gradients come to their formulas in 64 bits."""

import time

import numpy as np
import pytest

import mygrad_amd as mg
from mygrad_amd import _hip
from mygrad_amd.nnet import AttentionMask, RotaryTable, attention, head_norm
from oracle import attention as ora
from tests.attention_bars import CASES, Formulas, bars_of, formulas_and_bars, name_of, operands

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    if not mg.is_available():
        pytest.fail("libmygrad_hip.so / gfx950 device not available: the GPU tests need both")


def run(q, k, v, g, mask=None, **how):
    """out, dq, dk and dv as host arrays."""
    tensors = [mg.device_tensor(a) for a in (q, k, v)]
    out = attention(*tensors, mask=None if mask is None else AttentionMask(**mask), **how)
    out.backward(mg.device_tensor(g, constant=True))
    return [out.data] + [t.grad for t in tensors]


@pytest.mark.parametrize("B,TQ,TK,HQ,HK,D,cap,mask", [
    (9, 150, 150, 16, 4, 64, None, dict(causal=True)), (9, 150, 150, 16, 16, 128, 20.0, dict()), (3, 300, 200, 16, 8, 72, None, dict()),
    (5, 300, 300, 16, 2, 256, None, dict(causal=True)), (1, 700, 700, 4, 1, 128, None, dict(causal=True)), (2, 20, 900, 8, 2, 96, 20.0, dict())])
def test_float16_results_are_rounded_once(B, TQ, TK, HQ, HK, D, cap, mask):
    """A result is off by its own rounding to float16, e.  What else there is -- sums, exponentials and scores in 32 bits, weights and their
    gradients in two parts of float16 -- is some 2^-16 of it or less next to e of 2^-12.3, and adds in squares: 1% of e; twice that is allowed."""
    rng = np.random.default_rng([B, TQ, D])
    q, k, v, g = (rng.standard_normal(shape).astype(np.float16) for shape in ((B, TQ, HQ, D), (B, TK, HK, D), (B, TK, HK, D), (B, TQ, HQ, D)))
    seen = ora.visible(B, TQ, TK, **mask)
    exact = ora.forward(q, k, v, seen, cap=cap)[0], *ora.backward(q, k, v, g, seen, cap=cap)
    rms = lambda a: np.sqrt((a * a).mean())
    for name, have, want in zip(("out", "dq", "dk", "dv"), run(q, k, v, g, mask, cap=cap), exact):
        rounding = rms(want.astype(np.float16).astype(np.float64) - want)
        assert rms(have.astype(np.float64) - want) <= 1.02 * rounding, (name, rms(have - want) / rounding)


@pytest.mark.parametrize("dtype", [np.float16, np.float32, np.float64])
@pytest.mark.parametrize("as_tensor", [False, True])
def test_slopes_that_are_no_powers_of_two(dtype, as_tensor):
    """In float64 they keep their digits; the other types take them in float32."""
    rng = np.random.default_rng(12)
    q, k, v, g = (rng.standard_normal((1, 600, 12, 16)).astype(dtype) for _ in range(4))
    slopes = 2.0 ** (-8.0 * np.arange(1, 13) / 12)
    held = slopes if dtype == np.float64 else slopes.astype(np.float32)
    seen = ora.visible(1, 600, 600, causal=True)
    results = run(q, k, v, g, dict(causal=True), slopes=mg.tensor(slopes, constant=True) if as_tensor else slopes)
    for have, (want, bar) in zip(results, formulas_and_bars(dtype, q, k, v, g, seen, slopes=held)):
        assert (np.abs(have.astype(np.float64) - want) <= bar).all()


@pytest.mark.parametrize("dtype,TQ,cap,scale", [
    (np.float64, 40, 1e-50, None), (np.float64, 40, 1e40, None), (np.float32, 300, 1e-30, None), (np.float16, 300, 1e-30, None), (np.float32, 9, 1e-30, 1e20),
    (np.float32, 40, 1e30, None), (np.float16, 300, 1e30, None)])
def test_smallest_and_largest_caps(dtype, TQ, cap, scale):
    """Scores next to zero give the mean, behind the largest caps what no cap gives; rows of zeros among the queries."""
    rng = np.random.default_rng(TQ)
    q, k, v = (rng.standard_normal((9, TQ, 8, 32)).astype(dtype) for _ in range(3))
    q[:, ::7] = 0
    out = attention(q, k, v, cap=cap, scale=scale).data.astype(np.float64)
    seen = ora.visible(9, TQ, TQ)
    zeros = np.zeros_like(q)
    want, bar = formulas_and_bars(dtype, zeros if cap < 1 else q, k, v, zeros, seen)[0]
    assert (np.abs(out - want) <= bar).all()


def test_entry_points_refuse_scores_beyond_single_precision():
    from mygrad_amd import _device

    lib, buf = _hip.lib(), _device.DeviceBuffer(1 << 16)
    for dtype, status in ((0, -2), (2, -2), (1, 0)):
        for how in (dict(scale=0.25, cap=1e-50), dict(scale=0.25, cap=1e39), dict(scale=1e39, cap=0.0)):
            desc = _hip.AttentionDesc(dtype=dtype, B=1, TQ=4, TK=4, HQ=2, HK=1, D=16, **how)
            assert lib.mg_attention_fwd(desc, buf.ptr, buf.ptr, buf.ptr, buf.ptr + 8192, None, None) == status, (dtype, how)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("causal", [False, True])
def test_the_largest_window_is_none(dtype, causal):
    """With documents, whose tiles are sorted by an estimate of what they see."""
    rng = np.random.default_rng(3)
    q, k, v, g = (rng.standard_normal((9, 400, 16, 32)).astype(dtype) for _ in range(4))
    documents = np.repeat([0, 1, 2], [150, 30, 220])
    without = run(q, k, v, g, dict(causal=causal, documents=documents))
    for window in (400, 1 << 30, 1 << 40):
        for a, b in zip(without, run(q, k, v, g, dict(causal=causal, documents=documents, window=window))):
            assert np.array_equal(a, b)


def arguments(case, how):
    return {name: how[name] for name in ("scale", "cap", "slopes")}


@pytest.mark.parametrize("case", CASES, ids=name_of)
def test_results_within_their_bars(case):
    arrays, seen, how = operands(case)
    f = Formulas(*arrays, seen, **how)
    for name, have, want, bar in zip(("out", "dq", "dk", "dv"), run(*arrays, case["mask"], **arguments(case, how)), f.results, bars_of(case["dtype"], f)):
        over = np.abs(have.astype(np.float64) - want) - bar
        assert have.dtype == case["dtype"] and (over <= 0).all(), (name, over.max(), np.unravel_index(over.argmax(), over.shape))


EACH_WAY = [(1, 700, 4, 1, 36), (1, 600, 4, 1, 128), (1, 20, 4, 1, 100), (2, 140, 2, 2, 192), (9, 140, 16, 16, 64), (8, 140, 16, 4, 72)]


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, "lowest"])
@pytest.mark.parametrize("dtype,B,T,HQ,HK,D", [*((dtype, *shape) for dtype in (np.float16, np.float32) for shape in EACH_WAY),
                                               *((np.float64, *shape) for shape in EACH_WAY[:4])])
def test_beside_documents_of_no_numbers_results_are_within_their_bars(dtype, bad, B, T, HQ, HK, D):
    """What other documents of the same tiles hold changes nothing: the bars are those of the operands that are seen."""
    case = dict(dtype=dtype, shape=(B, T, T, HQ, HK, D), cap=None, bias=False, scale=None, grad_scale=1.0)
    documents = np.repeat([0, 1, 2], [T // 3, T // 2 - T // 3, T - T // 2])
    arrays, seen, how = operands(dict(case, mask=dict(causal=True, documents=documents)))
    f = Formulas(*arrays, seen, **how)
    spoilt = [a.copy() for a in arrays]
    for a in spoilt:
        a[:, documents == 1] = np.finfo(dtype).min if bad == "lowest" else bad
    rows = documents != 1
    for name, have, want, bar in zip(("out", "dq", "dk", "dv"), run(*spoilt, dict(causal=True, documents=documents)), f.results, bars_of(dtype, f)):
        over = (np.abs(have.astype(np.float64) - want) - bar)[:, rows]
        assert (over <= 0).all(), (name, np.nanmax(over), np.isnan(over).sum())


def test_float16_through_other_operations():
    """Bit for bit what the parts give one by one: a norm of heads before attention, one tensor in three places behind it."""
    rng = np.random.default_rng(31)
    x, w, g = (rng.standard_normal(shape).astype(np.float16) for shape in ((2, 40, 4, 32), (32,), (2, 40, 4, 32)))
    rotary = RotaryTable(16, 40).at(np.arange(40))
    tx, tw = mg.device_tensor(x), mg.device_tensor(w)
    y = head_norm(tx, tw, eps=1e-6, rotary=rotary)
    out = attention(y, y, y, mask=AttentionMask(causal=True))
    out.backward(mg.device_tensor(g, constant=True))
    leaf = y.data.copy()
    alone, dq, dk, dv = run(leaf, leaf, leaf, g, dict(causal=True))
    assert np.array_equal(out.data, alone)
    ux, uw = mg.device_tensor(x), mg.device_tensor(w)
    head_norm(ux, uw, eps=1e-6, rotary=rotary).backward(mg.device_tensor((dq + dk) + dv, constant=True))
    assert tx.grad.dtype == np.float16 and np.array_equal(tx.grad, ux.grad) and np.array_equal(tw.grad, uw.grad)


def milliseconds(operands, grad, mask):
    """Shortest of four forward and backward passes."""
    tensors, grad, best = [mg.device_tensor(a) for a in operands], mg.device_tensor(grad, constant=True), [np.inf, np.inf]
    for _ in range(4):
        at = []
        for step in (lambda: None, lambda: attention(*tensors, mask=mask), lambda: out.backward(grad)):
            out = step()
            _hip.synchronize()
            at.append(1e3 * time.perf_counter())
        best = [min(b, t) for b, t in zip(best, np.diff(at))]
    return best


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("B,T,HQ,HK,D", [(2, 2048, 8, 2, 64), (1, 700, 4, 1, 128), (2, 1500, 8, 8, 36)])
def test_an_overflow_costs_a_step_what_numbers_do(dtype, B, T, HQ, HK, D):
    """An upstream gradient of infinities (a scaled loss that overflowed), in all or in some values, operands that are no numbers, and a value of the
    first key that is infinite: every row of a block is no number by what it sees.  A row at a time they took 30 to 260 times as long; five times
    are allowed here."""
    rng = np.random.default_rng(T)
    q, k, v, g = (rng.standard_normal((B, T, heads, D)).astype(dtype) for heads in (HQ, HK, HK, HQ))
    mask = AttentionMask(causal=True)

    some = g.copy()
    some[:, T // 2:, :, 3] = np.inf
    clean = milliseconds((q, k, v), g, mask)
    one = v.copy()
    one[:, 0, :, 5] = np.inf
    for operands, grad in (((q, k, v), np.full_like(g, np.inf)), ((q, k, v), some), ([np.full_like(a, np.nan) for a in (q, k, v)], g), ((q, k, one), g),
                           ((q, k, np.full_like(v, np.nan)), g)):
        for way, spoilt in zip(clean, milliseconds(operands, grad, mask)):
            assert spoilt < 0.3 + 5 * way, (way, spoilt)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("B,T,HQ,HK,D", EACH_WAY)
def test_infinite_gradients_of_some_queries_and_values(dtype, B, T, HQ, HK, D):
    """dv of a key is no number where a query that sees it has none, and nowhere else; dk and dq wherever such a query has a part in them."""
    case = dict(dtype=dtype, shape=(B, T, T, HQ, HK, D), mask=dict(causal=True), cap=None, bias=False, scale=None, grad_scale=1.0)
    (q, k, v, g), seen, how = operands(case)
    f = Formulas(q, k, v, g, seen, **how)
    spoilt = g.copy()
    at, heads = [2, T // 2, T // 2 + 1], slice(HQ - 1, HQ)
    spoilt[:, at, heads, 1:3] = np.inf
    out, dq, dk, dv = run(q, k, v, spoilt, case["mask"])
    bars = bars_of(dtype, f)
    finite_q = np.ones(q.shape, bool)
    finite_q[:, at, heads] = False
    finite_k, finite_v = np.ones(k.shape, bool), np.ones(k.shape, bool)
    finite_k[:, :max(at) + 1, HK - 1] = False
    finite_v[:, :max(at) + 1, HK - 1, 1:3] = False
    for have, which, finite in ((out, 0, np.ones(q.shape, bool)), (dq, 1, finite_q), (dk, 2, finite_k), (dv, 3, finite_v)):
        assert np.array_equal(np.isfinite(have), finite), which
        over = np.abs(np.where(finite, have, 0).astype(np.float64) - np.where(finite, f.results[which], 0)) - bars[which]
        assert (over <= 0).all(), (which, over.max())


@pytest.mark.parametrize("dtype,B,T,HQ,HK,D", [*((dtype, *shape) for dtype in (np.float16, np.float32) for shape in EACH_WAY),
                                               *((np.float64, *shape) for shape in EACH_WAY[:4])])
@pytest.mark.parametrize("many", [False, True])
def test_values_that_are_no_numbers_reach_the_rows_that_see_them(dtype, B, T, HQ, HK, D, many):
    """In their places: an infinity as one, NaN or infinities of both signs as NaN; all others are as if those keys held numbers."""
    case = dict(dtype=dtype, shape=(B, T, T, HQ, HK, D), mask=dict(causal=True), cap=None, bias=False, scale=None, grad_scale=1.0)
    (q, k, v, g), seen, how = operands(case)
    f = Formulas(q, k, v, g, seen, **how)
    want, bar = f.results[0], bars_of(dtype, f)[0]
    spoilt = v.copy()
    if many:  # each key from a third of the row on, in some places
        spoilt[:, T // 3:, HK - 1, 1] = np.inf
        spoilt[:, T // 3::2, HK - 1, 2] = -np.inf
        spoilt[:, T // 2, HK - 1, 2] = np.nan
    else:
        spoilt[:, T // 3, HK - 1, 1] = np.inf
        spoilt[:, T // 3, HK - 1, 2] = -np.inf
        spoilt[:, T // 2, HK - 1, 2:4] = np.nan, np.inf
        spoilt[:, T // 2 + 1, HK - 1, 3] = -np.inf
    held = np.where(np.isfinite(spoilt), 0, spoilt).astype(np.float64)
    ups, downs = ((seen[:, :, :, None, None] & test[:, None]).any(2) for test in (~(held <= 0), ~(held >= 0)))
    expected = np.repeat(np.where(ups & downs, np.nan, np.where(ups, np.inf, np.where(downs, -np.inf, 0))), HQ // HK, axis=2)
    with mg.no_autodiff:
        out = attention(q, k, spoilt, mask=AttentionMask(causal=True)).data
    odd = expected != 0
    assert np.array_equal(out[odd].astype(np.float64), expected[odd], equal_nan=True)
    over = np.abs(np.where(odd, 0, out).astype(np.float64) - np.where(odd, 0, want)) - bar
    assert (over <= 0).all(), over.max()
