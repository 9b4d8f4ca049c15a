"""Layer norm against its formulas in 64 bits.

Bars: u is the unit of the sums (2^-24, 2^-53 for float64), r that of the type results are rounded to.  A sum over a row of D values is off by
less than (D / 16 + 16) u of the sum of their magnitudes (sixteen lanes or more add side by side): the mean by that of mean|x|, delta.  What is
left of x is rounded by u of itself and its own mean is off by (D / 16 + 16) u of the mean of its magnitudes, so x - mu is off by
(D / 16 + 20) u (|x - mu| + mean|x - mu| + 2 delta); 1 / sqrt by half of (D / 16 + 16) u (1 + delta^2 / var), and by 4 u.  The sums over rows add at
most 256 rows in turn in single precision."""

import numpy as np
import pytest

import mygrad_amd as mg
from mygrad_amd.nnet import layer_norm
from oracle import language as ora

pytestmark = pytest.mark.gpu

UNIT = {np.float16: (2.0**-24, 2.0**-11), np.float32: (2.0**-24, 2.0**-24), np.float64: (2.0**-53, 2.0**-53)}
SMALLEST = {np.float16: 2.0**-24, np.float32: 2.0**-126, np.float64: 2.0**-1022}
DTYPES = [np.float16, np.float32, np.float64]


@pytest.fixture(scope="module", autouse=True)
def device():
    if not mg.is_available():
        pytest.fail("libmygrad_hip.so / gfx950 device not available: the GPU tests need both")


def outside(have, want, bar):
    return int((~(np.abs(have - want) <= bar)).sum())


def bars(dtype, x, w, b, g, eps):
    """Of y, dx, dw and db, with what they should be."""
    u, r = UNIT[dtype]
    x, w, g = x.astype(ora.WIDE), np.ones(x.shape[-1]) if w is None else w.astype(ora.WIDE), g.astype(ora.WIDE)
    b = np.zeros(x.shape[-1]) if b is None else b.astype(ora.WIDE)
    want = ora.layer_norm(x, w, b, eps, g)
    dim, size = x.shape[-1], lambda a: np.abs(a).mean(-1, keepdims=True)
    chain = dim / 16 + 16
    middle = x - x.mean(-1, keepdims=True)
    inv = 1 / np.sqrt((middle**2).mean(-1, keepdims=True) + eps)
    n, delta = middle * inv, (chain * u) * size(x)
    off = inv * (chain + 4) * u * (np.abs(middle) + size(middle) + 2 * delta)
    rel = (chain / 2 + 8) * u * (1 + (delta * inv) ** 2)
    dn = off + np.abs(n) * rel
    y = np.abs(w) * dn + 4 * u * (np.abs(w * n) + np.abs(b))
    v = g * w
    mix = (v * n).mean(-1, keepdims=True)
    dx = inv * ((chain + 4) * u * size(v) + np.abs(n) * ((chain + 4) * u * size(v * n) + size(np.abs(v) * dn)) + dn * np.abs(mix)
                + 4 * u * (np.abs(v) + size(v) + np.abs(n * mix))) + rel * np.abs(want[1])
    rows = tuple(range(x.ndim - 1))
    count = min(x.size // dim, 256) + 16
    dw = (np.abs(g) * dn).sum(rows) + count * u * np.abs(g * n).sum(rows)
    db = count * u * np.abs(g).sum(rows)
    return [(a, bar + r * (np.abs(a) + bar) + SMALLEST[dtype]) for a, bar in zip(want, (y, dx, dw, db))]


def check(dtype, shape, weight=True, bias=True, eps=1e-5, seed=0, scale=1.0, offset=0.0):
    rng = np.random.default_rng([seed, *shape])
    dim = shape[-1]
    x = (rng.standard_normal(shape) * scale + offset).astype(dtype)
    g = rng.standard_normal(shape).astype(dtype)
    w = (1 + 0.3 * rng.standard_normal(dim)).astype(dtype) if weight else None
    b = rng.standard_normal(dim).astype(dtype) if bias else None
    tensors = [None if a is None else mg.device_tensor(a) for a in (x, w, b)]
    y = layer_norm(*tensors, eps=eps)
    y.backward(mg.device_tensor(g, constant=True))
    have = [y.data] + [None if t is None else t.grad for t in tensors]
    assert y.dtype == dtype
    for name, value, (want, bar) in zip(("y", "dx", "dw", "db"), have, bars(dtype, x, w, b, g, eps)):
        if value is not None:
            assert value.shape == want.shape and value.dtype == dtype
            assert outside(value, want, bar) == 0, (name, np.nanmax(np.abs(value - want) - bar), np.isnan(value).sum())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [1, 2, 7, 64, 65, 128, 511, 512, 513, 768, 1000, 1024, 1531, 2048, 4096, 4100, 8192, 9001, 16384, 16390, 40000, 70001])
def test_lengths_of_rows(dtype, dim):
    check(dtype, (5, dim))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [2, 7, 9, 64, 130, 511, 513, 1000, 1531, 2049, 4100, 8193, 9001, 16390, 20003, 40000, 70001])
def test_every_value_is_taken_once(dtype, dim):
    """Rows of zeros but for one value at an edge of what threads hold, and gradients likewise, at the same place and at another: what is left out or taken
    twice is all there is."""
    piece = 16 // np.dtype(dtype).itemsize
    every = piece * (8 if dim <= 4096 else 64 if dim <= 16384 else 512)
    at = np.arange(0, dim, every)
    at = np.concatenate((at, at - 1, [dim // piece * piece, dim // piece * piece - 1, dim - 1]))
    at = np.unique(at[(at >= 0) & (at < dim)])
    rows = np.arange(len(at))
    x = np.zeros((len(at), dim), dtype)
    x[rows, at] = 1
    for other in (at, np.roll(at, 1)):
        g = np.zeros((len(at), dim), dtype)
        g[rows, other] = 1
        tx, tb = mg.device_tensor(x), mg.device_tensor(np.zeros(dim, dtype))
        y = layer_norm(tx, None, tb, eps=1e-8)
        y.backward(mg.device_tensor(g, constant=True))
        wanted = bars(dtype, x, None, None, g, 1e-8)
        for have, (want, bar) in zip((y.data, tx.grad, tb.grad), (wanted[0], wanted[1], wanted[3])):
            assert outside(have, want, bar) == 0
        assert np.abs(wanted[0][0][rows, at]).min() > 100 * np.abs(wanted[0][1][rows, at]).max()  # the bar is small next to the value


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(64,), (1, 64), (2, 3, 4, 100), (4099, 24), (700, 515), (3000, 1024), (70000, 8), (2100, 4096)])
def test_numbers_of_rows(dtype, shape):
    check(dtype, shape)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("weight", [False, True])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dim", [96, 333, 20000])
def test_without_weight_or_bias(dtype, weight, bias, dim):
    check(dtype, (9, dim), weight, bias)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [96, 1001, 20000])
def test_small_values_and_rows_far_from_zero(dtype, dim):
    check(dtype, (6, dim), scale=1e-3, eps=1e-6)
    check(dtype, (6, dim), scale=50.0, eps=0.0)
    check(dtype, (6, dim), offset=500.0)
    check(dtype, (6, dim), offset=-3e4, scale=30.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_one_value_throughout(dtype):
    for dim in (3, 1024, 1000, 20000):
        x = mg.device_tensor(np.full((4, dim), 3.0, dtype))
        y = layer_norm(x, eps=1e-5)
        y.backward(mg.device_tensor(np.ones((4, dim), dtype)))
        assert not y.data.any() and np.abs(x.grad).max() <= 400 * (dim / 16 + 16) * UNIT[dtype][0]


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("weight", [False, True])
@pytest.mark.parametrize("dim", [1, 5, 20, 300, 1030, 2053, 4100, 9001, 16390, 40000, 40001])
def test_gradients_of_rows_of_one_value_far_from_zero(dtype, weight, dim):
    """What lies behind a row's end has no part in its sums, where the mean over the square root of eps (2^50) is beyond the type, too.  Norms are
    exactly 0; a mean of v = w grad is off by (D / 16 + 16) u of the mean of |v|, and what comes of it by 4 u of its parts."""
    u, r, chain, rng = *UNIT[dtype], dim / 16 + 16, np.random.default_rng(dim)
    value, g = dtype(2.0**80 if dtype == np.float32 else 2.0**1000), rng.standard_normal((4, dim)).astype(dtype)
    w = (1 + 0.3 * rng.standard_normal(dim)).astype(dtype) if weight else np.ones(dim, dtype)
    x, tw, tb = mg.device_tensor(np.full((4, dim), value)), mg.device_tensor(w) if weight else None, mg.device_tensor(np.zeros(dim, dtype))
    y = layer_norm(x, tw, tb, eps=2.0**-100)
    y.backward(mg.device_tensor(g, constant=True))
    v = g.astype(ora.WIDE) * w
    size = np.abs(v).mean(-1, keepdims=True)
    want = 2.0**50 * (v - v.mean(-1, keepdims=True))
    assert not y.data.any() and (tw is None or not tw.grad.any())
    assert outside(x.grad, want, 2.0**50 * ((chain + 4) * u * size + 4 * u * (np.abs(v) + size)) + r * np.abs(want)) == 0
    assert outside(tb.grad, g.astype(ora.WIDE).sum(0), 20 * u * np.abs(g).sum(0)) == 0


@pytest.mark.parametrize("dim", [64, 1000, 20000])
def test_rows_that_are_no_numbers_stay_alone(dim):
    rng = np.random.default_rng(dim)
    x, g = rng.standard_normal((2, 9, dim)).astype(np.float32)
    spoilt = x.copy()
    spoilt[2, dim // 3], spoilt[5, 0] = np.nan, np.inf
    results = []
    for values in (x, spoilt):
        t = mg.device_tensor(values)
        y = layer_norm(t, eps=1e-6)
        y.backward(mg.device_tensor(g, constant=True))
        results.append((y.data, t.grad))
    rest = [0, 1, 3, 4, 6, 7, 8]
    for clean, other in zip(*results):
        assert np.array_equal(clean[rest], other[rest]) and np.isnan(other[[2, 5]]).all()


@pytest.mark.parametrize("shape", [(4, 500, 768), (3, 20000), (1200, 1001)])
def test_the_same_bits_every_time_and_only_what_is_wanted(shape):
    rng = np.random.default_rng(0)
    given = [rng.standard_normal(shape).astype(np.float32), *(rng.standard_normal((2, shape[-1])).astype(np.float32))]
    g = rng.standard_normal(shape).astype(np.float32)
    runs = []
    for _ in range(3):
        tensors = [mg.tensor(a) for a in given]
        layer_norm(*tensors, eps=1e-6).backward(g)
        runs.append([t.grad.copy() for t in tensors])
    assert all(np.array_equal(a, b) for run in runs[1:] for a, b in zip(run, runs[0]))
    for wanted in range(1, 8):
        tensors = [mg.tensor(a, constant=not wanted >> n & 1) for n, a in enumerate(given)]
        layer_norm(*tensors, eps=1e-6).backward(g)
        for n, t in enumerate(tensors):
            assert t.grad is None if t.constant else np.array_equal(t.grad, runs[0][n])


@pytest.mark.parametrize("dim", [5, 130])
def test_differences(dim):
    rng = np.random.default_rng(4)
    given, g = [rng.standard_normal((3, dim)), rng.standard_normal(dim), rng.standard_normal(dim)], rng.standard_normal((3, dim))
    tensors = [mg.tensor(a) for a in given]
    layer_norm(*tensors, eps=1e-3).backward(g)
    f = lambda *ops: float((layer_norm(*ops, eps=1e-3).data * g).sum())
    for n, t in enumerate(tensors):
        for index in rng.permutation(t.size)[:8]:
            up, down = [a.copy() for a in given], [a.copy() for a in given]
            up[n].flat[index] += 1e-6
            down[n].flat[index] -= 1e-6
            assert abs((f(*up) - f(*down)) / 2e-6 - t.grad.flat[index]) < 1e-7


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [63, 64, 1024, 1537, 5000])
def test_memory_that_begins_anywhere(dtype, dim):
    """Through the C entry points, tensors that begin at any multiple of their values' size; nothing outside the results is written."""
    from mygrad_amd import _device, _hip

    rng, item, rows = np.random.default_rng(dim), np.dtype(dtype).itemsize, 7
    code, lib = _hip.storage_code(dtype), _hip.lib()
    x, g = rng.standard_normal((2, rows, dim)).astype(dtype)
    w, b = (1 + 0.3 * rng.standard_normal((2, dim))).astype(dtype)
    wants = bars(dtype, x, w, b, g, 1e-5)
    for shift in (1, 3, 8):
        def put(a):
            held = np.full(a.size + 16, 7, dtype)
            held[shift:shift + a.size] = a.ravel()
            return _device.from_host(held).buf
        given, out = [put(a) for a in (x, w, b, g)], [put(np.full(n, 5, dtype)) for n in (x.size, x.size, dim, dim)]
        px, pw, pb, pg, py, pdx, pdw, pdb = (buf.ptr + shift * item for buf in given + out)
        kept = _device.DeviceBuffer(3 * rows * 8)
        _hip.check(lib.mg_layer_norm_fwd(code, rows, dim, 1e-5, px, pw, pb, py, kept.ptr))
        _hip.check(lib.mg_layer_norm_bwd(code, rows, dim, px, pw, kept.ptr, pg, pdx, pdw, pdb))
        for buf, (want, bar) in zip(out, wants):
            held = np.empty(want.size + 16, dtype)
            buf.download_into(held)
            assert outside(held[shift:shift + want.size].reshape(want.shape), want, bar) == 0
            assert (held[:shift] == 7).all() and (held[shift + want.size:] == 7).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [1, 33, 5000])
def test_sums_over_no_rows_wherever_they_begin(dtype, dim):
    from mygrad_amd import _device, _hip

    item = np.dtype(dtype).itemsize
    for shift in (0, 1, 3):
        bufs = [_device.from_host(np.full(dim + 16, 7, dtype)).buf for _ in range(2)]
        for given in ((0, 1), (0,), (1,)):
            pdw, pdb = (bufs[n].ptr + shift * item if n in given else None for n in range(2))
            _hip.check(_hip.lib().mg_layer_norm_bwd(_hip.storage_code(dtype), 0, dim, None, None, None, None, None, pdw, pdb))
        for buf in bufs:
            held = np.empty(dim + 16, dtype)
            buf.download_into(held)
            assert not held[shift:shift + dim].any() and (held[:shift] == 7).all() and (held[shift + dim:] == 7).all()


def test_entry_points_refuse_bad_arguments():
    from mygrad_amd import _device, _hip

    lib, buf = _hip.lib(), _device.DeviceBuffer(1 << 16)
    p = buf.ptr
    for status, (dtype, rows, dim, eps) in ((-2, (7, 2, 8, 1e-5)), (-1, (0, -1, 8, 1e-5)), (-1, (0, 2, 0, 1e-5)), (-1, (0, 2, 8, -1.0)),
                                            (-1, (0, 2, 8, float("nan"))), (-2, (0, 1 << 31, 8, 1e-5)), (-2, (0, 2, (1 << 30) + 1, 1e-5))):
        assert lib.mg_layer_norm_fwd(dtype, rows, dim, eps, p, p, p, p, p) == status
        if eps == 1e-5:
            assert lib.mg_layer_norm_bwd(dtype, rows, dim, p, p, p, p, p, p, p) == status
    assert lib.mg_layer_norm_fwd(0, 2, 8, 1e-5, None, p, p, p, p) == -1 and lib.mg_layer_norm_fwd(0, 2, 8, 1e-5, p, p, p, None, p) == -1
    assert lib.mg_layer_norm_bwd(0, 2, 8, p, p, p, None, p, p, p) == -1 and lib.mg_layer_norm_bwd(0, 2, 8, p, p, p, p, None, None, None) == -1
    assert lib.mg_layer_norm_bwd(0, 2, 8, p, p, None, p, p, p, p) == -1
    assert lib.mg_layer_norm_fwd(0, 0, 8, 1e-5, None, None, None, None, None) == 0
    assert lib.mg_layer_norm_bwd(0, 0, 8, None, None, None, None, None, p, p) == 0  # sums over no rows
    held = np.ones(8, np.float32)
    buf.download_into(held)
    assert not held.any()


def test_more_rows_than_a_grid_has_blocks():
    rows = (1 << 24) + 1000
    x = np.random.default_rng(0).integers(-8, 8, (rows, 2)).astype(np.float16)
    x[:, 1] += x[:, 0] == x[:, 1]
    t, b = mg.device_tensor(x), mg.device_tensor(np.zeros(2, np.float16))
    y = layer_norm(t, None, b, eps=0.0)
    y.backward(mg.device_tensor(np.full((rows, 2), 2.0**-14, np.float16), constant=True))
    want = np.where(x == x.max(-1, keepdims=True), 1.0, -1.0)
    assert np.array_equal(y.data, want) and not t.grad.any() and np.abs(b.grad / (rows * 2.0**-14) - 1).max() < 2.0**-10


def test_empty_tensors():
    for shape in ((0, 8), (3, 0), (2, 0, 4)):
        x, w = mg.tensor(np.ones(shape, np.float32)), mg.tensor(np.ones(shape[-1], np.float32))
        y = layer_norm(x, w, eps=1e-5)
        y.backward()
        assert y.shape == shape and x.grad.shape == shape and not w.grad.any()
