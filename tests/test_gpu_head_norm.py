"""The norm of heads with rotary positions against its formulas in 64 bits.

Bars: u is the unit of the sums (2^-24, 2^-53 for float64), r that of the type results are rounded to.  1/sqrt(mean) is off by
(D / 2 + 4) u of itself, a turned value by 8 u of the pair's length and by the table's own u, and a result is rounded by r; the mean
in dx by (D + 8) u of the sum of its terms' magnitudes.  dw adds products of single precision in double."""

import numpy as np
import pytest

import mygrad_amd as mg
from mygrad_amd.nnet import RotaryTable, head_norm, rotate
from oracle import attention as ora

pytestmark = pytest.mark.gpu

UNIT = {np.float16: (2.0**-24, 2.0**-11), np.float32: (2.0**-24, 2.0**-24), np.float64: (2.0**-53, 2.0**-53)}
SMALLEST = {np.float16: 2.0**-24, np.float32: 2.0**-126, np.float64: 2.0**-1022}
DTYPES = [np.float16, np.float32, np.float64]


@pytest.fixture(scope="module", autouse=True)
def device():
    if not mg.is_available():
        pytest.fail("libmygrad_hip.so / gfx950 device not available: the GPU tests need both")


def _check(dtype, lead, heads, dim, sections=None, weight=None, eps=1e-5, interleaved=False, seed=0, scale=1.0, positions=None):
    rng = np.random.default_rng([seed, heads, dim, *lead])
    x = (rng.standard_normal((*lead, heads, dim)) * scale).astype(dtype)
    g = rng.standard_normal(x.shape).astype(dtype)
    w = None if weight is None else (1 + 0.3 * rng.standard_normal((heads, dim) if weight == "each" else dim)).astype(dtype)
    rotary, angle = None, None
    if sections is not None:
        if positions is None:
            positions = rng.integers(0, 5000, (*lead, len(sections)))
        rotary = RotaryTable(sections, 5000, interleaved=interleaved).at(positions)
        angle = ora.angles(sections, np.broadcast_to(positions, (*lead, len(sections))))
    tx, tw = mg.device_tensor(x), None if w is None else mg.device_tensor(w)
    y = rotate(tx, rotary) if eps is None else head_norm(tx, tw, eps=eps, rotary=rotary)
    y.backward(mg.device_tensor(g, constant=True))
    want = ora.head_norm(x, w, eps, angle, interleaved)
    dx, dw = ora.head_norm_backward(x, w, eps, g, angle, interleaved)
    u, r = UNIT[dtype]
    x64, g64 = x.astype(np.float64), g.astype(np.float64)
    inv = 1.0 if eps is None else 1 / np.sqrt((x64 * x64).mean(-1, keepdims=True) + eps)
    most = lambda a: np.abs(a).max(-1, keepdims=True)
    w64 = np.ones(dim) if w is None else w.astype(np.float64)
    size = 2 * most(x64 * w64) * inv  # a pair is at most sqrt(2) of its larger value long
    bar = (dim / 2 + 16) * u * size + 2 * r * np.abs(want) + SMALLEST[dtype]
    assert y.dtype == dtype and (np.abs(y.data - want) <= bar).all(), (np.abs(y.data - want) - bar).max()
    u64 = 2 * most(g64) * most(w64)
    mean = inv * inv * (u64 * np.abs(x64)).mean(-1, keepdims=True) * most(x64)
    bar = inv * ((dim / 2 + 16) * u * (u64 + mean) + (2 * dim + 16) * u * mean) + 2 * r * np.abs(dx) + SMALLEST[dtype]
    assert (np.abs(tx.grad - dx) <= bar).all(), (np.abs(tx.grad - dx) - bar).max()
    if w is not None:
        over = tuple(range(x.ndim - w.ndim))
        bar = ((dim / 2 + 24) * u * (2 * most(g64) * np.abs(x64) * inv)).sum(over) + 2 * r * np.abs(dw) + SMALLEST[dtype]
        assert tw.grad.shape == w.shape and (np.abs(tw.grad - dw) <= bar).all(), (np.abs(tw.grad - dw) - bar).max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [1, 2, 7, 32, 64, 72, 80, 96, 128, 130, 256, 513, 1024])
def test_head_dimensions(dtype, dim):
    _check(dtype, (2, 9), 3, dim, sections=(dim // 2,) if dim > 1 else None, weight="shared")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("sections", [(32,), (8, 24), (8, 12, 12), (3, 0, 5), (1, 2, 3, 4)])
@pytest.mark.parametrize("weight", [None, "shared", "each"])
def test_axes_and_weights(dtype, interleaved, sections, weight):
    _check(dtype, (2, 5), 6, 64, sections=sections, weight=weight, interleaved=interleaved)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lead,heads", [((1,), 1), ((1, 1), 8), ((3, 333), 5), ((2, 3, 4), 7), ((), 2), ((700,), 33)])
def test_tokens_and_heads(dtype, lead, heads):
    _check(dtype, lead, heads, 64, sections=(16, 16), weight="shared")


@pytest.mark.parametrize("dtype", DTYPES)
def test_rotation_alone_and_norm_alone(dtype):
    _check(dtype, (2, 30), 4, 80, sections=(40,), eps=None)
    _check(dtype, (2, 30), 4, 80, sections=(13, 7), eps=None, interleaved=True)
    _check(dtype, (2, 30), 4, 80, weight="shared")
    _check(dtype, (2, 30), 4, 80, sections=(40,), positions=np.arange(30)[:, None], weight="shared")  # the same for every sequence


@pytest.mark.parametrize("dtype", DTYPES)
def test_zeros_and_small_values(dtype):
    x = mg.device_tensor(np.zeros((3, 2, 16), dtype=dtype))
    y = head_norm(x, eps=1e-6)
    y.backward(mg.device_tensor(np.ones((3, 2, 16), dtype=dtype)))
    assert not y.data.any() and np.allclose(x.grad, 1e3, rtol=2 * UNIT[dtype][1] + 4 * UNIT[dtype][0])
    _check(dtype, (4,), 2, 64, sections=(32,), weight="shared", scale=1e-3, eps=1e-6)
    _check(dtype, (4,), 2, 64, sections=(32,), weight="shared", scale=200.0, eps=0.0)


def test_the_same_bits_every_time_and_only_what_is_wanted():
    rng = np.random.default_rng(0)
    xv, wv, gv = rng.standard_normal((4, 500, 8, 64)).astype(np.float32), np.ones(64, dtype=np.float32), rng.standard_normal((4, 500, 8, 64)).astype(np.float32)
    runs = []
    for _ in range(3):
        x, w = mg.tensor(xv), mg.tensor(wv)
        head_norm(x, w, eps=1e-6).backward(gv)
        runs.append((x.grad.copy(), w.grad.copy()))
    assert all(np.array_equal(a, b) for run in runs[1:] for a, b in zip(run, runs[0]))
    x, w = mg.tensor(xv, constant=True), mg.tensor(wv)
    head_norm(x, w, eps=1e-6).backward(gv)
    assert x.grad is None and np.array_equal(w.grad, runs[0][1])
    x, w = mg.tensor(xv), mg.tensor(wv, constant=True)
    head_norm(x, w, eps=1e-6).backward(gv)
    assert w.grad is None and np.array_equal(x.grad, runs[0][0])


def test_differences():
    rng = np.random.default_rng(4)
    xv, wv, gv = rng.standard_normal((2, 3, 2, 10)), rng.standard_normal((2, 10)), rng.standard_normal((2, 3, 2, 10))
    rotary = RotaryTable((1, 3), 40).at(rng.integers(0, 40, (2, 3, 2)))
    x, w = mg.tensor(xv), mg.tensor(wv)
    head_norm(x, w, eps=1e-3, rotary=rotary).backward(gv)
    f = lambda *ops: float((head_norm(*ops, eps=1e-3, rotary=rotary).data * gv).sum())
    for n, t in enumerate((x, w)):
        for index in rng.permutation(t.size)[:8]:
            up, down = [xv.copy(), wv.copy()], [xv.copy(), wv.copy()]
            up[n].flat[index] += 1e-6
            down[n].flat[index] -= 1e-6
            assert abs((f(*up) - f(*down)) / 2e-6 - t.grad.flat[index]) < 1e-7


def test_entry_points_refuse_bad_descriptors():
    from mygrad_amd import _device, _hip

    lib, buf = _hip.lib(), _device.DeviceBuffer(1 << 16)
    good = dict(dtype=0, norm=1, weight_heads=1, axes=1, tokens=2, heads=2, D=16, pairs=4, table_rows=3, eps=1e-6, positions=buf.ptr, axis_of=buf.ptr)
    for status, change in ((-2, dict(dtype=7)), (-1, dict(pairs=9)), (-1, dict(eps=-1.0)), (-1, dict(weight_heads=3)), (-1, dict(positions=None)),
                           (-1, dict(axes=0)), (-1, dict(table_rows=0)), (-2, dict(D=1025)), (-1, dict(tokens=-1))):
        desc = _hip.HeadNormDesc(**{**good, **change})
        assert lib.mg_head_norm_fwd(desc, *[buf.ptr] * 4) == status, change
        assert lib.mg_head_norm_bwd(desc, *[buf.ptr] * 6) == status, change
    assert lib.mg_head_norm_fwd(_hip.HeadNormDesc(**good), buf.ptr, None, buf.ptr, buf.ptr) == -1
    assert lib.mg_head_norm_bwd(_hip.HeadNormDesc(**{**good, "weight_heads": 0}), *[buf.ptr] * 6) == -1


KERNELS = [(64, (16,)), (64, (5, 6)), (72, (16, 9)), (130, (40,)), (7, (2,)), (1000, (300,))]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,sections", KERNELS)
def test_infinities_behind_the_pairs_stay_as_they_are(dtype, interleaved, dim, sections):
    """In each kernel: what a head's pairs leave over is handed on bit for bit, and so is its gradient."""
    rng = np.random.default_rng(dim)
    pairs = sum(sections)
    x, g = (rng.standard_normal((2, 9, 3, dim)).astype(dtype) for _ in range(2))
    spoilt = [a.copy() for a in (x, g)]
    for a in spoilt:
        a[..., 2 * pairs:] = rng.choice(np.array([np.inf, -np.inf, 1.5, -0.25], dtype), a[..., 2 * pairs:].shape)
    rotary = RotaryTable(sections, 50, interleaved=interleaved).at(rng.integers(0, 50, (2, 9, len(sections))))
    t = mg.device_tensor(x)
    y = rotate(t, rotary)
    y.backward(mg.device_tensor(spoilt[1], constant=True))
    for have, given in ((rotate(spoilt[0], rotary).data, spoilt[0]), (t.grad, spoilt[1])):
        assert np.array_equal(have[..., 2 * pairs:], given[..., 2 * pairs:])
        assert np.isfinite(have[..., :2 * pairs]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,sections", KERNELS)
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_the_gradient_of_a_rotation_has_no_part_of_its_input(dtype, dim, sections, bad):
    rng = np.random.default_rng(dim)
    rotary = RotaryTable(sections, 50).at(rng.integers(0, 50, (2, 9, len(sections))))
    g = rng.standard_normal((2, 9, 3, dim)).astype(dtype)
    grads = []
    for x in (np.ones_like(g), np.full_like(g, bad)):
        t = mg.device_tensor(x)
        rotate(t, rotary).backward(mg.device_tensor(g, constant=True))
        grads.append(t.grad)
    assert np.array_equal(*grads)
