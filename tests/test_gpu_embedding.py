"""Rows of a table by token, and the gradient of the table, against their formulas in 64 bits.

Bars: forward one rounding (float16: of a product in single precision with a rounded scale); a row of the gradient whose token occurs c times adds
c values in single precision (double for float64), c u of their magnitudes at most in any order, and is rounded once."""

import numpy as np
import pytest

import mygrad_amd as mg
from mygrad_amd.nnet import TokenIds, embedding
from oracle import language as ora

pytestmark = pytest.mark.gpu

UNIT = {np.float16: (2.0**-24, 2.0**-11), np.float32: (2.0**-24, 2.0**-24), np.float64: (2.0**-53, 2.0**-53)}
SMALLEST = {np.float16: 2.0**-24, np.float32: 2.0**-126, np.float64: 2.0**-1022}
DTYPES = [np.float16, np.float32, np.float64]


@pytest.fixture(scope="module", autouse=True)
def device():
    if not mg.is_available():
        pytest.fail("libmygrad_hip.so / gfx950 device not available: the GPU tests need both")


def check(dtype, ids, vocabulary, dim, scale=1.0, seed=0):
    rng = np.random.default_rng([seed, vocabulary, dim])
    ids = np.asarray(ids)
    weight, g = rng.standard_normal((vocabulary, dim)).astype(dtype), rng.standard_normal((*ids.shape, dim)).astype(dtype)
    t = mg.device_tensor(weight)
    y = embedding(t, ids, scale=scale)
    y.backward(mg.device_tensor(g, constant=True))
    u, r = UNIT[dtype]
    flat, g64 = ids.ravel(), g.reshape(ids.size, dim).astype(ora.WIDE)
    want = ora.embedding(weight, ids, scale)
    assert y.dtype == dtype and y.shape == want.shape
    assert int((~(np.abs(y.data - want) <= (r + 2 * u) * np.abs(want) + SMALLEST[dtype])).sum()) == 0
    if scale == 1.0:
        assert np.array_equal(y.data, want.astype(dtype))
    order = np.argsort(flat, kind="stable")
    order = order[flat[order] >= 0]
    want, size, count = np.zeros((vocabulary, dim), ora.WIDE), np.zeros((vocabulary, dim), ora.WIDE), np.bincount(flat[order], minlength=vocabulary)[:, None]
    if order.size:
        starts = np.flatnonzero(np.diff(flat[order], prepend=-1))
        held = flat[order][starts]
        want[held], size[held] = np.add.reduceat(g64[order], starts, 0), np.add.reduceat(np.abs(g64[order]), starts, 0)
    want, size = want * scale, size * abs(scale)
    bar = (count + 2) * u * size + r * np.abs(want) + (count > 0) * SMALLEST[dtype]
    assert t.grad.shape == weight.shape and t.grad.dtype == dtype
    assert int((~(np.abs(t.grad - want) <= bar)).sum()) == 0, np.nanmax(np.abs(t.grad - want) - bar)


def words(rng, count, vocabulary):
    """A few tokens often, most seldom."""
    return (np.exp(rng.random(count) * np.log(vocabulary + 1)).astype(np.int64) - 1).clip(0, vocabulary - 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [1, 2, 7, 64, 72, 100, 256, 511, 768, 1024, 2050, 4096, 9001])
def test_lengths_of_rows(dtype, dim):
    rng = np.random.default_rng(dim)
    check(dtype, words(rng, 97, 61), 61, dim)
    check(dtype, words(rng, 97, 61), 61, dim, scale=dim**0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count,vocabulary", [(1, 1), (1, 5), (2, 1), (31, 1), (1000, 1), (33, 2), (64, 3000), (255, 256), (257, 257), (4095, 300), (4096, 2047), (4097, 2048),
                                              (5000, 70001), (8193, 20), (20000, 5000), (70000, 333)])
def test_numbers_of_tokens(dtype, count, vocabulary):
    rng = np.random.default_rng(count)
    check(dtype, rng.integers(0, vocabulary, count), vocabulary, 24)
    check(dtype, words(rng, count, vocabulary), vocabulary, 10)


@pytest.mark.parametrize("dtype", DTYPES)
def test_vocabularies_of_more_bits(dtype):
    rng = np.random.default_rng(1)
    for count, vocabulary in ((300, 1 << 22), (9000, (1 << 22) + 77)):
        ids = rng.integers(0, vocabulary, count)
        ids[:4] = 0, vocabulary - 1, vocabulary - 1, 2047
        check(dtype, ids, vocabulary, 3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count", [1, 2, 50, 5000])
def test_no_tokens_among_tokens(dtype, count):
    rng = np.random.default_rng(count)
    check(dtype, np.where(rng.random(count) < 0.5, -1, rng.integers(0, 40, count)), 40, 33)
    check(dtype, np.full(count, -1), 40, 33)
    check(dtype, np.where(np.arange(count) == count // 2, 39, -1), 40, 64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(), (1,), (2, 3, 4), (5, 1)])
def test_shapes_of_tokens(dtype, shape):
    check(dtype, np.random.default_rng(0).integers(-1, 9, shape), 9, 16)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, -2.5, 0.1, 2.0**-30, 1e4])
def test_scales(dtype, scale):
    if dtype == np.float16 and scale == 1e4:
        scale = 1000.0  # of what single precision carries there, float16 holds no more
    check(dtype, np.random.default_rng(0).integers(-1, 9, 20), 9, 48, scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_are_no_numbers_stay_alone(dtype):
    weight = np.arange(40, dtype=dtype).reshape(5, 8)
    weight[3] = np.nan
    t = mg.device_tensor(weight)
    y = embedding(t, [0, 3, -1, 4], scale=2.0)
    assert np.isnan(y.data[1]).all() and np.array_equal(y.data[[0, 2, 3]], np.stack((weight[0] * 2, np.zeros(8), weight[4] * 2)))
    g = np.ones((4, 8), dtype)
    g[2] = np.nan  # of what is no token
    g[3] = np.inf
    y.backward(g)
    assert np.isinf(t.grad[4]).all() and np.array_equal(t.grad[:4], np.array([2, 0, 0, 2], dtype)[:, None] * np.ones(8, dtype))


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("count,dim", [(30011, 1001), (150001, 200), (1500, 20003), (4_000_001, 7)])
def test_more_rows_than_caches_hold(dtype, count, dim):
    rng = np.random.default_rng(dim)
    weight, ids = rng.standard_normal((301, dim)).astype(dtype), rng.integers(-1, 301, count)
    y = embedding(mg.device_tensor(weight, constant=True), ids).data
    assert y.nbytes > 5e7 and np.array_equal(y[ids < 0], np.zeros_like(y[ids < 0]))
    assert np.array_equal(y[ids >= 0], weight[ids[ids >= 0]])


@pytest.mark.parametrize("count,vocabulary", [(3000, 50), (20000, 700)])
def test_the_same_bits_every_time(count, vocabulary):
    rng = np.random.default_rng(0)
    ids, weight, g = words(rng, count, vocabulary), rng.standard_normal((vocabulary, 96)).astype(np.float32), rng.standard_normal((count, 96)).astype(np.float32)
    runs = []
    for _ in range(3):
        t = mg.tensor(weight)
        embedding(t, ids).backward(g)
        runs.append(t.grad.copy())
    assert all(np.array_equal(run, runs[0]) for run in runs)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count,vocabulary,dim", [(70_000, 50_001, 5), (5_000, 600_000, 3), (300_001, 5_003, 7), (300_001, 300, 7), (600_001, 40, 3), (2_200_000, 1_000, 2),
                                                  (40_000, 5_003, 2050), (66_000, 3_000, 1030)])
def test_gradients_of_many_tokens(dtype, count, vocabulary, dim):
    """Orders by two digits, chunks of 32 to 256 tokens, and runs that end in a chunk's first tokens, go on through several of its turns, or through several
    chunks.  Sums of whole numbers are exact, and a result is rounded once."""
    rng = np.random.default_rng([count, vocabulary])
    lengths = rng.choice([1, 1, 2, 3, 15, 16, 17, 31, 32, 33, 47, 48, 49, 64, 65, 300], vocabulary)
    lengths = lengths * max(1, count // int(lengths.sum())) + rng.integers(0, 18, vocabulary)
    ids = np.full(count, -1)
    there = np.repeat(rng.permutation(vocabulary), lengths)[:count]
    ids[:there.size] = there
    ids[rng.random(count) < 0.02] = -1
    ids = rng.permutation(ids)
    g = rng.integers(-2, 3, (count, dim)).astype(np.int8)
    t = mg.device_tensor(np.zeros((vocabulary, dim), dtype))
    embedding(t, ids).backward(mg.device_tensor(g.astype(dtype), constant=True))
    order = np.argsort(ids, kind="stable")
    order = order[ids[order] >= 0]
    starts = np.flatnonzero(np.diff(ids[order], prepend=-1))
    want = np.zeros((vocabulary, dim), np.int32)
    want[ids[order][starts]] = np.add.reduceat(g[order], starts, 0, dtype=np.int32)
    assert np.abs(want).max() < 2**15 and np.array_equal(t.grad, want.astype(dtype))


def test_a_table_that_is_used_twice():
    rng = np.random.default_rng(0)
    weight, g = rng.standard_normal((7, 4)), rng.standard_normal((2, 5, 4))
    first, second = rng.integers(0, 7, (2, 5))
    t = mg.tensor(weight)
    (embedding(t, first) * embedding(t, second)).backward(g[0])
    want = ora.embedding(weight, first, 1.0, g[0] * weight[second])[1] + ora.embedding(weight, second, 1.0, g[0] * weight[first])[1]
    assert np.abs(t.grad - want).max() < 1e-14


def test_differences():
    rng = np.random.default_rng(4)
    weight, ids, g = rng.standard_normal((6, 5)), [3, 3, 0, -1, 5], rng.standard_normal((5, 5))
    t = mg.tensor(weight)
    embedding(t, ids, scale=1.5).backward(g)
    f = lambda w: float((embedding(w, ids, scale=1.5).data * g).sum())
    for index in range(t.size):
        up, down = weight.copy(), weight.copy()
        up.flat[index] += 1e-6
        down.flat[index] -= 1e-6
        assert abs((f(up) - f(down)) / 2e-6 - t.grad.flat[index]) < 1e-8


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [5, 64, 130, 1024])
def test_memory_that_begins_anywhere(dtype, dim):
    """Through the C entry points, tensors that begin at any multiple of their values' size; nothing outside the results is written."""
    from mygrad_amd import _device, _hip

    rng, item, vocabulary = np.random.default_rng(dim), np.dtype(dtype).itemsize, 11
    code, lib = _hip.storage_code(dtype), _hip.lib()
    ids = np.array([3, -1, 3, 10, 0, 3], np.int32)
    weight, g = rng.integers(-9, 9, (vocabulary, dim)).astype(dtype), rng.integers(-9, 9, (ids.size, dim)).astype(dtype)
    y, dw = ora.embedding(weight, ids, 2.0, g)
    held_ids = _device.from_host(ids).buf
    for shift in (1, 3, 8):
        def put(a):
            held = np.full(a.size + 16, 7, dtype)
            held[shift:shift + a.size] = a.ravel()
            return _device.from_host(held).buf
        given, out = [put(a) for a in (weight, g)], [put(np.full(a.size, 5, dtype)) for a in (y, dw)]
        pw, pg, py, pdw = (buf.ptr + shift * item for buf in given + out)
        _hip.check(lib.mg_embedding_fwd(code, ids.size, vocabulary, dim, 2.0, held_ids.ptr, pw, py))
        _hip.check(lib.mg_embedding_bwd(code, ids.size, vocabulary, dim, 2.0, held_ids.ptr, pg, pdw))
        for buf, want in zip(out, (y, dw)):
            held = np.empty(want.size + 16, dtype)
            buf.download_into(held)
            assert np.array_equal(held[shift:shift + want.size].reshape(want.shape), want)
            assert (held[:shift] == 7).all() and (held[shift + want.size:] == 7).all()


def test_tokens_beyond_the_table_are_none_to_the_entry_points():
    """The operation refuses them; tokens that lie on the device are not looked at by the host."""
    from mygrad_amd import _device, _hip

    ids = _device.from_host(np.array([2, 5, 2**31 - 1, -7], np.int32)).buf
    weight, out = _device.from_host(np.ones((5, 8), np.float32)).buf, _device.from_host(np.full((4, 8), 9, np.float32)).buf
    dw = _device.from_host(np.full((5, 8), 9, np.float32)).buf
    _hip.check(_hip.lib().mg_embedding_fwd(0, 4, 5, 8, 1.0, ids.ptr, weight.ptr, out.ptr))
    _hip.check(_hip.lib().mg_embedding_bwd(0, 4, 5, 8, 1.0, ids.ptr, out.ptr, dw.ptr))
    y, sums = np.empty((4, 8), np.float32), np.empty((5, 8), np.float32)
    out.download_into(y)
    dw.download_into(sums)
    assert np.array_equal(y, np.array([1, 0, 0, 0], np.float32)[:, None] * np.ones(8)) and np.array_equal(sums, np.array([0, 0, 1, 0, 0])[:, None] * np.ones(8))


def test_no_tokens_leave_a_gradient_of_zeros():
    from mygrad_amd import _device, _hip

    for dtype in DTYPES:
        for shift in (0, 1, 3):
            held, item = np.full(16 + 7 * 33, 5, dtype), np.dtype(dtype).itemsize
            buf = _device.from_host(held).buf
            _hip.check(_hip.lib().mg_embedding_bwd(_hip.storage_code(dtype), 0, 7, 33, 1.0, None, None, buf.ptr + shift * item))
            buf.download_into(held)
            assert not held[shift:shift + 7 * 33].any() and (held[:shift] == 5).all() and (held[shift + 7 * 33:] == 5).all()


def test_entry_points_refuse_bad_arguments():
    from mygrad_amd import _device, _hip

    lib, p = _hip.lib(), _device.DeviceBuffer(1 << 16).ptr
    for status, (dtype, tokens, rows, dim, scale) in ((-2, (7, 2, 3, 8, 1.0)), (-1, (0, -1, 3, 8, 1.0)), (-1, (0, 2, -3, 8, 1.0)), (-1, (0, 2, 3, -8, 1.0)),
                                                      (-1, (0, 2, 3, 8, float("inf"))), (-1, (0, 2, 3, 8, float("nan"))), (-2, (0, 1 << 31, 3, 8, 1.0)), (-2, (0, 1 << 26, 3, 8, 1.0)),
                                                      (-2, (0, 2, 1 << 31, 8, 1.0)), (-2, (0, 2, 3, 1 << 31, 1.0))):
        assert lib.mg_embedding_fwd(dtype, tokens, rows, dim, scale, p, p, p) == status
        assert lib.mg_embedding_bwd(dtype, tokens, rows, dim, scale, p, p, p) == status
    for arguments in ((None, p, p), (p, None, p), (p, p, None)):
        assert lib.mg_embedding_fwd(0, 2, 3, 8, 1.0, *arguments) == -1 and lib.mg_embedding_bwd(0, 2, 3, 8, 1.0, *arguments) == -1
    assert lib.mg_embedding_fwd(0, 0, 3, 8, 1.0, None, None, None) == 0 and lib.mg_embedding_bwd(0, 0, 0, 8, 1.0, None, None, None) == 0


def test_empty_tables_and_no_tokens():
    weight = mg.tensor(np.ones((4, 3)))
    y = embedding(weight, np.zeros((2, 0), np.int64))
    y.backward()
    assert y.shape == (2, 0, 3) and np.array_equal(weight.grad, np.zeros((4, 3)))
    assert embedding(np.ones((4, 0)), [1, 2]).shape == (2, 0)
    assert np.array_equal(embedding(np.ones((0, 3)), [-1, -1]).data, np.zeros((2, 3)))


def test_tokens_that_a_kernel_found():
    """What log_probabilities names goes on to embedding without a copy to the host."""
    from mygrad_amd.nnet import log_probabilities

    rng = np.random.default_rng(0)
    logits, weight = rng.standard_normal((6, 9)), rng.standard_normal((9, 4))
    _, _, which = log_probabilities(logits, top=1)
    assert isinstance(which, TokenIds) and which._host is None and which.below == 9
    assert np.array_equal(embedding(weight, which.reshape(6)).data, weight[logits.argmax(-1)]) and which._host is None
    assert np.array_equal(which.data[:, 0], logits.argmax(-1))
