"""Log probabilities, entropies, the likeliest tokens and distillation against their formulas in 64 bits.

Bars: u is the unit of the sums (2^-24, 2^-53 for float64), r that of the type results are rounded to.  t = (z - m) / T is off by 4 u of itself,
its exponential by (4 |t| + 8) u, and a sum over V values by less than (V / 32 + 32) u of itself (32 lanes or more add side by side) and by what
its terms are, (4 |a| + 8) u with a the mean of t.  Logarithms are off by 4 u of themselves.  What single precision cannot hold is below 2^-126."""

import numpy as np
import pytest

import mygrad_amd as mg
from mygrad_amd.nnet import TokenIds, distillation, log_probabilities
from oracle import language as ora

pytestmark = pytest.mark.gpu

UNIT = {np.float16: (2.0**-24, 2.0**-11), np.float32: (2.0**-24, 2.0**-24), np.float64: (2.0**-53, 2.0**-53)}
SMALLEST = {np.float16: 2.0**-24, np.float32: 2.0**-126, np.float64: 2.0**-1022}
TINY = {np.float16: 2.0**-126, np.float32: 2.0**-126, np.float64: 2.0**-1022}
DTYPES = [np.float16, np.float32, np.float64]


@pytest.fixture(scope="module", autouse=True)
def device():
    if not mg.is_available():
        pytest.fail("libmygrad_hip.so / gfx950 device not available: the GPU tests need both")


def wide(dtype):
    return np.float64 if dtype == np.float64 else np.float32


class Bars:
    """How far a row's t, shares and sums may be off."""

    def __init__(self, dtype, z, per=1.0):
        self.u, self.r = UNIT[dtype]
        self.t, self.p, self.log_s = ora.softmax_row(z, per)
        self.bounded = np.where(self.p > 0, self.t, 0)
        self.a = (self.p * self.bounded).sum(-1, keepdims=True)
        self.sum = (z.shape[-1] / 32 + 40 + 4 * np.abs(self.a)) * self.u  # of s, relative
        self.share = (4 * np.abs(self.bounded) + 12) * self.u + self.sum  # of p, relative
        self.mean = (self.p * np.abs(self.bounded) * self.share).sum(-1, keepdims=True) + 2 * np.abs(self.a) * self.sum
        self.log = self.sum + 4 * self.u * np.abs(self.log_s)


def close(name, have, want, bar):
    same = (have == want) | (np.isnan(have) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        fits = same | (np.abs(have - want) <= bar)
    assert int((~fits).sum()) == 0, (name, np.argwhere(~fits)[:4], have[~fits][:4], want[~fits][:4])


def check(dtype, z, ids=None, entropy=False, top=0, seed=0, grads=True):
    """``z:(rows, V)``, of numbers and minus infinities."""
    rng, u = np.random.default_rng([seed, *z.shape]), UNIT[dtype][0]
    z = z.astype(dtype)
    planes = (ids is not None) + entropy
    g = rng.standard_normal((2, len(z))).astype(wide(dtype))
    t = mg.device_tensor(z)
    out = log_probabilities(t, ids, entropy=entropy, top=top)
    if top:
        out, likeliest, which = out
    scores, ent, dz = ora.log_probabilities(z, ids, g[0] if ids is not None else None, g[1] if entropy else None)
    b = Bars(dtype, z)
    if planes:
        assert out.dtype == wide(dtype) and out.shape == ((2, len(z)) if planes == 2 else (len(z),))
        have = out.data.reshape(planes, -1)
        if ids is not None:
            taken = np.abs(np.take_along_axis(b.bounded, np.maximum(ids, 0)[:, None], 1)[:, 0])
            close("scores", have[0], scores, b.log[:, 0] + 4 * u * taken + 2 * u * np.abs(scores))
        if entropy:
            close("entropy", have[-1], ent, (b.log + b.mean)[:, 0] + 4 * u * (np.abs(ent) + np.abs(b.a[:, 0])))
    if top:
        at = ora.likeliest(z, top)
        assert likeliest.shape == which.shape == (len(z), top) and likeliest.constant and likeliest.dtype == wide(dtype)
        assert np.array_equal(which.data, at)
        with np.errstate(invalid="ignore"):
            want = np.take_along_axis(b.t, at, 1) - b.log_s
        want[np.isneginf(b.log_s[:, 0])] = -np.inf
        close("likeliest", likeliest.data, want, b.log + 4 * u * np.abs(np.take_along_axis(b.bounded, at, 1)) + 2 * u * np.abs(want))
    if not planes or not grads:
        return
    out.backward(mg.device_tensor(g if planes == 2 else g[0] if ids is not None else g[1], constant=True))
    gs = np.abs(g[0][:, None]) * ((ids is not None) and (ids >= 0)[:, None])
    h = np.abs(g[1][:, None]) * entropy
    far = np.abs(b.bounded - b.a)
    size = b.p * (gs + h * far)
    bar = b.p * b.share * (gs + h * far) + b.p * h * (4 * u * (np.abs(b.bounded) + far) + b.mean) + 8 * u * (size + np.abs(dz))
    bar += 4 * TINY[dtype] * (1 + gs + h * (far + 200)) + b.r * (np.abs(dz) + bar) + SMALLEST[dtype]
    assert t.grad.shape == z.shape and t.grad.dtype == dtype
    close("dz", t.grad, dz, bar)


def made(rows, vocabulary, seed=0, scale=3.0):
    return np.random.default_rng([seed, rows, vocabulary]).standard_normal((rows, vocabulary)) * scale


def some(rows, vocabulary, seed=0):
    return np.random.default_rng([seed, rows, vocabulary, 1]).integers(0, vocabulary, rows)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocabulary", [1, 2, 3, 7, 8, 31, 33, 63, 64, 65, 127, 129, 255, 257, 511, 513, 1000, 1024, 2049, 4096, 8191, 8200, 32003, 50000, 131101])
def test_lengths_of_rows(dtype, vocabulary):
    check(dtype, made(3, vocabulary), some(3, vocabulary))
    check(dtype, made(3, vocabulary, 1), some(3, vocabulary, 1), entropy=True, top=min(7, vocabulary))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocabulary", [(1, 1000), (1, 70001), (40, 33), (257, 1001), (600, 5000), (3000, 640), (70000, 9), (4097, 2500), (4100, 1999),
                                             (1001, 200), (999, 300)])
def test_numbers_of_rows(dtype, rows, vocabulary):
    check(dtype, made(rows, vocabulary), some(rows, vocabulary), entropy=True)
    check(dtype, made(rows, vocabulary, 2), some(rows, vocabulary, 2), top=3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,entropy,top", [(False, True, 0), (False, True, 4), (False, False, 4), (True, False, 4)])
def test_what_is_asked_for(dtype, tokens, entropy, top):
    for rows, vocabulary in ((5, 900), (700, 333), (2, 40000)):
        check(dtype, made(rows, vocabulary), some(rows, vocabulary) if tokens else None, entropy, top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocabulary", [(6, 77), (6, 9000), (6, 70001), (600, 2500)])
def test_tokens_that_are_none_and_logits_that_are_ruled_out(dtype, rows, vocabulary):
    rng = np.random.default_rng(vocabulary)
    z, ids = made(rows, vocabulary), some(rows, vocabulary)
    z[:, rng.random(vocabulary) < 0.3] = -np.inf
    z[1] = -np.inf  # nothing is left
    z[2] = -np.inf
    z[2, vocabulary // 2] = 1.0  # one is
    ids[0] = ids[3] = -1
    z[4, ids[4]] = -np.inf  # the token itself is ruled out
    check(dtype, z, ids)
    check(dtype, z, ids, entropy=True, top=20)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocabulary", [20, 5000, 60000])
def test_logits_far_apart(dtype, vocabulary):
    z = made(4, vocabulary, scale=300.0)
    check(dtype, z, some(4, vocabulary), entropy=True, top=5)
    check(dtype, made(4, vocabulary) + 5e4 * (np.arange(4) - 1.5)[:, None] / 1.5, some(4, vocabulary), entropy=True)
    check(dtype, np.where(np.arange(vocabulary) == 11, 60000.0, -60000.0) * np.ones((3, 1)), np.array([11, 0, -1]), entropy=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocabulary", [(3, 129), (2, 4096), (3, 50001), (520, 3001)])
@pytest.mark.parametrize("top", [1, 2, 20, 128])
def test_the_likeliest_among_equals(dtype, rows, vocabulary, top):
    rng = np.random.default_rng(top)
    kinds = [np.zeros((rows, vocabulary)), rng.integers(0, 3, (rows, vocabulary)) * 1.0, np.sort(made(rows, vocabulary), 1), -np.sort(made(rows, vocabulary), 1),
             np.where(rng.random((rows, vocabulary)) < 0.5, -0.0, 0.0), np.full((rows, vocabulary), -np.inf)]
    few = np.full((rows, vocabulary), -np.inf)  # fewer than are asked for
    few[:, vocabulary // 3] = 2.0
    spread = np.zeros((rows, vocabulary))  # the largest side by side, and 8 apart
    spread[:, 8 * np.arange(min(vocabulary // 8, 150))] = 3.0
    spread[:, vocabulary - 60:] = 3.0
    for z in kinds + [few, spread]:
        check(dtype, z, None, entropy=False, top=top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocabulary", [100, 9000, 60000])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_rows_that_are_no_numbers_stay_alone(dtype, vocabulary, bad):
    z, ids = made(6, vocabulary).astype(dtype), some(6, vocabulary)
    spoilt = z.copy()
    spoilt[2, vocabulary // 3] = bad
    spoilt[4, 0] = bad
    ids[4] = -1
    results = []
    for values in (z, spoilt):
        runs = []
        for entropy in (False, True):
            t = mg.device_tensor(values)
            out, likeliest, which = log_probabilities(t, ids, entropy=entropy, top=3)
            out.backward()
            runs += [out.data.reshape(-1, 6).T, likeliest.data, which.data, t.grad]
        results.append(runs)
    for n, (clean, other) in enumerate(zip(*results)):
        assert np.array_equal(clean[[0, 1, 3, 5]], other[[0, 1, 3, 5]])
        if n % 4 != 2:
            assert np.isnan(other[2]).all()
    assert results[1][0][4] == 0 and not results[1][3][4].any()  # no token: neither a value nor a gradient
    assert results[1][4][4, 0] == 0 and np.isnan(results[1][4][4, 1]) and np.isnan(results[1][7][4]).all()
    assert results[1][2][2, 0] == vocabulary // 3 and results[1][2][4, 0] == 0  # they come before all others


@pytest.mark.parametrize("rows,vocabulary", [(3, 70001), (900, 1500)])
def test_the_same_bits_every_time(rows, vocabulary):
    z, ids = made(rows, vocabulary).astype(np.float32), some(rows, vocabulary)
    runs = []
    for _ in range(3):
        t = mg.device_tensor(z)
        out, likeliest, which = log_probabilities(t, ids, entropy=True, top=9)
        out.backward()
        runs.append((out.data, likeliest.data, which.data, t.grad))
    assert all(np.array_equal(a, b) for run in runs[1:] for a, b in zip(run, runs[0]))


def test_more_rows_than_a_grid_has_blocks():
    rows = (1 << 22) + 1000
    z = np.random.default_rng(0).integers(-8, 9, (rows, 3)).astype(np.float16)
    ids = np.arange(rows) % 3
    t = mg.device_tensor(z)
    out, likeliest, which = log_probabilities(t, ids, top=1)
    p = np.exp(z.astype(np.float64))
    p /= p.sum(-1, keepdims=True)
    assert np.array_equal(which.data[:, 0], z.argmax(-1)) and np.abs(out.data - np.log(p[np.arange(rows), ids])).max() < 1e-5
    assert np.abs(likeliest.data[:, 0] - np.log(p.max(-1))).max() < 1e-5
    out.backward()
    p[np.arange(rows), ids] -= 1
    assert np.abs(t.grad + p).max() < 2.0**-11 + 1e-6
    rows = (1 << 24) + 1000  # four to a block
    t = mg.device_tensor(np.ones((rows, 1), np.float16))
    out = log_probabilities(t, np.zeros(rows, np.int32), entropy=True)
    out.backward()
    assert not out.data.any() and not t.grad.any()
    t = mg.device_tensor(np.ones((rows, 1), np.float16))
    loss = distillation(t, np.zeros((rows, 1), np.int32), np.ones((rows, 1), np.float16))
    loss.backward()
    assert not loss.data.any() and not t.grad.any()


def edges(length, item):
    """Both sides of where a row's pieces, steps and parts may end: every 8th piece of 16 bytes, every 64th of a long row, and what the last piece begins with."""
    piece = 16 // item
    every = piece * (8 if length <= 4096 else 64)
    marks = np.arange(0, length, every)
    marks = np.concatenate((marks, marks - 1, [length // piece * piece, length // piece * piece - 1, length - 1]))
    return np.unique(marks[(marks >= 0) & (marks < length)])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocabulary", [*((3, n) for n in (1, 2, 3, 7, 8, 33, 65, 129, 257, 513, 1000, 1024, 2049, 4096, 4100, 8191, 8200, 16385, 32003, 50000, 131101)),
                                             *((40, n) for n in (255, 511, 2047, 70001)), *((300, n) for n in (2047, 4099, 16001, 50001)),
                                             *((4100, n) for n in (33, 250, 500, 1000, 2047, 2050, 4095, 8191))])
def test_every_logit_is_taken_once(dtype, rows, vocabulary):
    """K equal logits at the edges and all others so far below that their sum is less than half a unit: probabilities of 1 / K, and one that is left out or
    taken twice is 1 / K of the sum.  K itself is exact; its logarithm and its inverse are off by 4 u."""
    u, r = UNIT[dtype]
    at = edges(vocabulary, np.dtype(dtype).itemsize)
    count, z = len(at), np.full((rows, vocabulary), -100.0, dtype)
    z[:, at] = 3.0
    size, ids = float(np.log(count)), at[np.arange(rows) % count].astype(np.int32)
    assert 1 / count > 100 * 8 * u * size  # the bars are small next to a logit's part
    ids[::5] = 0 if at[0] == 0 else -1
    own = ids >= 0
    rng, top = np.random.default_rng(vocabulary), min(count, 128)
    g = rng.standard_normal((2, rows)).astype(wide(dtype))
    t = mg.device_tensor(z)
    out, likeliest, which = log_probabilities(t, ids, entropy=True, top=top)
    assert np.array_equal(which.data, np.tile(at[:top], (rows, 1)))
    close("scores", out.data, np.stack((np.where(own, -size, 0), np.full(rows, size))), 8 * u * size + 1e-30)
    close("likeliest", likeliest.data, np.full((rows, top), -size), 8 * u * size + 1e-30)
    alone = log_probabilities(mg.device_tensor(z, constant=True), ids)  # by other kernels where rows are short
    close("scores alone", alone.data, np.where(own, -size, 0), 8 * u * size + 1e-30)
    out.backward(mg.device_tensor(g, constant=True))
    want = np.zeros((rows, vocabulary))
    want[:, at] = -(g[0] * own)[:, None] / count
    want[np.arange(rows), ids] += g[0] * own
    given = np.abs(g[0])[:, None] + np.abs(g[1])[:, None]
    close("dz", t.grad, want, 8 * u * given * (want != 0) + 1e-30 * given + r * np.abs(want) + SMALLEST[dtype])
    taught = at[np.unique(np.linspace(0, count - 1, 4).astype(int))] if count >= 4 else at[:1]
    few = len(taught)
    for per in (1.0, 2.0):
        t = mg.device_tensor(z)
        loss = distillation(t, np.tile(taught, (rows, 1)), np.full((rows, few), 2.0, dtype), temperature=1 / per)
        loss.backward(mg.device_tensor(g[0], constant=True))
        close("loss", loss.data, np.full(rows, size - np.log(few)), 16 * u * (size + np.log(few)) + 1e-30)
        want[:], want[:, at] = 0, (g[0] * per / count)[:, None]
        want[:, taught] -= (g[0] * per / few)[:, None]
        close("dz of distillation", t.grad, want, 16 * u * per * given * (want != 0) + 1e-30 * given + r * np.abs(want) + 2 * SMALLEST[dtype])


def test_leading_shapes():
    z = made(12, 50)
    flat = log_probabilities(z, np.arange(12), entropy=True, top=2)
    for shape in ((3, 4), (2, 3, 2), (12, 1)):
        out, likeliest, which = log_probabilities(z.reshape(*shape, 50), np.arange(12).reshape(shape), entropy=True, top=2)
        assert out.shape == (2, *shape) and which.shape == likeliest.shape == (*shape, 2)
        assert np.array_equal(out.data.ravel(), flat[0].data.ravel()) and np.array_equal(which.data.ravel(), flat[2].data.ravel())
    out = log_probabilities(z[0], 3)
    assert out.shape == () and out.data == log_probabilities(z[:1], [3]).data[0]


def test_empty_rows_and_constants():
    t = mg.tensor(np.ones((0, 5)))
    out, likeliest, which = log_probabilities(t, np.zeros(0, np.int64), entropy=True, top=2)
    out.backward()
    assert out.shape == (2, 0) and likeliest.shape == which.shape == (0, 2) and t.grad.shape == (0, 5)
    _, likeliest, which = log_probabilities(t, top=2)
    assert likeliest.shape == which.shape == (0, 2)
    assert log_probabilities(mg.tensor(np.ones((2, 5)), constant=True), [0, 1]).constant
    with mg.no_autodiff:
        assert log_probabilities(mg.tensor(np.zeros((2, 5))), [0, -1]).data.round(3).tolist() == [-1.609, 0]


# ------------------------------------------------------------------------------------------------------------------ distillation
def check_distillation(dtype, z, ids, teacher, temperature=1.0, teacher_dtype=None, seed=0):
    rng, u = np.random.default_rng([seed, *z.shape]), UNIT[dtype][0]
    z, teacher, ids = z.astype(dtype), teacher.astype(teacher_dtype or dtype), np.asarray(ids)
    g = rng.standard_normal(len(z)).astype(wide(dtype))
    t = mg.device_tensor(z)
    loss = distillation(t, ids, mg.device_tensor(teacher, constant=True), temperature=temperature)
    want, dz = ora.distillation(z, ids, teacher, temperature, g)
    per = 1 / temperature
    b = Bars(dtype, z, per)
    y = np.where(ids < 0, -np.inf, teacher.astype(ora.WIDE))
    c = Bars(dtype, y, per)
    taken = np.take_along_axis(b.bounded, np.maximum(ids, 0), 1)
    with np.errstate(invalid="ignore"):
        log_q, log_p = np.where(c.p > 0, c.t - c.log_s, 0), np.where(c.p > 0, taken - b.log_s, 0)
        terms = np.abs(c.p * (log_q - log_p))
        bar = c.p * (c.share * np.abs(log_q - log_p) + 4 * u * (np.abs(c.bounded) + np.abs(taken)) + b.log + c.log)
        bar = np.where(c.p > 0, bar + 4 * u * (terms + c.p * (np.abs(log_q) + np.abs(log_p))), 0)
    bar = bar.sum(-1) + (ids.shape[1] + 8) * u * terms.sum(-1)
    assert loss.dtype == wide(dtype) and loss.shape == want.shape
    close("loss", loss.data, want, bar)
    loss.backward(mg.device_tensor(g, constant=True))
    q, dq = np.zeros_like(b.p), np.zeros_like(b.p)
    for k in range(ids.shape[1]):
        rows, at = np.flatnonzero(ids[:, k] >= 0), ids[ids[:, k] >= 0, k]
        q[rows, at] += c.p[rows, k]
        dq[rows, at] += c.p[rows, k] * (c.share[rows, k] + ids.shape[1] * u)
    size = np.abs(g[:, None]) * per
    bar = size * (b.p * b.share + dq + 8 * u * (b.p + q)) + 4 * TINY[dtype] * (1 + size) + 4 * u * np.abs(dz)
    bar += b.r * (np.abs(dz) + bar) + SMALLEST[dtype]
    assert t.grad.shape == z.shape and t.grad.dtype == dtype
    close("dz", t.grad, dz, bar)


def lessons(rows, vocabulary, count, seed=0):
    rng = np.random.default_rng([seed, rows, vocabulary, count])
    ids = rng.permuted(np.tile(np.arange(vocabulary), (rows, 1)), axis=1)[:, :count] if vocabulary < 3000 else rng.integers(0, vocabulary, (rows, count))
    return ids, -np.sort(-rng.standard_normal((rows, count)) * 2, axis=1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocabulary", [1, 2, 9, 64, 257, 1000, 4096, 4099, 8200, 32003, 70001, 131101])
def test_distillation_lengths_of_rows(dtype, vocabulary):
    check_distillation(dtype, made(4, vocabulary), *lessons(4, vocabulary, min(vocabulary, 8)))
    check_distillation(dtype, made(4, vocabulary), *lessons(4, vocabulary, min(vocabulary, 5)), temperature=2.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocabulary,count", [(1, 600, 1), (1, 5000, 256), (300, 300, 200), (700, 1999, 20), (20000, 17, 3), (2, 60000, 65), (4101, 2300, 70)])
def test_distillation_numbers_of_rows_and_tokens(dtype, rows, vocabulary, count):
    check_distillation(dtype, made(rows, vocabulary), *lessons(rows, vocabulary, count))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocabulary", [50, 120, 250, 500, 520])
@pytest.mark.parametrize("rows,count", [(67, 32), (35, 33), (19, 64), (17, 65), (5, 256)])
def test_distillation_of_short_rows(dtype, vocabulary, rows, count):
    z, (ids, teacher) = made(rows, vocabulary), lessons(rows, max(vocabulary, count), count)
    ids %= vocabulary
    ids[rows // 2, ::3] = ids[rows // 2, 0]  # the same token again and again
    ids[rows // 3] = -1  # a row without a teacher
    check_distillation(dtype, z, ids, teacher, temperature=1.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocabulary", [40, 9000, 70001])
def test_distillation_with_lists_of_all_kinds(dtype, vocabulary):
    ids, teacher = lessons(8, vocabulary, 16)
    z = made(8, vocabulary)
    ids[0] = -1  # none at all
    ids[1, 5:] = -1
    ids[2, ::2] = -1
    ids[3] = ids[3, 0]  # the same one throughout
    ids[4, 3] = ids[4, 9] = ids[4, 15] = vocabulary - 1
    teacher[5, 2:] = -np.inf
    teacher[6] = -np.inf  # none has a chance
    z[7] = -np.inf  # the row has no distribution: the loss is infinite
    check_distillation(dtype, z, ids, teacher)
    check_distillation(dtype, z, ids, teacher, temperature=0.25)


@pytest.mark.parametrize("dtype", DTYPES)
def test_distillation_of_a_token_that_is_ruled_out(dtype):
    ids, teacher = lessons(3, 50, 4)
    z = made(3, 50)
    z[0, ids[0, 1]] = -np.inf
    z[1, ids[1, 0]] = -np.inf
    teacher[1, 0] = -np.inf  # by the teacher, too
    check_distillation(dtype, z, ids, teacher)


@pytest.mark.parametrize("dtype,teacher_dtype", [(np.float16, np.float32), (np.float32, np.float16), (np.float64, np.float32), (np.float64, np.float16)])
def test_teachers_of_other_types(dtype, teacher_dtype):
    check_distillation(dtype, made(5, 700), *lessons(5, 700, 9), teacher_dtype=teacher_dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocabulary", [60, 9000, 70001])
def test_distillation_rows_that_are_no_numbers_stay_alone(dtype, vocabulary):
    ids, teacher = lessons(6, vocabulary, 7)
    z, teacher = made(6, vocabulary).astype(dtype), teacher.astype(dtype)
    ids[3, 4:] = -1
    spoilt, other_teacher = z.copy(), teacher.copy()
    spoilt[1, 2], spoilt[2, vocabulary - 1], other_teacher[3, 1], other_teacher[4, 0] = np.nan, np.inf, np.nan, np.inf
    other_teacher[5, 6], ids[5, 6] = np.nan, -1  # of no token
    results = []
    for values, taught in ((z, teacher), (spoilt, other_teacher)):
        t = mg.device_tensor(values)
        loss = distillation(t, ids, taught, temperature=1.5)
        loss.backward()
        results.append((loss.data, t.grad))
    for clean, other in zip(*results):
        assert np.array_equal(clean[[0, 5]], other[[0, 5]]) and np.isnan(other[1:5]).all()


def test_distillation_the_same_bits_every_time():
    for rows, vocabulary in ((3, 70001), (900, 1500)):
        (ids, teacher), z, runs = lessons(rows, vocabulary, 30), made(rows, vocabulary).astype(np.float32), []
        for _ in range(3):
            t = mg.device_tensor(z)
            loss = distillation(t, ids, teacher.astype(np.float32))
            loss.backward()
            runs.append((loss.data, t.grad))
        assert all(np.array_equal(a, b) for run in runs[1:] for a, b in zip(run, runs[0]))


def test_a_teacher_on_the_device():
    """A teacher's likeliest tokens go on to the student as log_probabilities leaves them."""
    rng = np.random.default_rng(2)
    teacher, student = rng.standard_normal((2, 5, 40)).astype(np.float32) * 2
    t = mg.device_tensor(student)
    _, likeliest, which = log_probabilities(teacher, top=6)
    loss = distillation(t, which, likeliest, temperature=2.0)
    loss.backward()
    assert which._host is None and likeliest.on_device
    want, dz = ora.distillation(student, which.data, np.take_along_axis(teacher, which.data, 1), 2.0, np.ones(5))
    assert np.abs(loss.data - want).max() < 1e-5 and np.abs(t.grad - dz).max() < 1e-6


@pytest.mark.parametrize("vocabulary", [250, 1000, 40001])
def test_gradients_of_many_logits_are_those_of_their_rows(vocabulary):
    rows = 84_000_000 // vocabulary  # half of them are less than 150 MB
    z = made(1000, vocabulary).astype(np.float16)[np.arange(rows) % 1000]
    ids, (lists, teacher) = some(rows, vocabulary), lessons(1000, vocabulary, 7)
    lists, teacher = lists[np.arange(rows) % 1000], teacher[np.arange(rows) % 1000].astype(np.float16)
    for loss in (lambda t, at: log_probabilities(t, ids[at]), lambda t, at: distillation(t, lists[at], teacher[at])):
        found = []
        for at in (slice(None), slice(0, rows // 2), slice(rows // 2, None)):
            t = mg.device_tensor(z[at])
            loss(t, at).backward()
            found.append(t.grad)
        assert np.abs(found[0]).max() > 0
        assert np.array_equal(found[0][: rows // 2], found[1]) and np.array_equal(found[0][rows // 2 :], found[2])


def test_distillation_leading_shapes_and_empty_rows():
    z, (ids, teacher) = made(12, 50), lessons(12, 50, 4)
    flat = distillation(z, ids, teacher).data
    assert np.array_equal(distillation(z.reshape(3, 4, 50), ids.reshape(3, 4, 4), teacher.reshape(3, 4, 4)).data.ravel(), flat)
    assert distillation(z[0], ids[0], teacher[0]).data == flat[0]
    t = mg.tensor(np.ones((0, 5)))
    loss = distillation(t, np.zeros((0, 2), np.int64), np.zeros((0, 2)))
    loss.backward()
    assert loss.shape == (0,) and t.grad.shape == (0, 5)


def test_differences():
    rng = np.random.default_rng(4)
    z, (ids, teacher) = made(3, 11), lessons(3, 11, 4)
    ids[1, 1] = ids[1, 0]
    tokens, g, h = TokenIds([4, -1, 10]), rng.standard_normal((2, 3)), rng.standard_normal(3)
    for f, weights in ((lambda v: log_probabilities(v, tokens, entropy=True), g), (lambda v: distillation(v, ids, teacher, temperature=1.7), h)):
        t = mg.tensor(z)
        f(t).backward(weights)
        total = lambda v: float((f(v).data * weights).sum())
        for index in range(z.size):
            up, down = z.copy(), z.copy()
            up.flat[index] += 1e-6
            down.flat[index] -= 1e-6
            assert abs((total(up) - total(down)) / 2e-6 - t.grad.flat[index]) < 1e-8


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocabulary", [(5, 130), (3, 20001), (600, 333)])
def test_memory_that_begins_anywhere(dtype, rows, vocabulary):
    """Through the C entry points, logits that begin at any multiple of their values' size give the same results; nothing outside is written."""
    from mygrad_amd import _device, _hip

    item, code, lib = np.dtype(dtype).itemsize, _hip.storage_code(dtype), _hip.lib()
    z, ids = made(rows, vocabulary).astype(dtype), some(rows, vocabulary).astype(np.int32)
    lists, teacher = lessons(rows, vocabulary, 5)
    ones = _device.from_host(np.ones(rows, wide(dtype))).buf
    small = [_device.from_host(a).buf for a in (ids, np.ascontiguousarray(lists, np.int32), teacher.astype(dtype))]
    want = []
    for loss in (lambda t: log_probabilities(t, ids, entropy=True, top=3), lambda t: distillation(t, lists, teacher.astype(dtype))):
        t = mg.device_tensor(z)
        out = loss(t)
        out = out[0] if isinstance(out, tuple) else out
        out.backward()
        want.append((out.data, t.grad))
    for shift in (1, 3, 8):
        held = np.full(z.size + 16, 7, dtype)
        held[shift:shift + z.size] = z.ravel()
        given, out, more = _device.from_host(held).buf, _device.from_host(np.full(z.size + 16, 7, dtype)).buf, [_device.DeviceBuffer(rows * 64) for _ in range(5)]
        pz, pdz, room = given.ptr + shift * item, out.ptr + shift * item, [b.ptr for b in more]
        back = np.empty(z.size + 16, dtype)
        _hip.check(lib.mg_log_probabilities_fwd(code, rows, vocabulary, 3, small[0].ptr, pz, *room))
        _hip.check(lib.mg_log_probabilities_bwd(code, rows, vocabulary, small[0].ptr, pz, room[2], ones.ptr, ones.ptr, pdz))
        out.download_into(back)
        assert np.array_equal(back[shift:shift + z.size].reshape(z.shape), want[0][1]) and (back[:shift] == 7).all() and (back[shift + z.size:] == 7).all()
        _hip.check(lib.mg_distillation_fwd(code, code, rows, vocabulary, 5, 1.0, pz, small[1].ptr, small[2].ptr, room[0], room[1], room[2]))
        _hip.check(lib.mg_distillation_bwd(code, rows, vocabulary, 5, 1.0, pz, small[1].ptr, room[1], room[2], ones.ptr, pdz))
        out.download_into(back)
        assert np.array_equal(back[shift:shift + z.size].reshape(z.shape), want[1][1]) and (back[:shift] == 7).all() and (back[shift + z.size:] == 7).all()


def test_entry_points_refuse_bad_arguments():
    from mygrad_amd import _device, _hip

    lib, p = _hip.lib(), _device.DeviceBuffer(1 << 16).ptr
    for status, (dtype, rows, vocabulary, top) in ((-2, (7, 2, 8, 0)), (-1, (0, -1, 8, 0)), (-1, (0, 2, 0, 0)), (-2, (0, 1 << 31, 8, 0)), (-2, (0, 2, 1 << 31, 0)),
                                                   (-1, (0, 2, 8, 9)), (-1, (0, 2, 8, -1)), (-2, (0, 2, 800, 129))):
        assert lib.mg_log_probabilities_fwd(dtype, rows, vocabulary, top, *[p] * 7) == status
        if top == 0:
            assert lib.mg_log_probabilities_bwd(dtype, rows, vocabulary, *[p] * 6) == status
    assert lib.mg_log_probabilities_fwd(0, 2, 8, 0, None, p, p, p, p, None, None) == -1 and lib.mg_log_probabilities_fwd(0, 2, 8, 0, p, None, p, p, p, None, None) == -1
    assert lib.mg_log_probabilities_fwd(0, 2, 8, 2, p, p, p, p, p, None, p) == -1 and lib.mg_log_probabilities_bwd(0, 2, 8, p, p, p, None, None, p) == -1
    for status, (dtype, teacher, rows, vocabulary, count, temperature) in (
            (-2, (7, 7, 2, 8, 2, 1.0)), (-2, (0, 1, 2, 8, 2, 1.0)), (-1, (0, 0, 2, 8, 0, 1.0)), (-2, (0, 0, 2, 8, 257, 1.0)), (-1, (0, 0, 2, 8, 2, 0.0)),
            (-1, (0, 0, 2, 8, 2, float("nan"))), (-1, (0, 0, 2, 8, 2, 1e40)), (-1, (0, 0, 2, 8, 2, -1.0)), (-1, (0, 0, -2, 8, 2, 1.0))):
        assert lib.mg_distillation_fwd(dtype, teacher, rows, vocabulary, count, temperature, *[p] * 6) == status
        if dtype == teacher:
            assert lib.mg_distillation_bwd(dtype, rows, vocabulary, count, temperature, *[p] * 6) == status
    assert lib.mg_distillation_fwd(0, 0, 2, 8, 2, 1.0, p, p, p, None, p, p) == -1 and lib.mg_distillation_bwd(0, 2, 8, 2, 1.0, p, p, p, p, p, None) == -1
    assert lib.mg_distillation_fwd(0, 0, 0, 8, 2, 1.0, *[None] * 6) == 0 and lib.mg_log_probabilities_bwd(0, 0, 8, *[None] * 6) == 0
