"""The operators of a language model together, as a program uses them: a model's gradients against differences and a plain
implementation, a student that learns from a teacher's likeliest tokens, tokens generated one at a time."""

import numpy as np
import pytest

import mygrad_amd as mg
from mygrad_amd.nnet import AttentionMask, KeyValueCache, TokenIds, attention, distillation, embedding, layer_norm, log_probabilities
from oracle import language as ora

pytestmark = pytest.mark.gpu

VOCABULARY, WIDTH, HEADS, DIM, EPS = 23, 12, 2, 8, 1e-5


@pytest.fixture(scope="module", autouse=True)
def device():
    if not mg.is_available():
        pytest.fail("libmygrad_hip.so / gfx950 device not available: the GPU tests need both")


def weights(seed=0, dtype=np.float64):
    rng = np.random.default_rng(seed)
    shapes = {"table": (VOCABULARY, WIDTH), "w1": (WIDTH,), "b1": (WIDTH,), "q": (WIDTH, HEADS, DIM), "k": (WIDTH, HEADS, DIM), "v": (WIDTH, HEADS, DIM),
              "out": (HEADS, DIM, WIDTH), "w2": (WIDTH,), "b2": (WIDTH,)}
    return {name: (rng.standard_normal(shape) * (0.3 if len(shape) > 1 else 0.1) + (name in ("w1", "w2"))).astype(dtype) for name, shape in shapes.items()}


def model(w, tokens, mask=None, cache=None):
    """Logits ``(batch, tokens, vocabulary)``; the table that tokens are looked up in gives the logits, too."""
    x = layer_norm(embedding(w["table"], tokens, scale=WIDTH**0.5), w["w1"], w["b1"], eps=EPS)
    q, k, v = (mg.einsum("btc,chd->bthd", x, w[name]) for name in "qkv")
    if cache is None:
        y = attention(q, k, v, mask=mask)
    else:
        cache.write(k, v, mask)
        y = cache.attend(q, mask=mask)
    y = layer_norm(mg.einsum("bthd,hdc->btc", y, w["out"]), w["w2"], w["b2"], eps=EPS)
    return mg.einsum("btc,vc->btv", y, w["table"])


def plain(w, ids):
    """The same in NumPy, one sequence after another."""
    w = {name: value.astype(ora.WIDE) for name, value in w.items()}
    x = ora.layer_norm(ora.embedding(w["table"], ids, WIDTH**0.5), w["w1"], w["b1"], EPS)
    q, k, v = (np.einsum("btc,chd->bthd", x, w[name]) for name in "qkv")
    s = np.einsum("bqhd,bkhd->bhqk", q, k) / DIM**0.5
    s = np.where(np.tril(np.ones(s.shape[-2:], bool)), s, -np.inf)
    p = np.exp(s - s.max(-1, keepdims=True))
    y = np.einsum("bhqk,bkhd->bqhd", p / p.sum(-1, keepdims=True), v)
    y = ora.layer_norm(np.einsum("bthd,hdc->btc", y, w["out"]), w["w2"], w["b2"], EPS)
    return np.einsum("btc,vc->btv", y, w["table"])


def batch(seed=1, rows=3, length=7):
    rng = np.random.default_rng(seed)
    ids = rng.integers(0, VOCABULARY, (rows, length + 1))
    ids[0, -2:] = -1  # a padded row
    return ids[:, :-1], ids[:, 1:]


def test_a_models_loss_and_its_gradients_by_differences():
    ids, targets = batch()
    given, told = weights(), TokenIds(targets)
    coefficients = np.random.default_rng(3).standard_normal((2, *targets.shape))

    def loss(w):
        return mg.sum(log_probabilities(model(w, TokenIds(ids), AttentionMask(causal=True)), told, entropy=True) * coefficients)

    tensors = {name: mg.device_tensor(value) for name, value in given.items()}
    out = loss(tensors)
    scores, entropy, _ = ora.log_probabilities(plain(given, ids).reshape(-1, VOCABULARY), targets.ravel())
    assert abs(float(out.data) - float((np.stack((scores, entropy)).reshape(coefficients.shape) * coefficients).sum())) < 1e-12
    out.backward()
    rng = np.random.default_rng(5)
    for name, value in given.items():
        assert tensors[name].grad.shape == value.shape
        for index in rng.permutation(value.size)[:5]:
            moved = []
            for step in (1e-6, -1e-6):
                changed = {**given, name: value.copy()}
                changed[name].flat[index] += step
                with mg.no_autodiff:
                    moved.append(float(loss(changed).data))
            assert abs((moved[0] - moved[1]) / 2e-6 - tensors[name].grad.flat[index]) < 2e-7, (name, index)


def test_a_student_and_its_teacher():
    """The teacher's alternatives stay on the device; the student's gradient against the formulas."""
    ids, _ = batch()
    teacher, student = weights(7, np.float32), weights(8, np.float32)
    with mg.no_autodiff:
        _, likeliest, which = log_probabilities(model(teacher, ids, AttentionMask(causal=True)), top=5)
    tensors = {name: mg.device_tensor(value) for name, value in student.items()}
    logits = model(tensors, ids, AttentionMask(causal=True))
    loss = distillation(logits, which, likeliest, temperature=2.0)
    loss.backward()
    assert which._host is None and likeliest.on_device and logits.on_device
    z = plain(student, ids).reshape(-1, VOCABULARY)
    want, dz = ora.distillation(z, which.data.reshape(-1, 5), likeliest.data.reshape(-1, 5), 2.0, np.ones(len(z)))
    assert np.abs(loss.data.ravel() - want).max() < 1e-5
    assert np.abs(logits.grad.reshape(z.shape) - dz).max() < 1e-5
    assert np.array_equal(which.data, ora.likeliest(plain(teacher, ids), 5))


def test_tokens_one_at_a_time():
    """Each likeliest token goes on to the embedding as the kernel left it; the cache gives what all tokens at once give."""
    given = weights(9)
    tensors = {name: mg.device_tensor(value, constant=True) for name, value in given.items()}
    ids = np.random.default_rng(2).integers(0, VOCABULARY, (2, 3))
    cache, row, length, step = KeyValueCache(2, 9, HEADS, DIM, dtype=np.float64), ids, 3, TokenIds(ids)
    with mg.no_autodiff:
        for _ in range(6):
            logits = model(tensors, step, AttentionMask(causal=True, lengths=length), cache)
            entropies, likeliest, which = log_probabilities(logits, entropy=True, top=1)
            want = plain(given, row)[:, -step.shape[1]:]
            assert np.abs(logits.data - want).max() < 1e-12 and np.abs(entropies.data - ora.log_probabilities(want.reshape(-1, VOCABULARY))[1].reshape(want.shape[:2])).max() < 1e-12
            last = which.data[:, -1:, 0] if step.shape[1] > 1 else None
            step = TokenIds(last) if last is not None else which.reshape(2, 1)
            row, length = np.concatenate((row, step.data), 1), length + 1
    assert row.shape == (2, 9) and np.array_equal(row[:, 3:], ora.likeliest(plain(given, row), 1)[:, 2:-1, 0])


def test_what_float16_chains():
    """Lookup, norm, attention and losses take float16 from one another; results against 64 bits of the same rounded operands."""
    rng = np.random.default_rng(0)
    table, w = (rng.standard_normal((VOCABULARY, 16)) * 0.5).astype(np.float16), rng.standard_normal(16).astype(np.float16)
    ids, targets = rng.integers(0, VOCABULARY, (2, 2, 6))
    t, tw = mg.device_tensor(table), mg.device_tensor(w)
    x = embedding(t, ids)
    y = layer_norm(x, tw, eps=EPS)
    scores = log_probabilities(y, targets % 16)
    assert x.dtype == y.dtype == np.float16 and scores.dtype == np.float32
    scores.backward()
    want = ora.log_probabilities(y.data.reshape(-1, 16), (targets % 16).ravel(), np.ones(12))
    assert np.abs(scores.data.ravel() - want[0]).max() < 1e-6
    dy = want[2].astype(np.float16)
    dx = ora.layer_norm(x.data, w, None, EPS, dy.reshape(y.shape))[1].astype(np.float16)
    dt = ora.embedding(table, ids, 1.0, dx)[1]
    # two roundings of float16 on the way, each of half a unit of its value and, where it falls the other way than here, one
    bar = 2.0**-10 * (np.abs(dt) + ora.embedding(table, ids, 1.0, np.abs(dx) + np.abs(dx).max(-1, keepdims=True))[1]) + 2.0**-24 * 12
    assert t.grad.dtype == np.float16 and (np.abs(t.grad - dt) <= bar).all()


def test_numbers_of_numpys_types():
    """``eps``, ``scale``, ``temperature`` and ``top`` as NumPy's scalars."""
    x = np.random.default_rng(0).standard_normal((3, 8)).astype(np.float32)
    assert np.array_equal(layer_norm(x, eps=np.float32(0.5)).data, layer_norm(x, eps=0.5).data)
    assert np.array_equal(embedding(x, [0, 2], scale=np.float32(0.25)).data, embedding(x, [0, 2], scale=0.25).data)
    assert np.array_equal(embedding(x, np.array([0, 2], np.uint8), scale=np.int64(2)).data, x[[0, 2]] * 2)
    assert np.array_equal(log_probabilities(x, top=np.int64(2))[2].data, log_probabilities(x, top=2)[2].data)
    assert np.array_equal(*(distillation(x, [[0], [1], [2]], x[:, :1], temperature=t).data for t in (np.float32(2), 2)))


@pytest.mark.parametrize("dtype", [np.float16, np.float32, np.float64])
def test_arrays_of_any_order(dtype):
    rng = np.random.default_rng(0)
    whole, ids, lists = rng.standard_normal((14, 22)).astype(dtype), rng.integers(0, 11, (7, 2)), rng.integers(0, 11, (14, 5))
    params, teacher = rng.standard_normal((11, 4)).astype(dtype), rng.standard_normal((14, 5)).astype(dtype)
    views = [(whole[::2, ::-2], ids[:, 1], params[:, 1], params[:, 2], lists[::-2, 1:3], teacher[1::2, ::3]),
             (np.asfortranarray(whole[:7, :11]), ids.T[0], params[::-1, 3], params[:, 0], np.asfortranarray(lists[:7]), np.asfortranarray(teacher[7:]))]
    for x, tokens, w, b, which, taught in views:
        for f in (lambda x, tokens, w, b, which, taught: layer_norm(x, w, b, eps=1e-3),
                  lambda x, tokens, w, b, which, taught: embedding(x, tokens % 7),
                  lambda x, tokens, w, b, which, taught: log_probabilities(x, tokens, entropy=True),
                  lambda x, tokens, w, b, which, taught: distillation(x, which, taught, temperature=2.0)):
            found = []
            for arrays in ((x, tokens, w, b, which, taught), tuple(np.ascontiguousarray(a) for a in (x, tokens, w, b, which, taught))):
                t, tw, tb = (mg.Tensor(arrays[n], copy=False) for n in (0, 2, 3))
                y = f(t, arrays[1], tw, tb, *arrays[4:])
                g = rng.standard_normal(y.shape).astype(y.dtype) if not found else found[-1]
                y.backward(np.asfortranarray(g))
                found += [[y.data] + [p.grad for p in (t, tw, tb) if p.grad is not None], g]
            assert len(found[0]) == len(found[2]) and all(np.array_equal(a, c) for a, c in zip(found[0], found[2]))


def test_one_tensor_in_several_places():
    """Its gradients are added up: those of a row that is its own weight and bias, and those of a table that is looked up, normed and scored."""
    rng = np.random.default_rng(1)
    x, g = rng.standard_normal(33), rng.standard_normal(33)
    t = mg.Tensor(x)
    layer_norm(t, t, t, eps=1e-2).backward(g)
    parts = ora.layer_norm(x, x, x, 1e-2, g)
    assert np.abs(t.grad - (parts[1] + parts[2] + parts[3])).max() < 1e-12
    table, ids = rng.standard_normal((9, 9)), rng.integers(0, 9, 6)
    t = mg.Tensor(table)
    log_probabilities(layer_norm(embedding(t, ids), t_row := mg.Tensor(table[0]), t_row, eps=1e-2), ids).backward()
    first = t.grad.copy()
    for n in range(9):
        moved = []
        for step in (1e-6, -1e-6):
            other = table.copy()
            other[ids[0], n] += step
            moved.append(log_probabilities(layer_norm(embedding(other, ids), table[0], table[0], eps=1e-2), ids).data.sum())
        assert abs((moved[0] - moved[1]) / 2e-6 - first[ids[0], n]) < 1e-7


@pytest.mark.parametrize("dtype", [np.float16, np.float32, np.float64])
def test_results_without_a_graph(dtype):
    """Arrays that no graph holds are sent for one call; operands of the same size do not take one another's place."""
    rng = np.random.default_rng(3)
    for rows, width in ((64, 8), (300, 1), (7, 33)):
        x, w, ids = rng.standard_normal((rows, width)).astype(dtype), rng.standard_normal(width).astype(dtype), rng.integers(0, width, rows)
        lists = rng.integers(0, width, (rows, width * x.itemsize // 4 or 1))
        teacher = rng.standard_normal(lists.shape).astype(dtype)
        for f in (lambda: layer_norm(x, w, w, eps=1e-3), lambda: embedding(x, ids % rows), lambda: log_probabilities(x, ids, entropy=True),
                  lambda: log_probabilities(x, top=1)[1], lambda: distillation(x, lists, teacher), lambda: distillation(x, lists, teacher, temperature=3)):
            with_graph = f().data.copy()
            with mg.no_autodiff:
                assert np.array_equal(f().data, with_graph)
            with mg.mem_guard_off:
                assert np.array_equal(f().data, with_graph)
        g = rng.standard_normal(rows)
        grads = []
        for switch in (mg.mem_guard_on, mg.mem_guard_off):
            with switch:
                for f in (lambda t: layer_norm(t, w, w, eps=1e-3), lambda t: embedding(t, ids % rows), lambda t: log_probabilities(t, ids),
                          lambda t: distillation(t, lists, teacher)):
                    t = mg.Tensor(x.copy())
                    y = f(t)
                    y.backward(g if y.ndim == 1 else g[:, None] * np.ones(width))
                    grads.append(t.grad)
        assert all(np.array_equal(a, b) for a, b in zip(grads[:4], grads[4:]))
