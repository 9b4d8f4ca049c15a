"""What embedding, layer norm, log probabilities and distillation check on the host, and the oracle they are held to."""

import numpy as np
import pytest

import mygrad_amd as mg
from mygrad_amd.nnet import TokenIds, distillation, embedding, layer_norm, log_probabilities
from oracle import language as ora
from tests.test_host import run_on_standins


@pytest.mark.parametrize("ids,error", [([0.0, 1.0], TypeError), ([True, False], TypeError), ([-2, 0], ValueError), ([2**31 - 1], ValueError), ([2**40], ValueError),
                                       (np.array([2**63], np.uint64), ValueError), (["a"], TypeError)])
def test_what_is_no_tokens(ids, error):
    with pytest.raises(error):
        TokenIds(ids)


def test_tokens_are_kept_as_they_were():
    ids = np.array([[3, -1], [0, 7]])
    tokens = TokenIds(ids)
    ids[0, 0] = 100
    assert tokens.data.dtype == np.int32 and tokens.data.tolist() == [[3, -1], [0, 7]] and tokens.below == 8 and tokens.shape == (2, 2) and tokens.size == 4
    for name in ("shape", "below", "data", "size", "ndim"):
        with pytest.raises(AttributeError):
            setattr(tokens, name, 1)
    with pytest.raises(ValueError):
        tokens.data[0, 0] = 1
    assert tokens.reshape(-1).data.tolist() == [3, -1, 0, 7] and tokens.reshape(4, 1).below == 8 and TokenIds([]).below == 0 and TokenIds(5).shape == ()
    assert TokenIds(mg.tensor([1, 2])).data.tolist() == [1, 2] and np.asarray(tokens).tolist() == tokens.data.tolist() and len(tokens) == 2
    with pytest.raises(ValueError):
        tokens.reshape(3)


W, X = np.ones((5, 4), np.float32), np.ones((2, 3, 4), np.float32)


@pytest.mark.parametrize("call,error", [
    (lambda: embedding(W, [5]), ValueError), (lambda: embedding(W, TokenIds([0, 5])), ValueError), (lambda: embedding(W, [0.5]), TypeError),
    (lambda: embedding(np.ones(5), [0]), ValueError), (lambda: embedding(np.ones((2, 5, 4)), [0]), ValueError), (lambda: embedding(W.astype(int), [0]), TypeError),
    (lambda: embedding(W, [0], scale=np.inf), ValueError), (lambda: embedding(W, [0], scale=np.nan), ValueError), (lambda: embedding(W, [0], scale=None), ValueError),
    (lambda: embedding(W, [0], scale=1e31), ValueError), (lambda: embedding(W, [[0], [1, 2]]), (TypeError, ValueError)),
])
def test_embedding_refuses(call, error):
    with pytest.raises(error):
        call()


@pytest.mark.parametrize("call,error", [
    (lambda: layer_norm(np.float32(3), eps=1e-5), ValueError), (lambda: layer_norm(X.astype(int), eps=1e-5), TypeError), (lambda: layer_norm(X, eps=None), TypeError),
    (lambda: layer_norm(X, eps=-1.0), ValueError), (lambda: layer_norm(X, eps=np.nan), ValueError), (lambda: layer_norm(X, eps=np.inf), ValueError),
    (lambda: layer_norm(X, np.ones(3, np.float32), eps=1e-5), ValueError), (lambda: layer_norm(X, np.ones((3, 4), np.float32), eps=1e-5), ValueError),
    (lambda: layer_norm(X, np.ones(4), eps=1e-5), TypeError), (lambda: layer_norm(X, None, np.ones(4, np.float16), eps=1e-5), TypeError),
    (lambda: layer_norm(X, np.ones(0, np.float32), eps=1e-5), ValueError), (lambda: layer_norm(X, None, np.ones((4, 0), np.float32), eps=1e-5), ValueError),
    (lambda: layer_norm(X, None, np.ones(1, np.float32), eps=1e-5), ValueError),
])
def test_layer_norm_refuses(call, error):
    with pytest.raises(error):
        call()


@pytest.mark.parametrize("call,error", [
    (lambda: log_probabilities(X), TypeError), (lambda: log_probabilities(X, np.zeros((2, 3), int) + 4), ValueError), (lambda: log_probabilities(X, [0, 1]), ValueError),
    (lambda: log_probabilities(X, np.zeros((2, 3))), TypeError), (lambda: log_probabilities(X, np.zeros((2, 3, 1), int)), ValueError),
    (lambda: log_probabilities(X, top=5), ValueError), (lambda: log_probabilities(X, top=-1), ValueError), (lambda: log_probabilities(X, top=1.0), ValueError),
    (lambda: log_probabilities(X, top=True), ValueError), (lambda: log_probabilities(np.ones((2, 500)), top=129), ValueError),
    (lambda: log_probabilities(X, entropy=1), TypeError), (lambda: log_probabilities(X.astype(int), top=1), TypeError), (lambda: log_probabilities(np.ones((3, 0)), top=0, entropy=True), ValueError),
    (lambda: log_probabilities(np.float32(1), entropy=True), ValueError), (lambda: log_probabilities(X, np.zeros((2, 3), int), constant=1), TypeError),
])
def test_log_probabilities_refuses(call, error):
    with pytest.raises((error, mg.HipUnavailable) if not mg.is_available() and error is TypeError else error):
        call()


IDS, TAUGHT = np.zeros((2, 3, 2), int), np.ones((2, 3, 2), np.float32)


@pytest.mark.parametrize("call,error", [
    (lambda: distillation(X, IDS[0], TAUGHT), ValueError), (lambda: distillation(X, IDS, TAUGHT[0]), ValueError), (lambda: distillation(X, IDS + 4, TAUGHT), ValueError),
    (lambda: distillation(X, IDS[:, :, :0], TAUGHT[:, :, :0]), ValueError), (lambda: distillation(X[0, 0], 0, np.float32(1)), ValueError),
    (lambda: distillation(np.ones((2, 9)), np.zeros((2, 257), int), np.ones((2, 257))), ValueError), (lambda: distillation(X, IDS, mg.tensor(TAUGHT)), ValueError),
    (lambda: distillation(X, IDS, TAUGHT.astype(np.float64)), TypeError), (lambda: distillation(X, IDS, TAUGHT.astype(int)), TypeError),
    (lambda: distillation(X.astype(int), IDS, TAUGHT), TypeError), (lambda: distillation(X, IDS * 0.5, TAUGHT), TypeError),
    (lambda: distillation(X, IDS, TAUGHT, temperature=0), ValueError), (lambda: distillation(X, IDS, TAUGHT, temperature=-1.0), ValueError),
    (lambda: distillation(X, IDS, TAUGHT, temperature=np.nan), ValueError), (lambda: distillation(X, IDS, TAUGHT, temperature=1e31), ValueError),
    (lambda: distillation(X, IDS, TAUGHT, temperature="1"), ValueError),
])
def test_distillation_refuses(call, error):
    with pytest.raises(error):
        call()


def test_a_refused_call_leaves_arrays_writeable():
    w, z = np.ones((5, 4)), np.ones((2, 4))
    for call in (lambda: embedding(w, [7]), lambda: layer_norm(z, w, eps=1e-5), lambda: log_probabilities(z, [4, 0]), lambda: distillation(z, IDS, z)):
        with pytest.raises(ValueError):
            call()
    w[0, 0] = z[0, 0] = 2


def test_what_is_refused_does_not_hang_on_the_calls_before(tmp_path):
    """Numbers of other types are equal to those of a call that was checked, and have its hash."""
    program = """
from decimal import Decimal
from fractions import Fraction
import numpy as np
import mygrad_amd as mg
from mygrad_amd.nnet import distillation, layer_norm, log_probabilities
z, ids, teacher = np.ones((2, 9), np.float32), np.zeros((2, 3), int), np.ones((2, 3), np.float32)
def refused(f):
    try:
        f()
    except (TypeError, ValueError) as error:
        return type(error)
for once in range(2):
    assert refused(lambda: distillation(z, ids, teacher, temperature=Decimal(2))) is ValueError
    assert refused(lambda: distillation(z, ids, teacher, temperature=2 + 0j)) is ValueError
    assert refused(lambda: layer_norm(z, eps=0.5 + 0j)) is TypeError
    assert refused(lambda: log_probabilities(z, top=2.0)) is ValueError and refused(lambda: log_probabilities(z, entropy=1)) is TypeError
    assert refused(lambda: log_probabilities(z, top=Fraction(2))) is ValueError
    for fits in (2.0, 2, np.float32(2), Fraction(2)):
        distillation(z, ids, teacher, temperature=fits)
    layer_norm(z, eps=0.5)
    log_probabilities(z, entropy=True, top=2)
print("the same")
"""
    assert "the same" in run_on_standins(tmp_path, program)


def test_alternatives_alone_refuse_a_constant_that_is_none(tmp_path):
    program = """
import numpy as np
import mygrad_amd as mg
from mygrad_amd.nnet import log_probabilities
for kwargs in (dict(top=1), dict(top=1, entropy=True), dict(entropy=True)):
    for rows in (0, 2):
        for constant in (1, "no"):
            try:
                log_probabilities(np.ones((rows, 5)), constant=constant, **kwargs)
            except TypeError:
                continue
            raise AssertionError((kwargs, rows, constant))
        for constant in (None, True, False):
            log_probabilities(np.ones((rows, 5)), constant=constant, **kwargs)
print("refused")
"""
    assert "refused" in run_on_standins(tmp_path, program)


def test_one_upload_of_tokens_and_of_what_they_go_with(tmp_path):
    """Tokens are sent once, whoever takes them; what a backward pass needs is kept for those that have one."""
    program = """
import numpy as np
import mygrad_amd as mg
from mygrad_amd.nnet import TokenIds, distillation, embedding, layer_norm, log_probabilities
tokens, lists = TokenIds([[1, -1, 2]]), TokenIds(np.zeros((1, 3, 2), int))
weight, x = mg.device_tensor(np.ones((4, 8), np.float16)), mg.device_tensor(np.ones((1, 3, 4), np.float16))
teacher = mg.device_tensor(np.ones((1, 3, 2), np.float16), constant=True)
for n in range(3):
    back = lambda out: out.backward(mg.device_tensor(np.ones(out.shape, out.dtype), constant=True))
    y = embedding(weight, tokens)
    z = layer_norm(y, eps=1e-5)
    back(z)
    assert weight.grad.shape == (4, 8) and weight.grad.dtype == np.float16
    scores, likeliest, which = log_probabilities(x, tokens, entropy=True, top=2)
    back(scores)
    assert x.grad.shape == (1, 3, 4) and x.grad.dtype == np.float16
    loss = distillation(x, lists, teacher)
    back(loss)
    assert x.grad.shape == (1, 3, 4) and x.grad.dtype == np.float16
    assert y.shape == z.shape == (1, 3, 8) and y.dtype == z.dtype == np.float16 and scores.dtype == loss.dtype == likeliest.dtype == np.float32
    assert scores.shape == (2, 1, 3) and loss.shape == (1, 3) and which.shape == likeliest.shape == (1, 3, 2) and likeliest.constant and not scores.constant
    if n == 0:
        held = tokens._buffer(), lists._buffer()
assert tokens._buffer() is held[0] and lists._buffer() is held[1]
constant = mg.device_tensor(np.ones((1, 3, 4), np.float16), constant=True)
assert log_probabilities(constant, tokens).creator._kept is None and distillation(constant, lists, teacher).creator._kept is None
seen = log_probabilities(x, top=1)
assert seen[0] is None and seen[2].below == 4 and seen[2].reshape(3).shape == (3,)
print("sent once")
"""
    assert "sent once" in run_on_standins(tmp_path, program)


def test_operands_live_until_the_launch(tmp_path):
    """What is sent for one call only (arrays that no graph holds, casts) is not given back, and so not given to the next who asks, before the call."""
    program = """
import weakref
import numpy as np
import mygrad_amd as mg
from mygrad_amd import _device, _hip
from mygrad_amd.nnet import distillation, embedding, layer_norm, log_probabilities
lib, live, seen = _hip.lib(), weakref.WeakSet(), set()
made = _device.DeviceBuffer.__init__
def init(self, nbytes):
    made(self, nbytes)
    live.add(self)
_device.DeviceBuffer.__init__ = init
class Watched:
    def __getattr__(self, name):
        f = getattr(lib, name)
        if not name.endswith(("_fwd", "_bwd")):
            return f
        def call(*args):
            held = [(b.ptr, b.ptr + max(b.nbytes, 1)) for b in live if b._owned is not None]
            for n, arg in enumerate(args):
                assert not isinstance(arg, int) or arg < 1 << 20 or any(first <= arg < end for first, end in held), (name, n)
            seen.add(name)
            return f(*args)
        return call
_hip._lib = Watched()
rng = np.random.default_rng(0)
for dtype in (np.float16, np.float32, np.float64):
    x, w, ids, lists = np.ones((6, 4), dtype), np.ones(4, dtype), np.zeros(6, int), np.zeros((6, 4), int)
    teacher = np.ones((6, 4), np.float16)
    calls = (lambda x: embedding(x, ids), lambda x: layer_norm(x, w, w, eps=1e-5), lambda x: log_probabilities(x, ids, entropy=True, top=2)[0],
             lambda x: log_probabilities(x, top=2)[1], lambda x: distillation(x, lists, teacher))
    for f in calls:
        with mg.no_autodiff:
            f(x)
        f(x)
        for switch in (mg.mem_guard_off, mg.mem_guard_on):
            with switch:
                t = mg.tensor(x)
                y = f(t)
                if not y.constant:
                    y.backward(np.ones(y.shape, np.float64))
                    assert t.grad.shape == x.shape
                    y = f(t)
                    y.backward(mg.device_tensor(np.ones(y.shape, y.dtype), constant=True))
assert len(seen) == 8, seen
print("live")
"""
    assert "live" in run_on_standins(tmp_path, program)


def test_as_many_tokens_as_are_allowed_fit_the_grids(tmp_path):
    """A lookup of long rows takes a block of 256 threads for four tokens, and a launch has fewer than 2^32 threads."""
    program = """
from mygrad_amd import _device, _hip
lib, p = _hip.lib(), _device.DeviceBuffer(1 << 16).ptr
for dtype in (0, 1, 2):
    for dim in (1, 700, 4096, 1 << 24):
        for tokens in ((1 << 26) - 5, (1 << 26) - 4, (1 << 26) - 3, (1 << 26) - 1):
            assert lib.mg_embedding_fwd(dtype, tokens, 3, dim, 1.0, p, p, p) == 0, (dtype, dim, tokens)
        assert lib.mg_embedding_fwd(dtype, 1 << 26, 3, dim, 1.0, p, p, p) == -2
    assert lib.mg_embedding_bwd(dtype, (1 << 26) - 1, 3, 1, 1.0, p, p, p) == 0
print("they fit")
"""
    assert "they fit" in run_on_standins(tmp_path, program)


# ------------------------------------------------------------------------------------------------------------------- the oracle
def test_the_oracles_gradients_by_differences():
    rng = np.random.default_rng(0)
    x, w, b, g = rng.standard_normal((3, 7)), rng.standard_normal(7), rng.standard_normal(7), rng.standard_normal((3, 7))
    z, ids, h = rng.standard_normal((3, 7)), np.array([2, -1, 6]), rng.standard_normal((2, 3))
    lists, teacher = np.array([[1, 4, 4], [0, -1, 6], [-1, -1, -1]]), rng.standard_normal((3, 3))
    total = lambda *ops: (ora.layer_norm(*ops, eps=1e-3) * g).sum()
    scored = lambda v: (np.stack(ora.log_probabilities(v, ids)[:2]) * h).sum()
    taught = lambda v: (ora.distillation(v, lists, teacher, 1.3) * h[0]).sum()
    cases = [(lambda v: total(v, w, b), x, ora.layer_norm(x, w, b, 1e-3, g)[1]), (lambda v: total(x, v, b), w, ora.layer_norm(x, w, b, 1e-3, g)[2]),
             (lambda v: total(x, w, v), b, ora.layer_norm(x, w, b, 1e-3, g)[3]), (scored, z, ora.log_probabilities(z, ids, *h)[2]),
             (taught, z, ora.distillation(z, lists, teacher, 1.3, h[0])[1]),
             (lambda v: (ora.embedding(v, ids, 0.7) * g).sum(), rng.standard_normal((8, 7)), ora.embedding(np.zeros((8, 7)), ids, 0.7, g)[1])]
    for f, at, grad in cases:
        for index in range(at.size):
            up, down = at.copy(), at.copy()
            up.flat[index] += 1e-6
            down.flat[index] -= 1e-6
            assert abs((f(up) - f(down)) / 2e-6 - grad.flat[index]) < 1e-7


def test_the_oracle_of_rows_without_a_distribution():
    z = np.array([[-np.inf, -np.inf], [0.0, -np.inf], [0.0, 0.0]])
    scores, entropy, dz = ora.log_probabilities(z, [0, 0, 1], np.ones(3), np.ones(3))
    two = float(np.log(2))
    assert scores.astype(float).tolist() == [-np.inf, 0.0, -two] and entropy.astype(float).tolist() == [0.0, 0.0, two] and not dz[:2].any()
    loss, dz = ora.distillation(z, [[0, 1]] * 3, np.zeros((3, 2)), 1.0, np.ones(3))
    assert np.isinf(loss[:2]).all() and loss[2] == 0 and not dz[0].any()
    assert ora.likeliest([[1.0, 2.0, 2.0, -np.inf]], 4).tolist() == [[1, 2, 0, 3]]


def test_a_tensor_that_is_only_read_collects_no_dead_operations(tmp_path):
    """Weights that answer and are never trained: what is gone is dropped, what lives is kept."""
    program = """
import numpy as np
import mygrad_amd as mg
from mygrad_amd.nnet import embedding
weight = mg.device_tensor(np.ones((4, 8), np.float32))
live = [embedding(weight, [n]) for n in range(3)]
for n in range(500):
    embedding(weight, [1])
assert len(weight._ops) <= 40 and {out.creator for out in live} <= {ref() for ref in weight._ops}
live[1].backward(mg.device_tensor(np.ones((1, 8), np.float32), constant=True))
assert weight.grad.shape == (4, 8)
print("dropped")
"""
    assert "dropped" in run_on_standins(tmp_path, program)


def test_a_tensor_that_feeds_many_live_operations(tmp_path):
    """What is looked through for dead references grows with the number of operations, not with its square; dropping them goes on once there are some."""
    program = """
import weakref
import numpy as np
import mygrad_amd as mg
from mygrad_amd import tensor_base
from mygrad_amd.nnet import embedding
looked = [0]
class Counted(weakref.ref):
    def __call__(self):
        looked[0] += 1
        return super().__call__()
tensor_base.ReferenceType = Counted
for weight in (mg.device_tensor(np.ones((4, 8), np.float32)), mg.tensor(np.ones((4, 8), np.float32))):
    looked[0], live = 0, []
    for n in range(3000):
        live.append(embedding(weight, [n % 4]))
    assert looked[0] <= 4 * 3000, looked  # the tensor's operations and those that hold it read-only, less than twice each
    assert {out.creator for out in live} <= {ref() for ref in weight._ops}
    looked[0] = 0
    for n in range(9000):
        embedding(weight, [1])
    assert len(weight._ops) <= 6000 and len(weight._guards) <= 6000 and looked[0] <= 4 * 9000, (len(weight._ops), looked)
    del live
    for n in range(9000):
        embedding(weight, [1])
    assert len(weight._ops) <= 32 and len(weight._guards) <= 32
print("counted")
"""
    assert "counted" in run_on_standins(tmp_path, program)


def test_arrays_read_from_a_live_graph_are_released_with_it(tmp_path):
    """Where all operands lie on the device, nothing is held until somebody reads them; then until the operation is gone."""
    program = """
import numpy as np
import mygrad_amd as mg
from mygrad_amd import _graph
from mygrad_amd.nnet import layer_norm
x, w = mg.device_tensor(np.ones((2, 8), np.float32)), mg.device_tensor(np.ones(8, np.float32))
y = layer_norm(x, w, eps=1e-5)
z = layer_norm(y, eps=1e-5)
assert _graph.held_count() == 0
arrays = [t.data for t in (x, y, w, z)]
assert _graph.held_count() == len(arrays) and not any(a.flags.writeable for a in arrays)
z.backward(mg.device_tensor(np.ones((2, 8), np.float32), constant=True))
assert _graph.held_count() == 0 and all(a.flags.writeable for a in arrays)
y = layer_norm(mg.device_tensor(np.ones((2, 8), np.float32)), eps=1e-5)
held = y.data
assert not held.flags.writeable
del y
assert held.flags.writeable and _graph.held_count() == 0
print("released")
"""
    assert "released" in run_on_standins(tmp_path, program)
