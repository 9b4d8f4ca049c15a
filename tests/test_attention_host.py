"""What attention and the norm of heads do without a GPU: their refusals, the masks' bookkeeping, and the oracle that the GPU
tests go by, itself held against differences."""

import ctypes

import numpy as np
import pytest

import mygrad_amd as mg
from mygrad_amd import _hip
from mygrad_amd.nnet import AttentionMask, KeyValueCache, RotaryTable, attention, head_norm, rotate
from mygrad_amd.nnet.layers.attention import _runs
from oracle import attention as ora


def test_descriptors_match_the_header():
    assert ctypes.sizeof(_hip.AttentionDesc) == 8 + 7 * 8 + 2 * 8 + 7 * 8
    assert ctypes.sizeof(_hip.HeadNormDesc) == 6 * 4 + 5 * 8 + 8 + 2 * 8


def test_attention_refuses_what_it_does_not_take():
    x = np.ones((2, 5, 4, 8), dtype=np.float32)
    for bad in (
        lambda: attention(x[0], x, x),  # axes
        lambda: attention(x, x[:1], x[:1]),  # batch
        lambda: attention(x, x[..., :4], x[..., :4]),  # head dimension
        lambda: attention(x, x, x[:, :4]),  # k and v differ
        lambda: attention(x, x[:, :, :3], x[:, :, :3]),  # heads that are no multiple
        lambda: attention(np.ones((1, 2, 1, 257)), *[np.ones((1, 2, 1, 257))] * 2),
        lambda: attention(x, x, x, scale=np.inf),
        lambda: attention(x, x, x, cap=-1.0),
        lambda: attention(x, x, x, slopes=np.ones(3)),
        lambda: attention(x, x, x, slopes=mg.tensor(np.ones(4))),  # would ask for a gradient
        lambda: attention(x, x, x, mask=AttentionMask(lengths=6)),
        lambda: attention(x, x, x, mask=AttentionMask(lengths=[1, 2, 3])),
        lambda: attention(x, x, x, mask=AttentionMask(True, prefix=[1, 2, 3])),
        lambda: attention(x, x, x, mask=AttentionMask(documents=[0, 0, 1])),
        lambda: attention(x, x, x, mask=AttentionMask(documents=np.zeros((3, 5), dtype=int))),
        lambda: AttentionMask(prefix=3),
        lambda: AttentionMask(True, prefix=3, window=2),
        lambda: AttentionMask(window=0),
        lambda: AttentionMask(lengths=-1),
        lambda: AttentionMask(lengths=[[1]]),
        lambda: AttentionMask(documents=[0, 1, 0]),
        lambda: AttentionMask(documents=3),
    ):
        with pytest.raises(ValueError):
            bad()
    for bad in (
        lambda: attention(x, x.astype(np.float64), x.astype(np.float64)),
        lambda: attention(*[np.ones((1, 2, 1, 4), dtype=np.int64)] * 3),
        lambda: attention(x, x, x, mask="causal"),
        lambda: attention(x, x, x, slopes=np.ones(4, dtype=np.int64)),
        lambda: AttentionMask(causal=1),
        lambda: AttentionMask(lengths=2.0),
        lambda: AttentionMask(window=2.0),
        lambda: AttentionMask(documents=[0.0, 1.0]),
    ):
        with pytest.raises(TypeError):
            bad()


def test_empty_attentions_need_no_device():
    for shape in ((0, 3, 2, 4), (2, 0, 2, 4)):
        q = mg.tensor(np.ones(shape))
        k = mg.tensor(np.ones((shape[0], 5, 1, 4)))
        out = attention(q, k, k)
        assert out.shape == shape and out.dtype == np.float64
        out.backward()
        assert q.grad.shape == shape and np.array_equal(k.grad, np.zeros(k.shape))


def test_head_norm_refuses_what_it_does_not_take():
    x = np.ones((2, 3, 4, 8), dtype=np.float32)
    table = RotaryTable((2, 2), 10)
    for bad in (
        lambda: head_norm(np.ones(3), eps=0.0),
        lambda: head_norm(x, np.ones(4, dtype=np.float32), eps=0.0),
        lambda: head_norm(x, eps=-1.0),
        lambda: head_norm(x, eps=np.nan),
        lambda: head_norm(np.ones((1, 1025)), eps=0.0),
        lambda: rotate(np.ones((2, 3, 4, 6)), table.at(np.zeros((3, 2), dtype=int))),  # 4 pairs in 6 values
        lambda: rotate(x, table.at(np.zeros((4, 2), dtype=int))),  # 4 positions for 3 tokens
        lambda: rotate(x, table.at(np.zeros((5, 2, 3, 2), dtype=int))),
        lambda: table.at(np.zeros((3, 1), dtype=int)),
        lambda: table.at([0, 1, 2]),
        lambda: table.at([[0, 10]]),
        lambda: table.at([[-1, 0]]),
        lambda: RotaryTable(0, 10),
        lambda: RotaryTable((), 10),
        lambda: RotaryTable((3, -1), 10),
        lambda: RotaryTable(4, 0),
        lambda: RotaryTable(4, 10, base=0.0),
    ):
        with pytest.raises(ValueError):
            bad()
    for bad in (
        lambda: head_norm(x, eps=None),
        lambda: head_norm(x, np.ones(8), eps=0.0),  # weight in another dtype
        lambda: head_norm(np.ones((2, 3), dtype=np.int32), eps=0.0),
        lambda: head_norm(x, eps=0.0, rotary=table),
        lambda: rotate(x, None),
        lambda: table.at([[0.0, 1.0]]),
        lambda: RotaryTable(4, 10, interleaved=1),
    ):
        with pytest.raises(TypeError):
            bad()
    assert head_norm(np.ones((0, 4, 8)), eps=1e-6).shape == (0, 4, 8)


def test_cache_refuses_what_it_does_not_take():
    for bad in (lambda: KeyValueCache(1, 0, 1, 8), lambda: KeyValueCache(1, 4, 1, 257)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: KeyValueCache(1, 4, 1, 8, dtype=np.int32), lambda: KeyValueCache(1, 4.0, 1, 8)):
        with pytest.raises(TypeError):
            bad()


@pytest.mark.parametrize("seed", range(20))
def test_runs_of_documents(seed):
    rng = np.random.default_rng(seed)
    sizes = rng.integers(1, 6, size=rng.integers(1, 8))
    names = rng.permutation(20)[: sizes.size] - 3  # some of them padding
    ids = np.repeat(names, sizes)[None]
    starts, ends = _runs(ids)
    for j, name in enumerate(ids[0]):
        if name < 0:
            assert starts[0, j] == ends[0, j] == 0
        else:
            where = np.flatnonzero(ids[0] == name)
            assert (starts[0, j], ends[0, j]) == (where[0], where[-1] + 1)


def test_oracle_gradients_against_differences():
    rng = np.random.default_rng(3)
    q, k, v = rng.standard_normal((2, 4, 4, 3)), rng.standard_normal((2, 5, 2, 3)), rng.standard_normal((2, 5, 2, 3))
    g = rng.standard_normal(q.shape)
    how = dict(cap=1.5, slopes=np.array([0.1, 0.2, 0.3, 0.0]), scale=0.7)
    seen = ora.visible(2, 4, 5, causal=True, prefix=2, lengths=[5, 3])
    assert not seen[1, 0].all()
    f = lambda *ops: (ora.forward(*ops, seen, lengths=[5, 3], **how)[0] * g).sum()
    for n, grad in enumerate(ora.backward(q, k, v, g, seen, lengths=[5, 3], **how)):
        for index in rng.permutation(grad.size)[:12]:
            ops = [[a.copy() for a in (q, k, v)] for _ in range(2)]
            step = 1e-6
            ops[0][n].flat[index] += step
            ops[1][n].flat[index] -= step
            # a central difference is off by step^2 of a third derivative and by rounding over the step
            assert abs((f(*ops[0]) - f(*ops[1])) / (2 * step) - grad.flat[index]) < 1e-8

    x, w, g = rng.standard_normal((3, 2, 7)), rng.standard_normal((2, 7)), rng.standard_normal((3, 2, 7))
    angle = ora.angles((1, 2), rng.integers(0, 50, (3, 2)))
    f = lambda x, w: (ora.head_norm(x, w, 1e-3, angle) * g).sum()
    dx, dw = ora.head_norm_backward(x, w, 1e-3, g, angle)
    for n, grad in enumerate((dx, dw)):
        for index in range(grad.size):
            ops = [[x.copy(), w.copy()] for _ in range(2)]
            ops[0][n].flat[index] += 1e-6
            ops[1][n].flat[index] -= 1e-6
            assert abs((f(*ops[0]) - f(*ops[1])) / 2e-6 - grad.flat[index]) < 1e-8
