"""The block of attention in ``examples/``: what its parts give together."""

import importlib.util
from pathlib import Path

import numpy as np
import pytest

import mygrad_amd as mg
from mygrad_amd.nnet import AttentionMask
from oracle import attention as ora

pytestmark = pytest.mark.gpu

spec = importlib.util.spec_from_file_location("attention_block", Path(__file__).resolve().parents[1] / "examples" / "attention_block.py")
example = importlib.util.module_from_spec(spec)
spec.loader.exec_module(example)

UNIT = {np.float32: 2.0**-24, np.float64: 2.0**-53}


@pytest.fixture(scope="module", autouse=True)
def device():
    if not mg.is_available():
        pytest.fail("libmygrad_hip.so / gfx950 device not available: the GPU tests need both")


def _bar(block, x):
    """How far two ways to a result may be apart: projections sum `width` products, scores `dim` of them, the results `heads dim`.  A score
    is at most sqrt(dim) times the gains' product, the weights are off by twice its error, and each stage adds its rounding."""
    u = UNIT[block.dtype]
    w = {name: np.abs(t.data.astype(np.float64)).max() for name, t in block.weights.items()}
    width, (heads, dim) = x.shape[-1], block.weights["q"].shape[1:]
    score = dim**0.5 * w["q_norm"] * w["k_norm"]
    steps = (width + 2 * dim + x.shape[1] + 68) * u  # of a projection, a norm, a turn, a score
    value = np.abs(np.einsum("btc,chd->bthd", x.astype(np.float64), block.weights["v"].data.astype(np.float64))).max()
    out = np.sqrt(heads * dim) * value * np.linalg.norm(block.weights["out"].data.astype(np.float64).reshape(-1, width), axis=0).max()
    return 2 * out * ((2 * score + 1) * steps + (heads * dim + 2) * u)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("pieces", [[1] * 9, [40, 1, 1, 1], [5, 3, 30, 8, 1]])
def test_a_token_at_a_time_gives_what_all_at_once_give(dtype, pieces):
    block = example.Block(dtype=dtype)
    length = sum(pieces)
    x = np.random.default_rng(length).standard_normal((3, length, 16)).astype(dtype)
    whole = block(mg.device_tensor(x, constant=True), block.table.at(np.arange(length)), AttentionMask(causal=True)).data
    cache, at, parts = block.cache(3, length + 5), 0, []
    for n in pieces:
        at += n
        parts.append(block.step(x[:, at - n:at], cache, at).data)
    assert np.abs(np.concatenate(parts, axis=1).astype(np.float64) - whole).max() <= _bar(block, x)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_documents_in_a_row_are_as_if_alone(dtype):
    block = example.Block(dtype=dtype)
    x, _, ids, places = example.documents(np.random.default_rng(4), (20, 1, 70, 9), 16)
    x = x.astype(dtype)
    packed = block(mg.device_tensor(x, constant=True), block.table.at(places), AttentionMask(causal=True, documents=ids)).data
    for n in range(4):
        alone = np.ascontiguousarray(x[:, ids == n])
        got = block(mg.device_tensor(alone, constant=True), block.table.at(np.arange(alone.shape[1])), AttentionMask(causal=True)).data
        assert np.abs(packed[:, ids == n].astype(np.float64) - got).max() <= _bar(block, x)


def test_gradients_of_the_block():
    """All weights' gradients against the formulas in 64 bits, in float64."""
    block = example.Block(width=24, heads=4, kv_heads=2, dim=8, dtype=np.float64)
    rng = np.random.default_rng(2)
    x, _, ids, places = example.documents(rng, (9, 14), 24)
    g = rng.standard_normal(x.shape)
    rotary = block.table.at(places)
    block(mg.device_tensor(x, constant=True), rotary, AttentionMask(causal=True, documents=ids)).backward(g)
    w = {name: t.data for name, t in block.weights.items()}
    turns, axis_of = block.table._turns[places], np.zeros(4, dtype=int)

    def loss(w):
        heads = [np.einsum("btc,chd->bthd", x, w[name]) for name in "qkv"]
        turned = []
        for a, gain in zip(heads, (w["q_norm"], w["k_norm"])):
            a = gain * a / np.sqrt((a**2).mean(-1, keepdims=True) + 1e-6)
            c, s = turns[None, :, None, :, 0], turns[None, :, None, :, 1]
            turned.append(np.concatenate([a[..., :4] * c - a[..., 4:] * s, a[..., 4:] * c + a[..., :4] * s], -1))
        out, _, _ = ora.forward(*turned, heads[2], ora.visible(1, 23, 23, causal=True, documents=ids))
        return (np.einsum("bthd,hdc->btc", out, w["out"]) * g).sum()

    for name, tensor in block.weights.items():
        way = rng.standard_normal(tensor.shape)
        up, down = ({**w, name: w[name] + by * way} for by in (1e-6, -1e-6))
        # rounding of the loss (a sum of 552 terms of some size 1) over the step, and the third derivative times its square
        assert abs((loss(up) - loss(down)) / 2e-6 - (tensor.grad * way).sum()) < 1e-6 * max(1.0, np.abs(tensor.grad * way).sum())


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_it_learns(dtype):
    block = example.Block(dtype=dtype)
    losses = example.train(block, 40)
    assert np.isfinite(losses).all() and np.mean(losses[-5:]) < 0.7 * np.mean(losses[:5])
