"""One block of attention, trained on packed documents and then run a token at a time.

Queries, keys and values are projections of the tokens (``einsum``); queries and keys are normed for each head and turned by
their positions in one pass (``head_norm``); ``attention`` joins them.  Training packs documents of different lengths into one
row of tokens, which ``AttentionMask`` keeps apart.  Generation feeds each result back as the next token: ``KeyValueCache``
holds the keys and values of what came before, so that a step computes one token only.

The task: tokens are vectors (the first value 4) that come again after ``PERIOD`` places, the block is to give the next one.

    python examples/attention_block.py [--steps 200]
"""

import argparse
import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import mygrad_amd as mg  # noqa: E402
from mygrad_amd.nnet import AttentionMask, KeyValueCache, RotaryTable, attention, head_norm  # noqa: E402

PERIOD = 4


class Block:
    def __init__(self, width=16, heads=4, kv_heads=2, dim=32, longest=256, dtype=np.float32, seed=0):
        rng = np.random.default_rng(seed)
        make = lambda fan_in, *shape: mg.device_tensor((rng.standard_normal(shape) * fan_in**-0.5).astype(dtype))
        self.dtype, self.kv_heads, self.dim = dtype, kv_heads, dim
        self.weights = {
            "q": make(width, width, heads, dim), "k": make(width, width, kv_heads, dim), "v": make(width, width, kv_heads, dim),
            "out": make(heads * dim, heads, dim, width),
            "q_norm": mg.device_tensor(np.full(dim, 4.0, dtype)), "k_norm": mg.device_tensor(np.full(dim, 1.0, dtype)),
        }
        self.table = RotaryTable(dim // 2, longest, base=100.0)

    def _heads(self, x, rotary):
        w = self.weights
        q, k, v = (mg.einsum("btc,chd->bthd", x, w[name]) for name in "qkv")
        return head_norm(q, w["q_norm"], eps=1e-6, rotary=rotary), head_norm(k, w["k_norm"], eps=1e-6, rotary=rotary), v

    def __call__(self, x, rotary, mask):
        """All tokens ``x:(batch, tokens, width)`` at once."""
        return mg.einsum("bthd,hdc->btc", attention(*self._heads(x, rotary), mask=mask), self.weights["out"])

    def step(self, x, cache, length):
        """The last tokens of a row of ``length`` that ends with them; the cache holds those before."""
        tokens = x.shape[1]
        with mg.no_autodiff:
            mask = AttentionMask(causal=True, lengths=length)
            q, k, v = self._heads(x, self.table.at(np.arange(length - tokens, length)))
            cache.write(k, v, mask)
            return mg.einsum("bthd,hdc->btc", cache.attend(q, mask=mask), self.weights["out"])

    def cache(self, batch, capacity):
        return KeyValueCache(batch, capacity, self.kv_heads, self.dim, dtype=self.dtype)


def documents(rng, lengths, width):
    """Tokens of some documents in a row, the tokens to come, each token's document and its place in it; a document's last
    ``PERIOD`` tokens are the first ones again."""
    rows = [np.resize(rng.standard_normal((PERIOD, width)), (n + 1, width)) for n in lengths]
    for row in rows:
        row[:, 0] = 4  # what is the same in all tokens lets a query ask for a distance
    x, y = np.concatenate([r[:-1] for r in rows]), np.concatenate([r[1:] for r in rows])
    return x[None], y[None], np.repeat(np.arange(len(lengths)), lengths), np.concatenate([np.arange(n) for n in lengths])


def train(block, steps, lengths=(60, 17, 100, 33, 90, 70), width=16, rate=0.01, seed=1, report=None):
    """Adam, its moments on the host; the losses of all steps."""
    rng, losses = np.random.default_rng(seed), []
    moments = {name: [np.zeros(w.shape), np.zeros(w.shape)] for name, w in block.weights.items()}
    _, _, ids, places = documents(rng, lengths, width)
    mask, rotary = AttentionMask(causal=True, documents=ids), block.table.at(places)  # for all steps
    told = places >= PERIOD - 1  # what comes next cannot be known before
    for n in range(1, steps + 1):
        x, y, _, _ = documents(rng, lengths, width)
        out = block(mg.device_tensor(x.astype(block.dtype), constant=True), rotary, mask)
        off = (out.data.astype(np.float64) - y) * told[:, None]
        losses.append(float((off**2).sum() / (told.sum() * width)))
        out.backward(off.astype(block.dtype))
        for name, w in block.weights.items():
            first, second = moments[name]
            grad = w.grad.astype(np.float64)
            first += 0.1 * (grad - first)
            second += 0.05 * (grad**2 - second)
            change = rate * first / (1 - 0.9**n) / (np.sqrt(second / (1 - 0.95**n)) + 1e-9)
            block.weights[name] = mg.device_tensor((w.data - change).astype(block.dtype))
        if report and n % 20 == 0:
            report(f"step {n}: loss {losses[-1]:.4f}")
    return losses


def generate(block, prompt, tokens):
    """``prompt:(batch, tokens, width)`` and as many tokens more, each the block's own last result."""
    batch, length, _ = prompt.shape
    cache = block.cache(batch, length + tokens)
    row = [np.asarray(prompt, dtype=block.dtype)]
    for _ in range(tokens):
        row.append(block.step(row[-1], cache, length).data[:, -1:])
        length += 1
    return np.concatenate(row, axis=1)


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--steps", type=int, default=200)
    args = parser.parse_args()
    block = Block()
    train(block, args.steps, report=print)
    prompt, _, _, _ = documents(np.random.default_rng(7), (2 * PERIOD,), 16)
    row = generate(block, prompt, 24)
    want = np.resize(prompt[0, :PERIOD], row.shape[1:])
    print(f"24 tokens after {2 * PERIOD}: off by {np.sqrt(((row[0] - want) ** 2).mean()):.4f} (tokens are 1 in size)")


if __name__ == "__main__":
    main()
