"""The bars that attention's gradients are held to would not let wrong ones pass."""

import numpy as np
import pytest

from oracle import attention as ora
from tests.attention_bars import CASES, Formulas, bars_of, name_of, operands, over_keys, over_queries


def _mistaken(f):
    """(name, which result, its values) of results with a mistake."""
    out, _, dk, dv = f.results
    for name, ds in (("no D", f.p * f.dp * f.through * f.scale), ("dS halved", f.ds / 2), ("zeros", 0 * f.ds), ("nothing of the scale", f.ds / f.scale),
                     ("nothing of the cap", f.p * (f.dp - f.delta) * f.scale)):
        if (name != "nothing of the cap" or f.cap) and (name != "nothing of the scale" or f.scale != 1):
            yield name, 1, over_keys(ds, f.k)
            yield name, 2, f.shared(over_queries(ds, f.q))
    yield "zeros", 0, 0 * out
    yield "halved", 0, out / 2
    yield "zeros", 3, 0 * dv
    yield "halved", 3, dv / 2
    even = f.seen / np.maximum(f.seen.sum(-1, keepdims=True), 1)
    yield "weights of equal size", 3, f.shared(over_queries(np.broadcast_to(even[:, None], f.p.shape), f.g))
    if f.group > 1:
        yield "a shared head left out", 2, f.by_head(over_queries(f.ds, f.q))[:, :, :, 1:].sum(3)
        yield "a shared head left out", 3, f.by_head(over_queries(f.p, f.g))[:, :, :, 1:].sum(3)


@pytest.mark.parametrize("case", CASES, ids=name_of)
def test_mistaken_results_exceed_the_bars(case):
    """In one value of twenty or more of those that are not zero (a tight cap makes weights nearly even, which leaves little of D)."""
    arrays, seen, how = operands(case)
    f = Formulas(*arrays, seen, **how)
    if f.q.size * f.shape[1] < 1 << 24:  # the same by other means, where that is quick
        for a, b in zip(f.results[1:], ora.backward(*arrays, seen, **how)):
            assert np.allclose(a, b, rtol=1e-9, atol=1e-13 + 1e-11 * np.abs(b).max())
    bars = bars_of(case["dtype"], f)
    for name, which, values in _mistaken(f):
        if seen.sum(-1).max() == 1 and (which in (1, 2) or name == "weights of equal size"):  # there is no dS, and weights are even
            continue
        over = (np.abs(values - f.results[which]) > bars[which])[f.results[which] != 0]
        assert over.mean() > 0.05, (name, which, over.mean())
