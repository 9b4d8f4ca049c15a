"""Tensors of more than 2^31 values: what lies behind that many is read and written where it is.  Through the C entry points, on memory that
is filled on the device and looked at in part."""

import ctypes

import numpy as np
import pytest

import mygrad_amd as mg
from mygrad_amd import _device, _hip
from oracle import language as ora

pytestmark = pytest.mark.gpu

F16 = 2


@pytest.fixture(scope="module", autouse=True)
def device():
    if not mg.is_available():
        pytest.fail("libmygrad_hip.so / gfx950 device not available: the GPU tests need both")


class Far:
    """``count`` values of float16 on the device, zeros but where they are put."""

    def __init__(self, count, fill=True):
        self.buf = _device.DeviceBuffer(2 * count)
        self.ptr = self.buf.ptr
        if fill:
            _hip.check(_hip.lib().mg_memset_zero(self.ptr, 2 * count))

    def put(self, at, values):
        values = np.ascontiguousarray(values, np.float16)
        _hip.check(_hip.lib().mg_memcpy_h2d(self.ptr + 2 * at, values.ctypes.data, values.nbytes))

    def get(self, at, count):
        out = np.empty(count, np.float16)
        _hip.check(_hip.lib().mg_memcpy_d2h(out.ctypes.data_as(ctypes.c_void_p), self.ptr + 2 * at, out.nbytes))
        return out


def test_a_table_of_more_than_two_to_the_31_values():
    rng, rows, dim = np.random.default_rng(0), 70001, 32768
    table, dtable = Far(rows * dim), Far(rows * dim, fill=False)
    ids = np.array([70000, 3, -1, 70000, 65537], np.int32)
    values, g = rng.standard_normal((3, dim)).astype(np.float16), rng.standard_normal((5, dim)).astype(np.float16)
    for row, value in zip((70000, 3, 65537), values):
        table.put(row * dim, value)
    out, grad, held = Far(5 * dim), Far(5 * dim), _device.from_host(ids).buf
    grad.put(0, g)
    lib = _hip.lib()
    _hip.check(lib.mg_embedding_fwd(F16, 5, rows, dim, 1.0, held.ptr, table.ptr, out.ptr))
    _hip.check(lib.mg_embedding_bwd(F16, 5, rows, dim, 1.0, held.ptr, grad.ptr, dtable.ptr))
    assert np.array_equal(out.get(0, 5 * dim).reshape(5, dim), np.stack((values[0], values[1], np.zeros(dim), values[0], values[2])))
    assert np.array_equal(dtable.get(70000 * dim, dim), (g[0].astype(np.float32) + g[3]).astype(np.float16))
    assert np.array_equal(dtable.get(3 * dim, dim), g[1]) and np.array_equal(dtable.get(65537 * dim, dim), g[4])
    for row in (0, 2, 4, 65536, 65538, 69999):
        assert not dtable.get(row * dim, dim).any()


def test_rows_of_layer_norm_behind_two_to_the_31_values():
    rng = np.random.default_rng(1)
    for rows, dim in ((70001, 32768), (2200, 1000001)):  # in registers, and not
        x, g, y, dx = Far(rows * dim), Far(rows * dim), Far(rows * dim, fill=False), Far(rows * dim, fill=False)
        w, b, dw, db = (Far(dim) for _ in range(4))
        kept = _device.DeviceBuffer(12 * rows)
        given = {rows - 1: rng.standard_normal((2, dim)).astype(np.float16), 5: rng.standard_normal((2, dim)).astype(np.float16)}
        weight = (1 + 0.1 * rng.standard_normal(dim)).astype(np.float16)
        w.put(0, weight)
        for row, (values, grads) in given.items():
            x.put(row * dim, values)
            g.put(row * dim, grads)
        lib = _hip.lib()
        _hip.check(lib.mg_layer_norm_fwd(F16, rows, dim, 1e-5, x.ptr, w.ptr, b.ptr, y.ptr, kept.ptr))
        _hip.check(lib.mg_layer_norm_bwd(F16, rows, dim, x.ptr, w.ptr, kept.ptr, g.ptr, dx.ptr, dw.ptr, db.ptr))
        sums = []
        for row, (values, grads) in given.items():
            want = ora.layer_norm(values[None], weight, None, 1e-5, grads[None])
            # half a unit of the result, and what single precision loses on rows of a million values (an eighth of a unit of float16 at most)
            assert np.abs(y.get(row * dim, dim) - want[0][0]).max() <= 2.0**-10 * np.abs(want[0]).max()
            assert np.abs(dx.get(row * dim, dim) - want[1][0]).max() <= 2.0**-10 * np.abs(want[1]).max()
            sums.append(want[2:])
        assert np.abs(dw.get(0, dim) - (sums[0][0] + sums[1][0])).max() <= 2.0**-9 * np.abs(sums[0][0] + sums[1][0]).max()
        assert np.abs(db.get(0, dim) - (sums[0][1] + sums[1][1])).max() <= 2.0**-9 * np.abs(sums[0][1] + sums[1][1]).max()
        for row in (0, rows // 2, rows - 2):
            assert not y.get(row * dim, dim).any() and not dx.get(row * dim, dim).any()


def test_logits_behind_two_to_the_31():
    rng, lib = np.random.default_rng(2), _hip.lib()
    for rows, vocabulary in ((9, (1 << 28) + 5), (1 << 16, 40001)):  # parts of rows, and a block each
        z, dz = Far(rows * vocabulary), Far(rows * vocabulary, fill=False)
        ids = np.full(rows, vocabulary - 2, np.int32)
        near = rng.standard_normal(1000).astype(np.float16) + np.float16(20)  # at the last row's end, far above the zeros
        z.put(rows * vocabulary - 1000, near)
        held, ones = _device.from_host(ids).buf, _device.from_host(np.ones(rows, np.float32)).buf
        out, entropy, kept, top, which = (_device.DeviceBuffer(12 * rows * 4) for _ in range(5))
        _hip.check(lib.mg_log_probabilities_fwd(F16, rows, vocabulary, 4, held.ptr, z.ptr, out.ptr, entropy.ptr, kept.ptr, top.ptr, which.ptr))
        _hip.check(lib.mg_log_probabilities_bwd(F16, rows, vocabulary, held.ptr, z.ptr, kept.ptr, ones.ptr, None, dz.ptr))
        scores, found = np.empty(rows, np.float32), np.empty((rows, 4), np.int32)
        out.download_into(scores)
        which.download_into(found)
        row = near.astype(np.float64)
        total = np.exp(row).sum() + (vocabulary - 1000)
        assert np.abs(scores[:-1] + np.log(vocabulary)).max() < 1e-5 and abs(scores[-1] - (row[-2] - np.log(total))) < 1e-5
        assert np.array_equal(found[-1], vocabulary - 1000 + np.argsort(-row, kind="stable")[:4]) and (found[:-1] == np.arange(4)).all()
        want = -np.exp(row) / total
        want[-2] += 1
        assert np.abs(dz.get(rows * vocabulary - 1000, 1000) - want).max() <= 2.0**-11
        assert abs(dz.get((rows - 1) * vocabulary - 2, 1)[0] - 1) <= 2.0**-11 and np.abs(dz.get((rows - 1) * vocabulary, 1000)).max() <= 2.0**-13
        lists, teacher = np.tile(np.array([vocabulary - 2, vocabulary - 1000], np.int32), (rows, 1)), np.zeros((rows, 2), np.float16)
        lists, teacher = _device.from_host(lists).buf, _device.from_host(teacher).buf
        _hip.check(lib.mg_distillation_fwd(F16, F16, rows, vocabulary, 2, 1.0, z.ptr, lists.ptr, teacher.ptr, out.ptr, kept.ptr, entropy.ptr))
        _hip.check(lib.mg_distillation_bwd(F16, rows, vocabulary, 2, 1.0, z.ptr, lists.ptr, kept.ptr, entropy.ptr, ones.ptr, dz.ptr))
        out.download_into(scores)
        assert abs(scores[-1] - (np.log(0.5) - 0.5 * (row[0] + row[-2]) + np.log(total))) < 1e-5
        want = np.exp(row) / total
        want[0] -= 0.5
        want[-2] -= 0.5
        assert np.abs(dz.get(rows * vocabulary - 1000, 1000) - want).max() <= 2.0**-11
