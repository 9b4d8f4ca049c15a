"""What attention and the norm of heads check and hold on the host."""

import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

from mygrad_amd.nnet import attention


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("how", [dict(cap=1e-50), dict(cap=1e-31), dict(cap=1e39), dict(scale=1e39), dict(scale=-1e39), dict(scale=1e31, cap=1.0)])
def test_scales_and_caps_beyond_single_precision_are_refused(dtype, how):
    """A cap that rounds to zero there was no cap, and an infinite scale gave no numbers."""
    x = np.ones((1, 3, 2, 8), dtype=dtype)
    with pytest.raises(ValueError, match="single precision"):
        attention(x, x, x, **how)


def test_rows_of_the_largest_window_see_no_fewer_keys_than_a_small_one_lets(tmp_path):
    """The estimate of a tile's work, by which packed documents are sorted: 2 * 2**30 keys both ways are no negative number."""
    if not shutil.which("hipcc"):
        pytest.skip("needs hipcc")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    source, library = tmp_path / "window.hip", tmp_path / "window.so"
    source.write_text('#include "attention_device.h"\nextern "C" unsigned estimate(int window, int causal, int rows) { return mg::window_of_rows(window, causal, rows); }\n')
    subprocess.run(["hipcc", "--offload-arch=gfx950", "-shared", "-fPIC", "-std=c++17", f"-I{root}/include", f"-I{root}/mygrad_amd/csrc", str(source), "-o", str(library)],
                   check=True, capture_output=True)
    estimate = ctypes.CDLL(str(library)).estimate
    estimate.restype = ctypes.c_uint
    for causal, each in ((1, 1), (0, 2)):
        for window in (1, 100, 1 << 29, 1 << 30):
            assert estimate(window, causal, 128) == each * window + 128
