"""What attention and the norm of heads check and hold on the host."""

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
