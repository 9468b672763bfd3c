"""An allocation that the device has no room for is refused, and the next calls do
not hear of it."""
import numpy as np
import pytest

import rgpu_b200
from rgpu_b200 import gpu as G

pytestmark = pytest.mark.gpu

LARGEST = (1 << 31) - 257


@pytest.mark.parametrize("too_large", [lambda g: g.mx4_zeros(LARGEST, LARGEST), lambda g: g.zeros((1 << 20, 1 << 24))],
                         ids=["mx4", "tensor"])
def test_a_refused_allocation_leaves_no_error_behind(too_large):
    gpu = rgpu_b200.Gpu(0)
    x, y = gpu.upload(np.array([[-1.0, 2.0]], np.float32)), gpu.zeros((1, 2))
    with pytest.raises(rgpu_b200.RtError) as e:
        too_large(gpu)
    assert e.value.code == G.RT_ERR_OOM
    gpu.relu(x, y)
    gpu.mx4_quantize(x)
    assert np.array_equal(gpu.download(y), [[0.0, 2.0]])
    gpu.close()
