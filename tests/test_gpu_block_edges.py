"""The residual-block norms at their edges."""
import numpy as np
import pytest

import rgpu_b200

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    g = rgpu_b200.Gpu(0)
    yield g
    g.close()


@pytest.mark.parametrize("shape", [(1, 1), (3, 1)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradient_of_a_gate_over_no_columns_is_zero(gpu, dtype, shape):
    e = gpu.zeros((3, 0), dtype)
    gate, dgate = gpu.upload(np.ones(shape, np.float32)), gpu.upload(np.full(shape, 9.0, np.float32))
    work = gpu.zeros((max(1, gpu.block_backward_workspace(3, 0)),))
    gpu.block_backward(e, y=e, gate=gate, dz=e, dr=gpu.zeros((3, 0), dtype), dy=gpu.zeros((3, 0), dtype), dgate=dgate, work=work)
    assert not gpu.download(dgate).any()
