"""Products with few columns: what an earlier launch left in shared memory does not
reach the result, whatever the depth."""
import numpy as np
import pytest

import rgpu_b200

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    g = rgpu_b200.Gpu(0)
    yield g
    g.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("layout", ["nn", "nt"])
@pytest.mark.parametrize("k", [72, 33, 95, 200])
def test_depths_that_are_no_multiple_of_32(gpu, k, layout, dtype):
    m, n = 8192, 5
    rng = np.random.default_rng(k)
    deep = (k + 31) // 32 * 32
    product = gpu.matmul if layout == "nn" else gpu.matmul_a_bt
    c = gpu.zeros((m, n))
    a = rng.standard_normal((m, k)).astype(np.float32)
    b = rng.standard_normal((k, n)).astype(np.float32)
    if dtype == "bf16":  # as the device holds them
        a, b = (gpu.download(gpu.upload(x, "bf16")) for x in (a, b))
    nan = np.full((deep, n), np.nan, np.float32)
    one, two = gpu.upload(np.ones((m, deep), np.float32), dtype), gpu.upload(a, dtype)
    b1, b2 = (gpu.upload(x if layout == "nn" else np.ascontiguousarray(x.T), dtype) for x in (nan, b))
    product(one, b1, c)
    product(two, b2, c)
    got, want = gpu.download(c).astype(np.float64), a.astype(np.float64) @ b
    # k products and sums in f32
    assert (np.abs(got - want) <= (k + 1) * 2.0**-24 * (np.abs(a).astype(np.float64) @ np.abs(b))).all()
