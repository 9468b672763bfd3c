"""Every 8-bit element under the smallest scales: where f32 is subnormal, and bf16 rounds."""
import numpy as np
import pytest

from tests import ref_tokens as R
from tests.test_gpu_fp8 import Held, _bf16, _upload, gpu  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pad,offset", [(0, 0), (5, 1)])
def test_smallest_scales(gpu, dtype, pad, offset):
    rows = 12  # scale bytes 0 to 11
    codes = np.tile(np.arange(256, dtype=np.uint8), (rows, 1))
    scales = np.repeat(np.arange(rows, dtype=np.uint8)[:, None], 2, 1)
    want = R.values(codes, scales, 256).astype(np.float32)
    assert want[0, 1] == 2.0 ** -136  # f32 holds all of them
    exact = want
    if dtype == "bf16":
        want = np.where(np.isnan(exact), np.nan, _bf16(np.nan_to_num(exact)))
        rounded = (want != exact) & ~np.isnan(exact)
        # four significant bits, the last one at least bf16's smallest, 2^-133, from 2^-130 on
        assert rounded.any() and np.abs(exact[rounded]).max() == 1.875 * 2.0 ** -131
    held = Held(gpu, rows, 256).set(codes, scales)
    dst, _k, view = _upload(gpu, np.zeros((rows, 256)), dtype, 256 + pad, offset)
    gpu.fp8_dequantize(held.q, dst)
    gpu.sync()
    assert np.array_equal(view.float().cpu().numpy(), want, equal_nan=True)
