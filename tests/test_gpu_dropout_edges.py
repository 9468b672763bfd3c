"""Dropout's row numbers at the ends of what a C caller can pass."""
import ctypes as C

import numpy as np
import pytest

import rgpu_b200
from rgpu_b200 import gpu as G
from tests import ref_tokens as R
from tests.test_gpu_fp8 import gpu  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


def _call(gpu, x, y, first_row):
    mask = G.DropoutMask(0.5, 1, 0, 0, None, first_row)
    status = rgpu_b200.lib().rt_dropout(gpu.handle, x.handle, None, y.handle, C.byref(mask))
    return status, rgpu_b200.lib().rt_last_error().decode()


def test_first_rows_past_the_end_are_refused_and_named(gpu):
    x, y = gpu.upload(np.ones((3, 8), np.float32)), gpu.upload(np.full((3, 8), 7.0))
    for first in (2 ** 63 - 1, 2 ** 63 - 4, 2 ** 62, 2 ** 32 + 1, 2 ** 32, 2 ** 32 - 2, -1, -2 ** 63):
        status, message = _call(gpu, x, y, first)
        assert status == G.RT_ERR_INVALID and f"3 rows from row {first} " in message, message
    assert (gpu.download(y) == 7).all()


def test_the_last_rows_are_taken(gpu):
    x, y = gpu.upload(np.ones((3, 8), np.float32)), gpu.zeros((3, 8))
    status, message = _call(gpu, x, y, 2 ** 32 - 3)
    assert status == 0, message
    kept, _ = R.keep(3, 8, 0.5, 1, first_row=2 ** 32 - 3)
    assert np.array_equal(gpu.download(y), np.where(kept, 2.0, 0.0))
