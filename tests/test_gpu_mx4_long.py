"""4-bit products whose rings of stages turn over: several turns, turns that end
inside a tile, tiles that start inside a turn, and k split over a cluster in
unequal shares."""
import numpy as np
import pytest

import rgpu_b200
from tests.test_gpu_mx4 import _operand, _product_check, _upload

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def gpu():
    g = rgpu_b200.Gpu(0)
    yield g
    g.close()


def _product(gpu, m, n, k, dtype, pad, seed):
    a, av = _operand(gpu, m, k, seed)
    b, bv = _operand(gpu, n, k, seed + 1)
    bias = np.random.default_rng(n).standard_normal((1, n)).astype(np.float32) * 10
    c, buf, view = _upload(gpu, np.zeros((m, n)), dtype, n + pad, 0)
    for _ in range(2):  # the second call meets what the first one left in shared memory and TMEM
        buf.fill_(float("nan"))
        torch.cuda.synchronize()
        gpu.mx4_matmul(a.q, b.q, c, bias=gpu.upload(bias), relu=False)
        gpu.sync()
        _product_check(view.double().cpu().numpy(), av, bv, bias.astype(np.float64), False, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(2600, 2050, 2100),   # 99 tiles of pairs on 74, 9 stages each: 18 of a ring of 6
                                   (2600, 2048, 1792),   # 7 stages: a turn and one
                                   (2561, 2304, 1536),   # 6 stages: whole turns
                                   (1600, 2304, 3393),   # 63 tiles, 14 stages, the last one block of 32 and one element
                                   (4100, 3001, 1281)])  # 204 tiles, 6 stages, the last of one element
def test_pairs_of_many_stages(gpu, m, n, k, dtype):
    for pad in (-n % 16, 3):  # rows of C in 16 bytes and not
        _product(gpu, m, n, k, dtype, pad, m + k)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(7, 1000, 4352),      # 17 stages over 4: 5, 5, 5, 2
                                   (40, 700, 3300),      # 13 over 2: 7, 6
                                   (3, 520, 8200),       # 33 over 8: seven of 5 and 3
                                   (33, 300, 9216),      # 36 over 8: seven of 5 and 1
                                   (64, 900, 2305),      # 10 over 2, the last of one element
                                   (1, 128, 65569)])     # 257 over 8: seven of 33 and 26
def test_unequal_shares_of_k(gpu, m, n, k, dtype):
    for pad in (-n % 16, 3):
        _product(gpu, m, n, k, dtype, pad, m + k)
