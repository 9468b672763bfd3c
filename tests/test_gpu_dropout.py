"""Dropout on the GPU: the mask bit for bit the generator's, the values exactly rounded."""
import numpy as np
import pytest

import rgpu_b200
from rgpu_b200 import Dropout
from rgpu_b200 import gpu as G
from tests import ref_tokens as R
from tests.test_gpu_fp8 import _bf16, _upload, gpu  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

SEED = 0xFEDCBA9876543210


def _want(x, add, kept, share, dtype):
    """Each step rounded as the operator states it: the scale and the product in f32, the sum in f32, the result."""
    scale = np.float32(1.0 / share) if share else np.float32(0)
    y = np.where(kept, (x.astype(np.float32) * scale).astype(np.float32), np.float32(0))
    if add is not None:
        y = (add + y).astype(np.float32)
    return _bf16(y) if dtype == "bf16" else y


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7), (2, 8), (3, 9), (5, 255), (7, 256), (33, 257), (40, 513), (129, 100),
                                       (130, 520), (300, 33), (3, 1100)])
def test_values(gpu, rows, cols, dtype):
    rng = np.random.default_rng(rows * 31 + cols)
    x, add = (rng.standard_normal((rows, cols)).astype(np.float32) for _ in range(2))
    if dtype == "bf16":
        x, add = _bf16(x), _bf16(add)
    for n, (pad, offset, p, where) in enumerate(((0, 0, 0.1, {}), (3, 1, 0.5, dict(site=7, step=123)),
                                                 (-cols % 16, 8, 0.25, dict(site=2 ** 32 - 1, step=5, first_row=2 ** 32 - rows)),
                                                 (8 - cols % 8, 0, 0.9, dict(first_row=1000)))):
        kept, share = R.keep(rows, cols, p, SEED + n, **where)
        mask = Dropout(p, SEED + n, **where)
        tx, _k, vx = _upload(gpu, x, dtype, cols + pad, offset)
        ta, _k2, _ = _upload(gpu, add, dtype, cols + pad, offset)
        for with_add in (False, True):
            y, buf, view = _upload(gpu, np.zeros((rows, cols)), dtype, cols + pad, offset)
            before = buf.clone()
            gpu.dropout(tx, y, mask, add=ta if with_add else None)
            gpu.sync()
            assert np.array_equal(view.float().cpu().numpy(), _want(x, add if with_add else None, kept, share, dtype))
            view.copy_(before[offset:offset + rows * (cols + pad)].view(rows, cols + pad)[:, :cols])
            assert torch.equal(buf.isnan(), before.isnan()), "elements beside y were written"
        gpu.dropout(tx, tx, mask)  # in place
        gpu.sync()
        assert np.array_equal(vx.float().cpu().numpy(), _want(x, None, kept, share, dtype))


def test_in_place_on_the_sum(gpu):
    rng = np.random.default_rng(1)
    x, r = (_bf16(rng.standard_normal((70, 333)).astype(np.float32)) for _ in range(2))
    kept, share = R.keep(70, 333, 0.2, 5)
    for pad, offset in ((3, 0), (0, 1)):
        tx, _k, _ = _upload(gpu, x, "bf16", 333 + pad, offset)
        tr, _k2, view = _upload(gpu, r, "bf16", 333 + pad, offset)
        gpu.dropout(tx, tr, Dropout(0.2, 5), add=tr)
        gpu.sync()
        assert np.array_equal(view.float().cpu().numpy(), _want(x, r, kept, share, "bf16"))


def test_nothing_and_everything(gpu):
    x = gpu.upload(np.full((9, 50), 2.0))
    y = gpu.upload(np.full((9, 50), 9.0))
    gpu.dropout(x, y, Dropout(0.0, 1))
    assert (gpu.download(y) == 2).all()
    gpu.dropout(x, y, Dropout(1.0, 1))
    assert (gpu.download(y) == 0).all()
    gpu.dropout(x, y, Dropout(1.0, 1), add=x)
    assert (gpu.download(y) == 2).all()


def test_dropped_infinities_and_nan_do_not_come_through(gpu):
    kept, share = R.keep(20, 64, 0.5, 3)
    for bad in (np.inf, np.nan, -np.inf):
        x = np.where(kept, 1.0, bad)
        y = gpu.zeros((20, 64))
        gpu.dropout(gpu.upload(x), y, Dropout(0.5, 3))
        assert np.array_equal(gpu.download(y), np.where(kept, 2.0, 0.0))
        gpu.dropout(gpu.upload(np.where(kept, bad, 1.0)), y, Dropout(0.5, 3))
        assert np.array_equal(gpu.download(y), np.where(kept, bad, 0.0), equal_nan=True)


def test_a_row_has_its_mask_in_any_batch(gpu):
    # the rows of a batch alone, split over two calls, in another type and stride
    x = gpu.upload(np.ones((40, 300)))
    whole = gpu.zeros((40, 300))
    gpu.dropout(x, whole, Dropout(0.3, 11, first_row=7))
    want = gpu.download(whole) != 0
    part = gpu.zeros((15, 300), "bf16")
    gpu.dropout(gpu.upload(np.ones((15, 300)), "bf16"), part, Dropout(0.3, 11, first_row=7 + 25))
    assert np.array_equal(gpu.download(part) != 0, want[25:])


def test_gradient_is_the_same_call(gpu):
    # linear in x: <c, f(w)> = <f'(c), w> whatever the mask
    rng = np.random.default_rng(3)
    w, c = (rng.integers(-8, 9, (33, 200)).astype(np.float32) for _ in range(2))
    y, dx = gpu.zeros((33, 200)), gpu.zeros((33, 200))
    mask = Dropout(0.5, 77, site=1, step=2)
    gpu.dropout(gpu.upload(w), y, mask)
    gpu.dropout(gpu.upload(c), dx, mask)
    assert (gpu.download(y).astype(np.float64) * c).sum() == (gpu.download(dx).astype(np.float64) * w).sum()  # whole numbers


def test_steps_on_the_device_in_a_captured_graph(gpu):
    step = torch.zeros(1, dtype=torch.int32, device="cuda")
    x, y = gpu.upload(np.ones((8, 64))), gpu.zeros((8, 64))
    at = gpu.wrap(step.data_ptr(), (1,), "u32")
    gpu.sync()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    gpu.set_stream(stream.cuda_stream)
    try:
        with torch.cuda.graph(graph, stream=stream):
            gpu.dropout(x, y, Dropout(0.5, 1, step=10, step_at=at))
    finally:
        gpu.set_stream(None)
    seen = []
    for i in (0, 1, 5, -10):
        step.fill_(i)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        seen.append(gpu.download(y) != 0)
        assert np.array_equal(seen[-1], R.keep(8, 64, 0.5, 1, step=10 + i)[0])
    assert not np.array_equal(seen[0], seen[1])


def test_empty_extents(gpu):
    gpu.dropout(gpu.zeros((0, 8)), gpu.zeros((0, 8)), Dropout(0.5, 1, first_row=2 ** 32))
    gpu.dropout(gpu.zeros((8, 0)), gpu.zeros((8, 0)), Dropout(0.5, 1))
    gpu.sync()


def test_refusals(gpu):
    x, y = gpu.zeros((4, 8)), gpu.zeros((4, 8))
    m = Dropout(0.5, 1)

    def refused(call, word):
        with pytest.raises(rgpu_b200.RtError) as e:
            call()
        assert e.value.code == G.RT_ERR_INVALID and word in str(e.value), str(e.value)

    refused(lambda: gpu.dropout(x, gpu.zeros((4, 9)), m), "y 4x9")
    refused(lambda: gpu.dropout(x, y, m, add=gpu.zeros((3, 8))), "add 3x8")
    refused(lambda: gpu.dropout(x, gpu.zeros((4, 8), "bf16"), m), "one type")
    refused(lambda: gpu.dropout(gpu.zeros((4, 8), "u32"), gpu.zeros((4, 8), "u32"), m), "f32 or bf16")
    refused(lambda: gpu.dropout(x, y, Dropout(-0.1, 1)), "in [0, 1]")
    refused(lambda: gpu.dropout(x, y, Dropout(float("nan"), 1)), "in [0, 1]")
    refused(lambda: gpu.dropout(x, y, Dropout(0.5, 1, first_row=2 ** 32 - 3)), "2^32")
    refused(lambda: gpu.dropout(x, y, Dropout(0.5, 1, step_at=gpu.zeros((1,)))), "one u32")
    refused(lambda: gpu.dropout(x, y, Dropout(0.5, 1, step_at=gpu.zeros((2,), "u32"))), "one u32")
    other = rgpu_b200.Gpu(0)
    refused(lambda: gpu.dropout(x, other.zeros((4, 8)), m), "another context")
    gone = gpu.zeros((1,), "u32")
    m = Dropout(0.5, 1, step_at=gone)
    gone.free()
    refused(lambda: gpu.dropout(x, y, m), "after free")
