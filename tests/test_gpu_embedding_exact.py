"""The embedding's gradient of whole numbers, whose sums below 2^24 are exact in f32: a row that
is lost or added twice shows, however often its token occurs. Of other numbers within the bound of the
tree that the sums make."""
import numpy as np
import pytest

import rgpu_b200
from tests.test_gpu_embedding import BACK, U, _tokens
from tests.test_gpu_fp8 import _upload, gpu  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def _whole(count, n, seed=0):
    """Rows of whole numbers from 1 to 47 that differ from those of neighbouring positions; at most 300000 of them sum to less than 2^24."""
    i, j = np.arange(count, dtype=np.int64)[:, None], np.arange(n)[None]
    return ((i * 31 + i // 47 * 5 + j * 17 + seed) % 47 + 1).astype(np.float32)


def _sums(vocabulary, tokens, dy):
    d = np.zeros((vocabulary, dy.shape[1]))
    real = tokens < vocabulary
    order = np.argsort(tokens[real], kind="stable")
    t = tokens[real][order]
    if len(t):
        first = np.flatnonzero(np.r_[True, t[1:] != t[:-1]])
        d[t[first]] = np.add.reduceat(dy[real][order].astype(np.float64), first, axis=0)
    return d


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind,count,n,vocabulary", BACK + [("one", 300000, 36, 5), ("one", 70000, 260, 2), ("runs", 65536, 20, 9),
                                                            ("zipf", 65536, 520, 9000), ("uniform", 9000, 1024, 20000)])
def test_whole_numbers_are_exact(gpu, kind, count, n, vocabulary, dtype):
    tokens = _tokens(kind, np.random.default_rng(count * 5 + n), count, vocabulary).astype(np.uint32)
    dy = _whole(count, n)
    want = _sums(vocabulary, tokens, dy)
    assert want.max(initial=0) < 2 ** 24
    t, words = rgpu_b200.upload_labels(gpu, tokens), gpu.embedding_backward_workspace(count, vocabulary, n)
    for pad, offset in ((0, 0), (3, 1)):
        work = torch.full((words,), float("nan"), device="cuda")
        tdy, _k, _ = _upload(gpu, dy, dtype, n + pad, offset)
        out, _k2, view = _upload(gpu, np.full((vocabulary, n), 7.0), "f32", n + pad, offset)
        w = gpu.wrap(work.data_ptr(), (words,))
        gpu.embedding_backward(t, tdy, out, w, scale=0.5)
        gpu.sync()
        assert torch.equal(view, torch.from_numpy(want * 0.5).float().cuda())
        gpu.embedding_backward(t, tdy, out, w, scale=0.25, accumulate=True)
        gpu.sync()
        assert torch.equal(view, torch.from_numpy(want * 0.75).float().cuda())


def _depth(count, times, n):
    """Additions on the longest way of a row of dy into the sum of its token, and those after: the tree that the operator's
    pieces, warps' shares and joins make, by its own sizes or ones that are no smaller."""
    cut = 64
    while cut > 16 and (count // cut) * -(-n // 256) < 8 * 148:
        cut //= 2
    pieces = times // cut + 2
    # a piece, or a light row; then one warp's or eight warps' partial sums
    long = np.minimum(times, cut) + np.where(times > cut, np.maximum(18, -(-pieces // 8) + 8), 0)
    # in one launch: a warp's equal share of the CTA's positions, and the others' joined to it
    few = np.minimum(times, -(-count // 8)) + 16
    return (np.maximum(long, few) if count <= 8192 else long) + 2  # the scale, the sum with what was there


@pytest.mark.parametrize("kind,count,n,vocabulary", [("one", 65537, 12, 100), ("zipf", 65536, 40, 3000), ("zipf", 300000, 8, 50257),
                                                     ("one", 5000, 264, 3), ("zipf", 9000, 260, 1500)])
def test_rounding(gpu, kind, count, n, vocabulary):
    # each addition is off by at most half a step of its result, which is at most the sum of magnitudes below it (and its
    # own roundings, of second order: 1.01)
    rng = np.random.default_rng(count + n)
    tokens = _tokens(kind, rng, count, vocabulary).astype(np.uint32)
    dy = rng.standard_normal((count, n)).astype(np.float32)
    want, size = _sums(vocabulary, tokens, dy), _sums(vocabulary, tokens, np.abs(dy))
    times = np.bincount(tokens[tokens < vocabulary], minlength=vocabulary)
    d = gpu.zeros((vocabulary, n))
    gpu.embedding_backward(rgpu_b200.upload_labels(gpu, tokens), gpu.upload(dy), d,
                           gpu.zeros((gpu.embedding_backward_workspace(count, vocabulary, n),)), scale=1.5)
    bound = 1.01 * U * _depth(count, times, n)[:, None] * 1.5 * size
    assert np.all(np.abs(gpu.download(d) - 1.5 * want) <= bound)


@pytest.mark.parametrize("pad,offset", [(0, 0), (4, 4), (3, 1)])
@pytest.mark.parametrize("count,n,vocabulary", [(4200, 16500, 255), (9000, 16500, 255), (9000, 1024, 20000), (5000, 1021, 9000), (40000, 48, 90000),
                                                (4500, 8, 600000), (70000, 256, 20000)])
def test_large_tables(gpu, count, n, vocabulary, pad, offset):
    # absent rows get their zeros beside the sort or beside the pieces, by the table's size: every row is written, once
    rng = np.random.default_rng(count + n)
    tokens = torch.from_numpy(_tokens("zipf", rng, count, vocabulary).astype(np.int64)).cuda()
    dy = torch.full((offset + count * (n + pad),), float("nan"), device="cuda")
    rows = dy[offset:].view(count, n + pad)[:, :n]
    rows.copy_(torch.from_numpy(_whole(count, n)))
    want = torch.zeros(vocabulary, n, dtype=torch.float64, device="cuda")
    real = tokens < vocabulary
    want.index_add_(0, tokens[real], rows[real].double())
    out = torch.full((offset + vocabulary * (n + pad),), float("nan"), device="cuda")
    work = torch.full((gpu.embedding_backward_workspace(count, vocabulary, n),), float("nan"), device="cuda")
    ids = tokens.int()
    torch.cuda.synchronize()
    gpu.embedding_backward(gpu.wrap(ids.data_ptr(), (count,), "u32"), gpu.wrap(dy.data_ptr() + offset * 4, (count, n), ld=n + pad),
                           gpu.wrap(out.data_ptr() + offset * 4, (vocabulary, n), ld=n + pad), gpu.wrap(work.data_ptr(), (work.numel(),)))
    gpu.sync()
    got = out[offset:].view(vocabulary, n + pad)
    assert torch.equal(got[:, :n].double(), want)
    assert got[:, n:].isnan().all() and out[:offset].isnan().all(), "elements beside dtable were written"
