"""The embedding and its gradient on the GPU against numpy in 64 bits."""
import numpy as np
import pytest

import rgpu_b200
from rgpu_b200 import gpu as G
from tests import ref_tokens as R
from tests.test_gpu_fp8 import _bf16, _upload, gpu  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -24  # half a step of f32
HALF = {"f32": U, "bf16": 2.0 ** -8}


def _round(x, dtype):
    return _bf16(x) if dtype == "bf16" else np.ascontiguousarray(x, np.float32)


SIZES = [(1, 1, 1), (1, 8, 2), (3, 7, 5), (5, 256, 300), (17, 257, 64), (64, 1000, 1000), (130, 33, 70000), (1000, 520, 17)]


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("table", ["f32", "bf16"])
@pytest.mark.parametrize("count,n,vocabulary", SIZES)
def test_lookup(gpu, count, n, vocabulary, table, out):
    rng = np.random.default_rng(count + n)
    e = _round(rng.standard_normal((vocabulary, n)), table)
    tokens = rng.integers(0, vocabulary, count).astype(np.uint32)
    tokens[::5] = vocabulary  # padding
    tokens[3::11] = 0xFFFFFFFF
    tokens[count // 2] = vocabulary - 1
    want = R.embedding(e.astype(np.float64), tokens, np.float64(np.float32(3.7)))
    t = rgpu_b200.upload_labels(gpu, tokens)
    for pad, offset in ((0, 0), (3, 1), (-n % 16, 8)):
        te, _k, _ = _upload(gpu, e, table, n + pad, offset)
        y, buf, view = _upload(gpu, np.zeros((count, n)), out, n + pad, offset)
        before = buf.clone()
        gpu.embedding_forward(te, t, y, scale=3.7)
        gpu.sync()
        got = view.double().cpu().numpy()
        # one product in f32, one more rounding to bf16
        assert np.all(np.abs(got - want) <= (U + (HALF["bf16"] * (1 + U) if out == "bf16" else 0)) * np.abs(want))
        view.copy_(before[offset:offset + count * (n + pad)].view(count, n + pad)[:, :n])
        assert torch.equal(buf.isnan(), before.isnan()), "elements beside y were written"


def test_infinities_and_nan_of_the_table_stay_in_their_rows(gpu):
    e = np.ones((4, 300), np.float32)
    e[1], e[2] = np.inf, np.nan
    y = gpu.zeros((5, 300))
    gpu.embedding_forward(gpu.upload(e), rgpu_b200.upload_labels(gpu, [0, 1, 2, 3, 4]), y, scale=2.0)
    got = gpu.download(y)
    assert (got[[0, 3]] == 2).all() and np.isposinf(got[1]).all() and np.isnan(got[2]).all() and (got[4] == 0).all()


def _tokens(kind, rng, count, vocabulary):
    if kind == "uniform":
        return rng.integers(0, vocabulary, count)
    if kind == "one":
        return np.full(count, vocabulary // 2)
    if kind == "padding":
        return np.full(count, vocabulary) + rng.integers(0, 100, count)
    if kind == "runs":  # runs of 1, 63, 64, 65, 127 ... positions: on, before and behind the pieces' borders
        lengths = [1, 63, 64, 65, 127, 1, 128, 200, 3, 61, 700]
        t = np.concatenate([np.full(n, i % max(1, vocabulary)) for i, n in enumerate(lengths * (count // sum(lengths) + 1))])[:count]
        return rng.permutation(t)
    p = 1.0 / np.arange(1, vocabulary + 1)  # zipf
    t = rng.permutation(vocabulary)[rng.choice(vocabulary, count, p=p / p.sum())]
    t[rng.random(count) < 0.1] = vocabulary
    return t


BACK = [("uniform", 1, 1, 1), ("uniform", 5, 3, 2), ("uniform", 63, 256, 300), ("one", 64, 40, 7), ("one", 65, 257, 1),
        ("one", 5000, 264, 3), ("padding", 100, 16, 9), ("padding", 3000, 8, 70000), ("zipf", 1023, 100, 255),
        ("zipf", 2047, 1000, 256), ("zipf", 1025, 30, 257), ("zipf", 10000, 512, 5000), ("zipf", 4096, 24, 70001),
        ("uniform", 2049, 17, 2 ** 21 - 1), ("uniform", 70000, 9, 300), ("runs", 2500, 300, 11), ("runs", 9000, 72, 1000),
        ("zipf", 300000, 8, 50257),
        # the sorts' other forms: over launches with more buckets than warps' counters, keys of three digits, wide gaps
        ("uniform", 70000, 5, 2 ** 21 - 1), ("zipf", 66000, 4, 300000), ("uniform", 70000, 1, 17000000), ("one", 65537, 12, 100), ("padding", 70000, 4, 1000),
        ("zipf", 8192, 100, 1300), ("one", 8191, 40, 1000), ("uniform", 5000, 256, 1600), ("padding", 8000, 24, 70000), ("runs", 8100, 33, 1001),
        ("zipf", 8193, 64, 1000), ("uniform", 4097, 16, 255), ("zipf", 4097, 513, 1384), ("uniform", 6001, 1021, 511), ("zipf", 17000, 40, 70000),
        ("uniform", 5000, 5, 2 ** 21 - 1), ("one", 4097, 8, 2000003), ("zipf", 65536, 4, 66000), ("uniform", 12289, 130, 9000)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind,count,n,vocabulary", BACK)
def test_gradient(gpu, kind, count, n, vocabulary, dtype):
    rng = np.random.default_rng(count * 7 + n)
    tokens = _tokens(kind, rng, count, vocabulary).astype(np.uint32)
    dy = _round(rng.standard_normal((count, n)) + 0.3, dtype)
    scale = np.float32(2.5)
    d, size, times = R.embedding_backward(vocabulary, tokens, dy.astype(np.float64), np.float64(scale))
    # an f32 sum of `times` addends in any order: times - 1 roundings of at most the sum of magnitudes, the product with
    # the scale, and (accumulated) one more sum
    tol = (times[:, None] + 1) * U * size
    t = rgpu_b200.upload_labels(gpu, tokens)
    words = gpu.embedding_backward_workspace(count, vocabulary, n)
    for pad, offset in ((0, 0), (3, 1), (-n % 8, 8)):
        work = torch.full((words + 64,), float("nan"), device="cuda")
        tdy, _k, _ = _upload(gpu, dy, dtype, n + pad, offset)
        out, buf, view = _upload(gpu, np.full((vocabulary, n), 7.0), "f32", n + pad, offset)
        outside = torch.ones_like(buf, dtype=torch.bool)
        outside[offset:offset + vocabulary * (n + pad)].view(vocabulary, n + pad)[:, :n] = False
        w = gpu.wrap(work.data_ptr(), (words,))
        gpu.embedding_backward(t, tdy, out, w, scale=float(scale))
        gpu.sync()
        got = view.double().cpu().numpy()
        assert np.all(np.abs(got - d) <= tol)
        first = view.clone()
        old = torch.full((1, 1), 1.5, device="cuda")
        view.copy_(old.expand(vocabulary, n))
        torch.cuda.synchronize()
        gpu.embedding_backward(t, tdy, out, w, scale=float(scale), accumulate=True)
        gpu.sync()
        got = view.double().cpu().numpy()
        assert np.all(np.abs(got - (d + 1.5)) <= tol + U * (np.abs(d) + tol + 1.5))
        assert (got[times == 0] == 1.5).all(), "a row that does not occur was touched"
        gpu.embedding_backward(t, tdy, out, w, scale=float(scale))
        gpu.sync()
        assert torch.equal(view, first), "the same call gave other bits"
        assert buf[outside].isnan().all() and work[words:].isnan().all(), "elements beside dtable or work were written"


def test_gradient_against_differences(gpu):
    # the forward pass's own differences: linear in the table, so only roundings separate the two
    rng = np.random.default_rng(4)
    count, n, vocabulary = 300, 40, 50
    tokens = rng.integers(0, vocabulary + 5, count).astype(np.uint32)
    c, way = rng.standard_normal((count, n)).astype(np.float32), rng.standard_normal((vocabulary, n)).astype(np.float32)
    t = rgpu_b200.upload_labels(gpu, tokens)
    y, d = gpu.zeros((count, n)), gpu.zeros((vocabulary, n))
    gpu.embedding_forward(gpu.upload(way), t, y, scale=0.5)
    gpu.embedding_backward(t, gpu.upload(c), d, gpu.zeros((gpu.embedding_backward_workspace(count, vocabulary, n),)), scale=0.5)
    slope = (gpu.download(y).astype(np.float64) * c).sum()
    assert abs(slope - (gpu.download(d).astype(np.float64) * way).sum()) <= count * U * (np.abs(gpu.download(y)) * np.abs(c)).sum()


def test_infinities_stay_in_their_rows(gpu):
    tokens = np.arange(500, dtype=np.uint32) % 7
    dy = np.ones((500, 20), np.float32)
    dy[6], dy[5] = np.inf, np.nan  # of tokens 6 and 5
    d = gpu.zeros((7, 20))
    gpu.embedding_backward(rgpu_b200.upload_labels(gpu, tokens), gpu.upload(dy), d,
                           gpu.zeros((gpu.embedding_backward_workspace(500, 7, 20),)))
    got = gpu.download(d)
    assert np.isposinf(got[6]).all() and np.isnan(got[5]).all() and np.isfinite(got[:5]).all()


@pytest.mark.parametrize("count", [300, 9000, 70000])
def test_what_padding_rows_hold_does_not_matter(gpu, count):
    rng = np.random.default_rng(count)
    tokens = rng.integers(0, 60, count).astype(np.uint32)
    tokens[rng.random(count) < 0.5] = 40 + 20 + rng.integers(0, 9)  # half of them: past the 40 rows of the table
    dy = rng.integers(-3, 4, (count, 24)).astype(np.float32)
    want = R.embedding_backward(40, tokens, dy.astype(np.float64), 1.0)[0]
    dy[tokens >= 40] = np.nan
    d = gpu.zeros((40, 24))
    gpu.embedding_backward(rgpu_b200.upload_labels(gpu, tokens), gpu.upload(dy), d,
                           gpu.zeros((gpu.embedding_backward_workspace(count, 40, 24),)))
    assert np.array_equal(gpu.download(d), want)  # whole numbers


def test_two_contexts_at_once(gpu):
    # each with its own stream and workspace, their launches between one another's
    other = rgpu_b200.Gpu(0)
    rng = np.random.default_rng(8)
    jobs = []
    for g, count in ((gpu, 5000), (other, 66000)):
        tokens = rng.integers(0, 700, count).astype(np.uint32)
        dy = rng.integers(-3, 4, (count, 40)).astype(np.float32)
        jobs.append((g, rgpu_b200.upload_labels(g, tokens), g.upload(dy), g.zeros((650, 40)),
                     g.zeros((g.embedding_backward_workspace(count, 650, 40),)), R.embedding_backward(650, tokens, dy.astype(np.float64), 2.0)[0]))
    for _ in range(20):
        for g, t, dy, d, work, _w in jobs:
            g.embedding_backward(t, dy, d, work, scale=2.0)
    for g, _t, _dy, d, _work, want in jobs:
        assert np.array_equal(g.download(d), want)
    del jobs
    other.close()


def test_empty_extents(gpu):
    none = gpu.wrap(gpu.zeros((4,)).ptr, (0,), "u32")
    work = gpu.zeros((gpu.embedding_backward_workspace(0, 5, 8),))
    d = gpu.upload(np.full((5, 8), 3.0))
    gpu.embedding_backward(none, gpu.zeros((0, 8)), d, work, accumulate=True)
    assert (gpu.download(d) == 3).all()
    gpu.embedding_backward(none, gpu.zeros((0, 8)), d, work)
    assert (gpu.download(d) == 0).all()
    gpu.embedding_forward(gpu.zeros((5, 8)), none, gpu.zeros((0, 8)))
    y = gpu.upload(np.full((2, 8), 3.0))
    gpu.embedding_forward(gpu.zeros((0, 8)), rgpu_b200.upload_labels(gpu, [0, 1]), y)  # no rows at all: every token is padding
    assert (gpu.download(y) == 0).all()
    gpu.embedding_backward(rgpu_b200.upload_labels(gpu, [0, 1]), gpu.zeros((2, 8)), gpu.zeros((0, 8)),
                           gpu.zeros((gpu.embedding_backward_workspace(2, 0, 8),)))
    gpu.sync()


def test_captured_and_on_another_stream(gpu):
    rng = np.random.default_rng(9)
    count, n, vocabulary = 3000, 264, 500
    e = rng.standard_normal((vocabulary, n)).astype(np.float32)
    tokens = torch.from_numpy(rng.integers(0, vocabulary, count).astype(np.int32)).cuda()
    te, y, d = gpu.upload(e), gpu.zeros((count, n)), gpu.zeros((vocabulary, n))
    t = gpu.wrap(tokens.data_ptr(), (count,), "u32")
    work = gpu.zeros((gpu.embedding_backward_workspace(count, vocabulary, n),))
    gpu.sync()
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    gpu.set_stream(stream.cuda_stream)
    try:
        with torch.cuda.graph(graph, stream=stream):
            gpu.embedding_forward(te, t, y, scale=2.0)
            gpu.embedding_backward(t, y, d, work)
    finally:
        gpu.set_stream(None)
    for seed in (1, 2):
        new = np.random.default_rng(seed).integers(0, vocabulary + 20, count).astype(np.int32)
        tokens.copy_(torch.from_numpy(new))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = R.embedding(e.astype(np.float64), new, 2.0)
        assert np.array_equal(gpu.download(y), want)  # a product with two is exact
        g, size, times = R.embedding_backward(vocabulary, new, want, 1.0)
        assert np.all(np.abs(gpu.download(d) - g) <= (times[:, None] + 1) * U * size)


def test_refusals(gpu):
    e, y = gpu.zeros((10, 8)), gpu.zeros((3, 8))
    t = rgpu_b200.upload_labels(gpu, [1, 2, 3])
    work = gpu.zeros((gpu.embedding_backward_workspace(3, 10, 8),))
    short = gpu.zeros((gpu.embedding_backward_workspace(3, 10, 8) - 1,))

    def refused(call, word):
        with pytest.raises(rgpu_b200.RtError) as err:
            call()
        assert err.value.code == G.RT_ERR_INVALID and word in str(err.value), str(err.value)

    refused(lambda: gpu.embedding_forward(e, t, gpu.zeros((3, 9))), "table is 10x8")
    refused(lambda: gpu.embedding_forward(e, t, gpu.zeros((4, 8))), "3 tokens for 4 rows")
    refused(lambda: gpu.embedding_forward(e, gpu.zeros((3,)), y), "vector of u32")
    refused(lambda: gpu.embedding_forward(gpu.zeros((10, 8), "u32"), t, y), "f32 or bf16")
    refused(lambda: gpu.embedding_forward(e, t, gpu.zeros((3, 8), "u32")), "f32 or bf16")
    refused(lambda: gpu.embedding_backward(t, y, e, short), "packed f32")
    refused(lambda: gpu.embedding_backward(t, y, gpu.zeros((10, 8), "bf16"), work), "must be f32")
    refused(lambda: gpu.embedding_backward(t, y, gpu.zeros((10, 9)), work), "dtable 10x9")
    refused(lambda: gpu.embedding_backward(t, gpu.zeros((4, 8)), e, work), "3 tokens for 4 rows")
    refused(lambda: gpu.embedding_backward(t, gpu.zeros((3, 8), "u32"), e, work), "f32 or bf16")
    refused(lambda: gpu.embedding_backward(t, gpu.zeros((3, 1)), gpu.wrap(e.ptr, (1 << 31, 1)), work), "2^31")
    other = rgpu_b200.Gpu(0)
    refused(lambda: gpu.embedding_forward(other.zeros((10, 8)), t, y), "another context")
    refused(lambda: gpu.embedding_backward(t, y, e, other.zeros((5000,))), "another context")


def test_offsets_past_32_bits(gpu):
    # a table and a gradient of more than 2^31 elements: rows at both ends
    vocabulary, n, count = 1100000, 2048, 5000
    table = torch.zeros(vocabulary, n, dtype=torch.bfloat16, device="cuda")
    table[-1], table[0], table[vocabulary // 2] = 3.0, 1.0, 2.0
    tokens = np.random.default_rng(0).choice([0, vocabulary // 2, vocabulary - 1, vocabulary], count).astype(np.uint32)
    torch.cuda.synchronize()
    t, y = rgpu_b200.upload_labels(gpu, tokens), torch.zeros(count, n, device="cuda")
    ty = gpu.wrap(y.data_ptr(), (count, n))
    gpu.embedding_forward(gpu.wrap(table.data_ptr(), (vocabulary, n), "bf16"), t, ty)
    gpu.sync()
    want = np.select([tokens == 0, tokens == vocabulary // 2, tokens == vocabulary - 1], [1.0, 2.0, 3.0], 0.0)
    assert np.array_equal(y.cpu().numpy(), np.repeat(want[:, None], n, 1))
    del table
    d = torch.full((vocabulary, n), 7.0, device="cuda")
    torch.cuda.synchronize()
    gpu.embedding_backward(t, ty, gpu.wrap(d.data_ptr(), (vocabulary, n)),
                           gpu.zeros((gpu.embedding_backward_workspace(count, vocabulary, n),)))
    gpu.sync()
    for row, value in ((0, 1), (vocabulary // 2, 2), (vocabulary - 1, 3)):
        assert (d[row] == value * np.sum(tokens == row)).all()  # whole numbers
        d[row] = 0
    assert not d.any(), "a row of a token that does not occur is not zero"


def test_a_vector_of_tokens_may_be_a_column(gpu):
    t = gpu.wrap(rgpu_b200.upload_labels(gpu, [3, 1, 2]).ptr, (3,), "u32")
    column = gpu.wrap(t.ptr, (3, 1), "u32")
    e, y, z = gpu.upload(np.arange(32).reshape(4, 8)), gpu.zeros((3, 8)), gpu.zeros((3, 8))
    gpu.sync()
    gpu.embedding_forward(e, t, y)
    gpu.embedding_forward(e, column, z)
    assert np.array_equal(gpu.download(y), gpu.download(z))
