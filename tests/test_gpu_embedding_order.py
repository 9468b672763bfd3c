"""The embedding's gradient called again and again on one workspace, with other tokens each
time and nothing waited for between the calls; captured; with and without programmatic dependent launches."""
import os

import numpy as np
import pytest

import rgpu_b200
from rgpu_b200 import Dropout
from tests.test_gpu_embedding import _round, _tokens
from tests.test_gpu_embedding_exact import _sums, _whole
from tests.test_gpu_fp8 import _upload, gpu  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("count,n,vocabulary", [(3000, 264, 500), (9000, 200, 700), (9000, 1024, 20000), (60000, 64, 3000), (70000, 40, 3000)])
def test_one_workspace_and_other_tokens_at_each_call(gpu, count, n, vocabulary, dtype):
    calls = 8
    rng = np.random.default_rng(count + n)
    tokens = [_tokens(("zipf", "uniform", "runs", "one")[i % 4], rng, count, vocabulary).astype(np.uint32) for i in range(calls)]
    dys = [_whole(count, n, seed) for seed in (0, 11)]
    words = gpu.embedding_backward_workspace(count, vocabulary, n)
    work = torch.full((words,), float("nan"), device="cuda")
    out = torch.full((calls, vocabulary, n), float("nan"), device="cuda")
    t = [rgpu_b200.upload_labels(gpu, v) for v in tokens]
    tdy = [_upload(gpu, v, dtype) for v in dys]
    w = gpu.wrap(work.data_ptr(), (words,))
    d = [gpu.wrap(out[i].data_ptr(), (vocabulary, n)) for i in range(calls)]
    torch.cuda.synchronize()
    for _ in range(3):
        for i in range(calls):
            gpu.embedding_backward(t[i], tdy[i % 2][0], d[i], w)
    gpu.sync()
    for i in range(calls):
        want = torch.from_numpy(_sums(vocabulary, tokens[i], dys[i % 2])).float().cuda()
        assert torch.equal(out[i], want), f"call {i}"


@pytest.mark.parametrize("count,n,vocabulary", [(9000, 200, 700), (9000, 1024, 20000), (70000, 40, 3000)])
def test_captured_with_other_tokens_at_each_replay(gpu, count, n, vocabulary):
    replays = 6
    rng = np.random.default_rng(count)
    tokens = [_tokens(("zipf", "uniform", "one")[i % 3], rng, count, vocabulary).astype(np.int64).astype(np.uint32) for i in range(replays)]
    dy = _whole(count, n)
    every = torch.from_numpy(np.stack(tokens).view(np.int32)).cuda()
    now = every[0].clone()
    tdy, _k, _ = _upload(gpu, dy, "f32")
    t, d = gpu.wrap(now.data_ptr(), (count,), "u32"), torch.empty(vocabulary, n, device="cuda")
    td = gpu.wrap(d.data_ptr(), (vocabulary, n))
    work = gpu.zeros((gpu.embedding_backward_workspace(count, vocabulary, n),))
    gpu.sync()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    gpu.set_stream(stream.cuda_stream)
    try:
        with torch.cuda.graph(graph, stream=stream):
            gpu.embedding_backward(t, tdy, td, work)
            gpu.embedding_backward(t, tdy, td, work, accumulate=True)
    finally:
        gpu.set_stream(None)
    got = []
    with torch.cuda.stream(stream):
        for i in range(replays):
            now.copy_(every[i])
            graph.replay()
            got.append(d.clone())
    torch.cuda.synchronize()
    for i in range(replays):
        assert torch.equal(got[i], torch.from_numpy(2 * _sums(vocabulary, tokens[i], dy)).float().cuda()), f"replay {i}"


def _chain(pdl, count, n, vocabulary, dtype):
    """Embedding, dropout, 8-bit operands both ways, their product, and the gradient back, three times over without waiting."""
    saved = os.environ.get("RTGPU_PDL")
    os.environ["RTGPU_PDL"] = pdl
    try:
        g = rgpu_b200.Gpu(0)
    finally:
        if saved is None:
            del os.environ["RTGPU_PDL"]
        else:
            os.environ["RTGPU_PDL"] = saved
    rng = np.random.default_rng(count)
    table, weights = (g.upload(_round(rng.standard_normal(s), dtype), dtype) for s in ((vocabulary, n), (n, 200)))
    y, dx, out = g.zeros((count, n), dtype), g.zeros((count, n), dtype), g.zeros((count, 200), dtype)
    d, work = g.zeros((vocabulary, n)), g.zeros((g.embedding_backward_workspace(count, vocabulary, n),))
    tokens = [rgpu_b200.upload_labels(g, _tokens("zipf", rng, count, vocabulary).astype(np.uint32)) for _ in range(3)]
    qy, qw, qd, qv = g.fp8_zeros(count, n), g.fp8_zeros(200, n), g.fp8_zeros(count, 200), g.fp8_zeros(n, 200)
    g.sync()
    for step, t in enumerate(tokens):
        mask = Dropout(0.25, 99, step=step)
        g.embedding_forward(table, t, y, scale=3.0)
        g.dropout(y, y, mask)
        g.fp8_matmul(g.fp8_quantize(y, qy), g.fp8_quantize(weights, qw, axis=0), out)
        g.fp8_matmul(g.fp8_quantize(out, qd), g.fp8_quantize(weights, qv), dx)
        g.dropout(dx, dx, mask)
        g.embedding_backward(t, dx, d, work, accumulate=step > 0)
    result = [g.download(x) for x in (y, out, dx, d)]
    g.close()
    return result


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("count,n,vocabulary", [(700, 130, 90), (9000, 256, 700), (70000, 64, 3000)])
def test_dependent_launches_change_no_bit(count, n, vocabulary, dtype):
    for a, b in zip(_chain("0", count, n, vocabulary, dtype), _chain("1", count, n, vocabulary, dtype)):
        assert np.array_equal(a, b) and np.isfinite(a).all() and a.any()
