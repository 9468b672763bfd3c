"""The residual MLP over windows of tokens: embedding, dropout and 8-bit products together."""
import os
import subprocess
import sys

import numpy as np
import pytest

import rgpu_b200
from rgpu_b200 import Dropout
from rgpu_b200 import tape as T
from rgpu_b200.residual import ResidualMlp, TokenResidualMlp, sentences
from tests import ref_tokens as R
from tests.test_gpu_fp8 import _product_check, gpu  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
U = 2.0 ** -24


def _masks(m, batch, sizes):
    out = []
    for site, n in enumerate(sizes):
        kept, share = R.keep(batch, n, m.dropout, m.seed, site=site, step=m.steps)
        out.append(kept / share)
    return out


@pytest.mark.parametrize("dropout", [0.0, 0.25])
def test_gradients_with_f32_products(gpu, dropout):
    vocabulary, context, embed, batch, hidden = 50, 5, 12, 90, 96
    m = TokenResidualMlp(gpu, vocabulary, context, embed, width=72, hidden=hidden, classes=7, blocks=2, batch=batch,
                         scale=0.5, dropout=dropout, products="f32", seed=3)
    m.steps = 17
    rng = np.random.default_rng(2)
    tokens = rng.integers(0, vocabulary + 5, (batch, context)).astype(np.uint32)
    labels = rng.integers(0, 7, batch).astype(np.uint32)
    t = rgpu_b200.upload_labels(gpu, tokens.ravel())
    m.forward(t)
    m.backward(t, rgpu_b200.upload_labels(gpu, labels))
    p = {k: gpu.download(v).astype(np.float64) for k, v in m.params.items()}
    loss, want = R.token_model(p, tokens, labels, 2, 0.5, _masks(m, batch, [context * embed, hidden, hidden]))
    assert abs(m.loss() - loss) < 1e-5
    assert sorted(want) == sorted(m.grads)
    for k, w in want.items():
        got = gpu.download(m.grads[k])
        # the f32 bar of the framework's gradients, 1e-4 relative in the 2-norm
        assert np.linalg.norm(got - w) <= 1e-4 * np.linalg.norm(w), k


def test_products_in_8_bits_are_those_of_the_quantised_operands(gpu):
    vocabulary, context, embed, batch = 40, 4, 36, 150
    m = TokenResidualMlp(gpu, vocabulary, context, embed, width=200, hidden=260, classes=30, blocks=1, batch=batch,
                         scale=0.5, dropout=0.2, seed=4)
    rng = np.random.default_rng(3)
    tokens = rng.integers(0, vocabulary + 3, (batch, context)).astype(np.uint32)
    t, labels = rgpu_b200.upload_labels(gpu, tokens.ravel()), rgpu_b200.upload_labels(gpu, rng.integers(0, 30, batch))
    m.forward(t)
    m.backward(t, labels)
    p = {k: gpu.download(v) for k, v in m.params.items()}
    down = {k: gpu.download(v).astype(np.float64) for k, v in (("h", m._h[-1]), ("a", m._a[0]), ("delta", m._delta),
                                                               ("dz", m._dz), ("x", m._x_rows), ("dx", m._dx_rows), ("y", m._y[0]))}

    def val(t):
        return R.values(*R.quantize(t), t.shape[1])

    _product_check(gpu.download(m._logits).astype(np.float64), val(down["h"]), val(p["w_out"].T), p["b_out"], False, "f32")
    _product_check(down["y"], val(down["a"]), val(p["w2_0"].T), p["b2_0"], False, "f32")
    for w, x, dy in (("w_out", "h", "delta"), ("w_in", "x", "dz")):
        _product_check(gpu.download(m.grads[w]).astype(np.float64), val(down[x].T), val(down[dy].T), None, False, "f32")
    # the embeddings: what was looked up and dropped, and the way back
    masks = _masks(m, batch, [context * embed])
    x = R.embedding(p["embedding"].astype(np.float64), tokens.ravel(), np.sqrt(embed)).reshape(batch, -1) * masks[0]
    assert np.all(np.abs(down["x"] - x) <= 4 * U * np.abs(x))  # scale, two products, 1 / (1 - p)
    dropped = masks[0] == 0
    assert (down["dx"][dropped] == 0).all()
    free = np.where(dropped, 0.0, down["dx"] / masks[0].max())
    a, b = val(down["dz"]), val(p["w_in"])
    size = np.abs(a) @ np.abs(b).T
    assert np.all(np.abs(free - np.where(dropped, 0.0, a @ b.T)) <= (2 * (a.shape[1] + 2) + 2) * U * size + 1e-37)
    g, size, times = R.embedding_backward(vocabulary, tokens.ravel(), down["dx"].reshape(batch * context, -1), np.sqrt(embed))
    assert np.all(np.abs(gpu.download(m.grads["embedding"]) - g) <= (times[:, None] + 2) * U * size)


def test_a_step_changes_every_parameter_and_prediction_drops_nothing(gpu):
    m = TokenResidualMlp(gpu, 61, 8, 32, width=128, hidden=256, classes=61, blocks=2, batch=256, scale=0.5)
    before = {k: gpu.download(v) for k, v in m.params.items()}
    for step in range(3):
        x, labels = sentences(256, 8, 61, step)
        m.step(rgpu_b200.upload_labels(gpu, x.ravel()), rgpu_b200.upload_labels(gpu, labels), 1e-3)
    for k, v in m.params.items():
        assert not np.array_equal(gpu.download(v), before[k]) and np.isfinite(gpu.download(v)).all(), k
    x, _ = sentences(256, 8, 61, 99)
    one = m.predict(x)
    m.steps += 1  # another step's masks would change what a training pass answers
    assert np.array_equal(one, m.predict(x)) and m.training


def test_refusals(gpu):
    with pytest.raises(ValueError):
        TokenResidualMlp(gpu, 10, 2, 6, 8, 8, 3, 1, 4)
    with pytest.raises(ValueError):
        TokenResidualMlp(gpu, 10, 2, 8, 8, 8, 3, 1, 4, products="fp4")


def test_on_the_tape(gpu):
    # one table looked up twice, dropout, and a Dense layer: every adjoint
    rng = np.random.default_rng(6)
    e, w = rng.standard_normal((30, 20)).astype(np.float32), rng.standard_normal((20, 4)).astype(np.float32)
    first, second = rng.integers(0, 33, 70), rng.integers(0, 33, 70)
    c = rng.standard_normal((70, 4)).astype(np.float32)
    pe, pw, tape = T.Param(gpu, e), T.Param(gpu, w), T.Tape(gpu)
    mask = Dropout(0.4, 9, site=2, step=5)
    table = pe.watch(tape)
    x = table.embedding(rgpu_b200.upload_labels(gpu, first), 1.5).add(table.embedding(rgpu_b200.upload_labels(gpu, second)))
    y = x.dropout(mask).matmul(pw.watch(tape))
    grads = y.mul(T.constant(tape, c)).sum().backward()
    kept, share = R.keep(70, 20, 0.4, 9, site=2, step=5)
    d = kept / share
    xs = R.embedding(e.astype(np.float64), first, 1.5) + R.embedding(e.astype(np.float64), second, 1.0)
    assert np.allclose(y.value(), (xs * d) @ w, rtol=1e-5, atol=1e-5)
    dx = (c.astype(np.float64) @ w.T) * d
    want = R.embedding_backward(30, first, dx, 1.5)[0] + R.embedding_backward(30, second, dx, 1.0)[0]
    for got, ref in ((grads.of(pe), want), (grads.of(pw), (xs * d).T @ c)):
        assert np.linalg.norm(got - ref) <= 1e-5 * np.linalg.norm(ref)  # f32 products of 20 and 70 terms
    # the same token and variable once more, and what the tape refuses
    with pytest.raises(rgpu_b200.RtError):
        T.constant(T.Tape(gpu), c).dropout(Dropout(0.5, 1, step_at=gpu.zeros((1,), "u32")))
    with pytest.raises(rgpu_b200.RtError):
        T.constant(T.Tape(gpu), e).embedding(gpu.zeros((4,)))


def test_the_command(gpu):
    out = subprocess.run([sys.executable, "-c", "from rgpu_b200 import residual; residual.main_tokens(steps=3)"], cwd=ROOT,
                         capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "next token right" in out.stdout, out.stderr[-2000:]
