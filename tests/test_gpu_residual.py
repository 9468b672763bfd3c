"""The residual MLP: every gradient against numpy in 64 bits, training, and the
4-bit model against the f32 one."""
import numpy as np
import pytest

import rgpu_b200
from rgpu_b200.residual import Mx4ResidualMlp, ResidualMlp, quadrants
from tests import ref_mx4 as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    g = rgpu_b200.Gpu(0)
    yield g
    g.close()


def _reference(p, x, labels, blocks, scale, norm):
    """Loss and gradients of the model in 64 bits."""
    eps, one = 1e-5, 0.0
    z, h, a, y = [x @ p["w_in"] + p["b_in"]], [], [], []
    h.append(R.norm(z[0], norm, eps, p["pre_0"], one))
    for i in range(blocks):
        a.append(np.maximum(h[i] @ p[f"w1_{i}"] + p[f"b1_{i}"], 0))
        y.append(a[i] @ p[f"w2_{i}"] + p[f"b2_{i}"])
        zi, hi = R.block_forward(z[i], y[i], (norm, eps, p[f"post_{i}"], one), p[f"gate_{i}"], scale,
                                 (norm, eps, p[f"pre_{i + 1}"], one))
        z.append(zi)
        h.append(hi)
    logits = h[-1] @ p["w_out"] + p["b_out"]
    e = np.exp(logits - logits.max(1, keepdims=True))
    prob = e / e.sum(1, keepdims=True)
    rows = np.arange(len(x))
    loss = -np.log(prob[rows, labels]).mean()
    delta = prob.copy()
    delta[rows, labels] -= 1
    delta /= len(x)
    g = {"w_out": h[-1].T @ delta, "b_out": delta.sum(0, keepdims=True)}
    dh, dz = delta @ p["w_out"].T, 0.0
    for i in reversed(range(blocks)):
        b = R.block_backward(z[i + 1], y[i], (norm, eps, p[f"post_{i}"], one), p[f"gate_{i}"], scale,
                             (norm, eps, p[f"pre_{i + 1}"], one), dz, dh)
        g[f"pre_{i + 1}"], g[f"post_{i}"], g[f"gate_{i}"] = b["dgamma_pre"], b["dgamma_post"], b["dgate"].sum(0, keepdims=True)
        dz, dy = b["dr"], b["dy"]
        g[f"w2_{i}"], g[f"b2_{i}"] = a[i].T @ dy, dy.sum(0, keepdims=True)
        da = (dy @ p[f"w2_{i}"].T) * (a[i] > 0)
        g[f"w1_{i}"], g[f"b1_{i}"] = h[i].T @ da, da.sum(0, keepdims=True)
        dh = da @ p[f"w1_{i}"].T
    b = R.block_backward(z[0], None, None, None, 1.0, (norm, eps, p["pre_0"], one), dz, dh)
    g["pre_0"] = b["dgamma_pre"]
    g["w_in"], g["b_in"] = x.T @ b["dr"], b["dr"].sum(0, keepdims=True)
    return loss, g


@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_gradients(gpu, norm):
    m = ResidualMlp(gpu, inputs=24, width=72, hidden=96, classes=5, blocks=2, batch=90, scale=0.5, norm=norm, seed=1)
    rng = np.random.default_rng(2)
    x, labels = rng.standard_normal((90, 24)).astype(np.float32), rng.integers(0, 5, 90).astype(np.uint32)
    tx = gpu.upload(x)
    m.forward(tx)
    m.backward(tx, rgpu_b200.upload_labels(gpu, labels))
    p = {k: gpu.download(v).astype(np.float64) for k, v in m.params.items()}
    loss, want = _reference(p, x.astype(np.float64), labels, 2, 0.5, norm)
    assert abs(m.loss() - loss) < 1e-5
    assert sorted(want) == sorted(m.grads)
    for k, w in want.items():
        got = gpu.download(m.grads[k])
        # the f32 bar of the framework's gradients, 1e-4 relative in the 2-norm
        assert np.linalg.norm(got - w) <= 1e-4 * np.linalg.norm(w), k


def test_training_and_serving_in_4_bits(gpu):
    m = ResidualMlp(gpu, inputs=32, width=128, hidden=256, classes=4, blocks=2, batch=512, scale=0.5)
    first = None
    for step in range(100):
        x, labels = quadrants(512, 32, step)
        m.step(gpu.upload(x), rgpu_b200.upload_labels(gpu, labels), 1e-3)
        if first is None:
            first = m.loss()
    assert m.loss() < 0.5 * first
    x, labels = quadrants(512, 32, 10**6)
    full = gpu.download(m.forward(gpu.upload(x)))
    q = Mx4ResidualMlp(m, 512)
    small = gpu.download(q.forward(gpu.upload(x)))
    assert np.mean(full.argmax(1) == labels) > 0.8
    # a 4-bit operand is off by at most a quarter of its block's scale at 1/16 of the largest element or more; over
    # 32 and more terms that is about a tenth of the result
    assert np.mean(full.argmax(1) == small.argmax(1)) > 0.85
    one = Mx4ResidualMlp(m, 1)  # a single row takes the same values
    got = gpu.download(one.forward(gpu.upload(x[:1])))
    assert np.allclose(got, small[:1], rtol=2e-2, atol=2e-2)
