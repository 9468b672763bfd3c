"""A residual MLP on the residual-block norms, trained in f32 and served in 4 bits.

The stream z [rows, width] passes ``blocks`` feed-forward blocks,

    h = pre(z),  y = relu(h W1 + b1) W2 + b2,  z = z + scale * gate * post(y),

between a stem (x W + b) and a head (norm, W, b) with softmax cross-entropy.
The end of one block and the norm before the next are one ``Gpu.block_forward``,
their gradients one ``Gpu.block_backward``.  ``Mx4ResidualMlp`` holds the trained
weights in microscaled 4-bit floating point and answers with 4-bit products.
The reference has neither (its networks are plain Dense stacks, nn.rs:161-207).

    python -m rgpu_b200.residual        trains on points in four quadrants and
                                        compares the f32 and the 4-bit answers
"""
from __future__ import annotations

import numpy as np

from .gpu import Gpu, GpuTensor, Norm, upload_labels


class ResidualMlp:
    """Parameters, their Adam state and the buffers of one batch size, f32."""

    def __init__(self, gpu: Gpu, inputs: int, width: int, hidden: int, classes: int, blocks: int, batch: int, *,
                 scale: float = 1.0, norm: str = "rms", eps: float = 1e-5, seed: int = 0):
        self.gpu, self.blocks, self.batch, self.scale, self.norm, self.eps = gpu, blocks, batch, scale, norm, eps
        self.inputs, self.width, self.hidden, self.classes = inputs, width, hidden, classes
        rng = np.random.default_rng(seed)

        def kaiming(d, n):
            b = np.sqrt(6.0 / d)
            return rng.uniform(-b, b, (d, n)).astype(np.float32)

        host = {"w_in": kaiming(inputs, width), "b_in": np.zeros((1, width), np.float32)}
        for i in range(blocks):
            host |= {f"w1_{i}": kaiming(width, hidden), f"b1_{i}": np.zeros((1, hidden), np.float32),
                     f"w2_{i}": kaiming(hidden, width), f"b2_{i}": np.zeros((1, width), np.float32),
                     f"post_{i}": np.ones((1, width), np.float32),
                     f"gate_{i}": np.full((1, width), 0.5, np.float32)}
        for i in range(blocks + 1):
            host[f"pre_{i}"] = np.ones((1, width), np.float32)
        host |= {"w_out": kaiming(width, classes), "b_out": np.zeros((1, classes), np.float32)}
        self.params = {k: gpu.upload(v) for k, v in host.items()}
        self.grads = {k: gpu.zeros(v.shape) for k, v in host.items()}
        self._m = {k: gpu.zeros(v.shape) for k, v in host.items()}
        self._v = {k: gpu.zeros(v.shape) for k, v in host.items()}
        self.steps = 0
        m = batch
        self._z = [gpu.zeros((m, width)) for _ in range(blocks + 1)]
        self._h = [gpu.zeros((m, width)) for _ in range(blocks + 1)]
        self._a = [gpu.zeros((m, hidden)) for _ in range(blocks)]
        self._y = [gpu.zeros((m, width)) for _ in range(blocks)]
        self._logits, self._delta, self._loss = gpu.zeros((m, classes)), gpu.zeros((m, classes)), gpu.zeros((m,))
        self._dz, self._dy, self._dh, self._da = (gpu.zeros((m, n)) for n in (width, width, width, hidden))
        self._work = gpu.zeros((gpu.block_backward_workspace(m, width),))
        widest = max(width, hidden, classes)
        self._colsum = gpu.zeros((-(-m // 64), widest))

    def _pre(self, i: int) -> Norm:
        return Norm(self.norm, self.eps, self.params[f"pre_{i}"])

    def _post(self, i: int) -> Norm:
        return Norm(self.norm, self.eps, self.params[f"post_{i}"])

    def forward(self, x: GpuTensor) -> GpuTensor:
        """Logits [batch, classes] of x [batch, inputs]."""
        g, p = self.gpu, self.params
        g.matmul_bias(x, p["w_in"], self._z[0], p["b_in"], False)
        g.block_forward(self._z[0], pre=self._pre(0), h=self._h[0])
        for i in range(self.blocks):
            g.matmul_bias(self._h[i], p[f"w1_{i}"], self._a[i], p[f"b1_{i}"], True)
            g.matmul_bias(self._a[i], p[f"w2_{i}"], self._y[i], p[f"b2_{i}"], False)
            g.block_forward(self._z[i], y=self._y[i], post=self._post(i), gate=p[f"gate_{i}"], scale=self.scale,
                            z=self._z[i + 1], pre=self._pre(i + 1), h=self._h[i + 1])
        g.matmul_bias(self._h[-1], p["w_out"], self._logits, p["b_out"], False)
        return self._logits

    def _dense_grads(self, x: GpuTensor, dy: GpuTensor, w: str, b: str):
        self.gpu.matmul_at_b(x, dy, self.grads[w])
        self.gpu.colsum(dy, self.grads[b], self._colsum)

    def backward(self, x: GpuTensor, labels: GpuTensor):
        """Gradients of the mean softmax cross-entropy of the last forward pass."""
        g, p, d = self.gpu, self.params, self.grads
        g.softmax_xent(self._logits, labels, self._delta, self._loss)
        self._dense_grads(self._h[-1], self._delta, "w_out", "b_out")
        g.matmul_a_bt(self._delta, p["w_out"], self._dh)
        dz = None  # the last block's stream has no reader but the norm before the head
        for i in reversed(range(self.blocks)):
            g.block_backward(self._z[i + 1], y=self._y[i], post=self._post(i), gate=p[f"gate_{i}"], scale=self.scale,
                             pre=self._pre(i + 1), dz=dz, dh=self._dh, dr=self._dz, dy=self._dy,
                             dgamma_post=d[f"post_{i}"], dgamma_pre=d[f"pre_{i + 1}"], dgate=d[f"gate_{i}"],
                             work=self._work)
            dz = self._dz
            self._dense_grads(self._a[i], self._dy, f"w2_{i}", f"b2_{i}")
            g.matmul_a_bt(self._dy, p[f"w2_{i}"], self._da)
            g.relu_bwd(self._a[i], self._da)
            self._dense_grads(self._h[i], self._da, f"w1_{i}", f"b1_{i}")
            g.matmul_a_bt(self._da, p[f"w1_{i}"], self._dh)
        g.block_backward(self._z[0], pre=self._pre(0), dz=dz, dh=self._dh, dr=self._dz, dgamma_pre=d["pre_0"],
                         work=self._work)
        self._dense_grads(x, self._dz, "w_in", "b_in")

    def step(self, x: GpuTensor, labels: GpuTensor, lr: float):
        """Forward, backward and one Adam update; reads nothing back."""
        self.forward(x)
        self.backward(x, labels)
        self.steps += 1
        for k, v in self.params.items():
            self.gpu.adam(v, self._m[k], self._v[k], self.grads[k], lr, self.steps)

    def loss(self) -> float:
        """Mean loss of the last backward pass (waits for the device)."""
        return float(self.gpu.download(self._loss).mean())

    def predict(self, x: np.ndarray) -> np.ndarray:
        return self.gpu.download(self.forward(self.gpu.upload(x))).argmax(1)


class Mx4ResidualMlp:
    """A trained ResidualMlp with its weights in 4 bits, for batches of `batch`
    rows: the stream and the blocks' outputs are bf16, every product's operands
    4-bit.  The norms write their 4-bit output themselves."""

    def __init__(self, model: ResidualMlp, batch: int):
        g = self.gpu = model.gpu
        self.model, self.batch = model, batch
        self._w = {k: g.mx4_quantize(v, axis=0) for k, v in model.params.items() if k.startswith("w")}
        n, f = model.width, model.hidden
        self._xq, self._hq, self._aq = g.mx4_zeros(batch, model.inputs), g.mx4_zeros(batch, n), g.mx4_zeros(batch, f)
        self._z, self._y, self._a = g.zeros((batch, n), "bf16"), g.zeros((batch, n), "bf16"), g.zeros((batch, f), "bf16")
        self._logits = g.zeros((batch, model.classes))

    def forward(self, x: GpuTensor) -> GpuTensor:
        """f32 logits [batch, classes] of x [batch, inputs], f32 or bf16."""
        g, m, p = self.gpu, self.model, self.model.params
        g.mx4_quantize(x, self._xq)
        g.mx4_matmul(self._xq, self._w["w_in"], self._z, bias=p["b_in"])
        g.block_forward(self._z, pre=m._pre(0), hq=self._hq)
        for i in range(m.blocks):
            g.mx4_matmul(self._hq, self._w[f"w1_{i}"], self._a, bias=p[f"b1_{i}"], relu=True)
            g.mx4_quantize(self._a, self._aq)
            g.mx4_matmul(self._aq, self._w[f"w2_{i}"], self._y, bias=p[f"b2_{i}"])
            g.block_forward(self._z, y=self._y, post=m._post(i), gate=p[f"gate_{i}"], scale=m.scale, z=self._z,
                            pre=m._pre(i + 1), hq=self._hq)
        g.mx4_matmul(self._hq, self._w["w_out"], self._logits, bias=p["b_out"])
        return self._logits

    def predict(self, x: np.ndarray) -> np.ndarray:
        return self.gpu.download(self.forward(self.gpu.upload(x))).argmax(1)


def quadrants(rows: int, inputs: int, seed: int):
    """Points with normal coordinates; the label is the quadrant of the first two."""
    x = np.random.default_rng(seed).standard_normal((rows, inputs)).astype(np.float32)
    return x, (x[:, 0] > 0).astype(np.uint32) + 2 * (x[:, 1] > 0).astype(np.uint32)


def main(steps: int = 150):
    gpu = Gpu(0)
    model = ResidualMlp(gpu, inputs=32, width=256, hidden=512, classes=4, blocks=3, batch=1024, scale=0.5)
    for step in range(steps):
        x, labels = quadrants(1024, 32, step)
        model.step(gpu.upload(x), upload_labels(gpu, labels), 1e-3)
        if step % 30 == 0 or step == steps - 1:
            print(f"step {step}: loss {model.loss():.4f}")
    x, labels = quadrants(1024, 32, 10**6)
    full = model.predict(x)
    small = Mx4ResidualMlp(model, 1024).predict(x)
    print(f"accuracy: f32 {np.mean(full == labels):.3f}, 4-bit {np.mean(small == labels):.3f}; "
          f"they agree on {np.mean(full == small):.3f}")


if __name__ == "__main__":
    main()
