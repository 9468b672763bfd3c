"""A residual MLP on the residual-block norms, trained in f32 and served in 4 bits.

The stream z [rows, width] passes ``blocks`` feed-forward blocks,

    h = pre(z),  y = relu(h W1 + b1) W2 + b2,  z = z + scale * gate * post(y),

between a stem (x W + b) and a head (norm, W, b) with softmax cross-entropy.
The end of one block and the norm before the next are one ``Gpu.block_forward``,
their gradients one ``Gpu.block_backward``.  ``Mx4ResidualMlp`` holds the trained
weights in microscaled 4-bit floating point and answers with 4-bit products.
The reference has neither (its networks are plain Dense stacks, nn.rs:161-207).

``TokenResidualMlp`` is the same over a window of tokens: embeddings, dropout,
and the Dense layers' products in 8 bits.

    python -m rgpu_b200.residual        trains on points in four quadrants and
                                        compares the f32 and the 4-bit answers
    python -m rgpu_b200.residual tokens trains to say the next token of a text
                                        drawn from a random grammar
"""
from __future__ import annotations

import numpy as np

from .gpu import Dropout, Gpu, GpuTensor, Norm, upload_labels


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
        self._dense(x, "w_in", "b_in", self._z[0])
        g.block_forward(self._z[0], pre=self._pre(0), h=self._h[0])
        for i in range(self.blocks):
            self._dense(self._h[i], f"w1_{i}", f"b1_{i}", self._a[i], relu=True)
            self._drop(self._a[i], i)
            self._dense(self._a[i], f"w2_{i}", f"b2_{i}", self._y[i])
            g.block_forward(self._z[i], y=self._y[i], post=self._post(i), gate=p[f"gate_{i}"], scale=self.scale,
                            z=self._z[i + 1], pre=self._pre(i + 1), h=self._h[i + 1])
        self._dense(self._h[-1], "w_out", "b_out", self._logits)
        return self._logits

    # What a kind of model does its own way: a Dense layer's products, and dropout of block i's hidden activations or
    # of their gradient (in place; here there is none).
    def _dense(self, x: GpuTensor, w: str, b: str, y: GpuTensor, relu: bool = False):
        self.gpu.matmul_bias(x, self.params[w], y, self.params[b], relu)

    def _dense_dx(self, dy: GpuTensor, w: str, dx: GpuTensor):
        self.gpu.matmul_a_bt(dy, self.params[w], dx)

    def _drop(self, a: GpuTensor, i: int):
        pass

    def _dense_grads(self, x: GpuTensor, dy: GpuTensor, w: str, b: str):
        self.gpu.matmul_at_b(x, dy, self.grads[w])
        self.gpu.colsum(dy, self.grads[b], self._colsum)

    def backward(self, x: GpuTensor, labels: GpuTensor):
        """Gradients of the mean softmax cross-entropy of the last forward pass."""
        g, p, d = self.gpu, self.params, self.grads
        g.softmax_xent(self._logits, labels, self._delta, self._loss)
        self._dense_grads(self._h[-1], self._delta, "w_out", "b_out")
        self._dense_dx(self._delta, "w_out", self._dh)
        dz = None  # the last block's stream has no reader but the norm before the head
        for i in reversed(range(self.blocks)):
            g.block_backward(self._z[i + 1], y=self._y[i], post=self._post(i), gate=p[f"gate_{i}"], scale=self.scale,
                             pre=self._pre(i + 1), dz=dz, dh=self._dh, dr=self._dz, dy=self._dy,
                             dgamma_post=d[f"post_{i}"], dgamma_pre=d[f"pre_{i + 1}"], dgate=d[f"gate_{i}"],
                             work=self._work)
            dz = self._dz
            self._dense_grads(self._a[i], self._dy, f"w2_{i}", f"b2_{i}")
            self._dense_dx(self._dy, f"w2_{i}", self._da)
            self._drop(self._da, i)
            g.relu_bwd(self._a[i], self._da)
            self._dense_grads(self._h[i], self._da, f"w1_{i}", f"b1_{i}")
            self._dense_dx(self._da, f"w1_{i}", self._dh)
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


class TokenResidualMlp(ResidualMlp):
    """A ResidualMlp over a window of tokens: its input is their embeddings side
    by side, scaled by sqrt(embed); a place of the window without a token holds
    an index past the vocabulary and gives zeros.  While it trains, a share
    `dropout` of the embeddings and of every block's hidden activations is
    dropped.  products: "fp8" takes the Dense layers' three products in 8 bits
    (parameters, stream and gradients stay f32), "f32" as they are."""

    def __init__(self, gpu: Gpu, vocabulary: int, context: int, embed: int, width: int, hidden: int, classes: int,
                 blocks: int, batch: int, *, dropout: float = 0.1, products: str = "fp8", seed: int = 0, **kw):
        if embed % 4:
            raise ValueError("embed must be a multiple of 4: a window's embeddings lie side by side")
        if products not in ("fp8", "f32"):
            raise ValueError(f"unknown products {products!r}")
        super().__init__(gpu, context * embed, width, hidden, classes, blocks, batch, seed=seed, **kw)
        self.vocabulary, self.context, self.embed = vocabulary, context, embed
        self.dropout, self.seed, self.training, self.fp8 = dropout, seed, True, products == "fp8"
        table = np.random.default_rng(seed + 1).standard_normal((vocabulary, embed)).astype(np.float32) / np.sqrt(embed)
        self.params["embedding"] = gpu.upload(table)
        for held in (self.grads, self._m, self._v):
            held["embedding"] = gpu.zeros(table.shape)
        rows = batch * context
        self._x, self._dx = (gpu.zeros((rows, embed)) for _ in range(2))
        # the same memory as rows of the batch
        self._x_rows, self._dx_rows = (gpu.wrap(t.ptr, (batch, self.inputs)) for t in (self._x, self._dx))
        self._embedding_work = gpu.zeros((gpu.embedding_backward_workspace(rows, vocabulary, embed),))
        self._held = {}  # buffers of the 8-bit operands by layer, role and axis

    def _mask(self, site: int) -> Dropout:
        # the step that is under way: backward sees the same as forward
        return Dropout(self.dropout, self.seed, site=site, step=self.steps)

    def _drop(self, a: GpuTensor, i: int):
        if self.training and self.dropout:
            self.gpu.dropout(a, a, self._mask(1 + i))

    def _quantized(self, layer: str, role: str, t: GpuTensor, axis: int):
        """t in 8 bits, in the buffer of the layer's operand of that role."""
        key = (layer, role, axis)
        self._held[key] = self.gpu.fp8_quantize(t, self._held.get(key), axis=axis)
        return self._held[key]

    def _dense(self, x, w, b, y, relu=False):
        if not self.fp8:
            return super()._dense(x, w, b, y, relu)
        self.gpu.fp8_matmul(self._quantized(w, "x", x, 1), self._quantized(w, "w", self.params[w], 0), y, bias=self.params[b],
                            relu=relu)

    def _dense_dx(self, dy, w, dx):
        if not self.fp8:
            return super()._dense_dx(dy, w, dx)
        self.gpu.fp8_matmul(self._quantized(w, "dy", dy, 1), self._quantized(w, "w", self.params[w], 1), dx)

    def _dense_grads(self, x, dy, w, b):
        if not self.fp8:
            return super()._dense_grads(x, dy, w, b)
        self.gpu.fp8_matmul(self._quantized(w, "x", x, 0), self._quantized(w, "dy", dy, 0), self.grads[w])
        self.gpu.colsum(dy, self.grads[b], self._colsum)

    def forward(self, tokens: GpuTensor) -> GpuTensor:
        """Logits [batch, classes] of tokens, u32 [batch * context]."""
        g = self.gpu
        g.embedding_forward(self.params["embedding"], tokens, self._x, scale=float(np.sqrt(self.embed)))
        if self.training and self.dropout:
            g.dropout(self._x_rows, self._x_rows, self._mask(0))
        return super().forward(self._x_rows)

    def backward(self, tokens: GpuTensor, labels: GpuTensor):
        g = self.gpu
        super().backward(self._x_rows, labels)
        self._dense_dx(self._dz, "w_in", self._dx_rows)
        if self.training and self.dropout:
            g.dropout(self._dx_rows, self._dx_rows, self._mask(0))
        g.embedding_backward(tokens, self._dx, self.grads["embedding"], self._embedding_work,
                             scale=float(np.sqrt(self.embed)))

    def predict(self, tokens: np.ndarray) -> np.ndarray:
        """Classes of tokens [batch, context], without dropout."""
        was, self.training = self.training, False
        try:
            return self.gpu.download(self.forward(upload_labels(self.gpu, tokens.ravel()))).argmax(1)
        finally:
            self.training = was


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


def sentences(rows: int, context: int, vocabulary: int, seed: int):
    """Windows of a text in which a token is followed by one of three that depend
    on it and the one before, and the tokens that follow; places before the
    beginning hold the index `vocabulary`."""
    rng = np.random.default_rng(seed)
    t = np.full((rows, context + 1), vocabulary, np.int64)
    begin = rng.integers(0, context, rows)  # padding in front
    for j in range(context + 1):
        before, last = (t[:, j - k] % vocabulary if j >= k else np.zeros(rows, np.int64) for k in (2, 1))
        following = (7 * last + 3 * before + rng.integers(0, 3, rows)) % vocabulary
        t[:, j] = np.where(j < begin, vocabulary, np.where(j == begin, rng.integers(0, vocabulary, rows), following))
    return t[:, :-1].astype(np.uint32), t[:, -1].astype(np.uint32)


def main_tokens(steps: int = 300, vocabulary: int = 61):
    gpu = Gpu(0)
    models = {kind: TokenResidualMlp(gpu, vocabulary, context=8, embed=32, width=256, hidden=512, classes=vocabulary,
                                     blocks=3, batch=1024, scale=0.5, products=kind) for kind in ("f32", "fp8")}
    for step in range(steps):
        x, labels = sentences(1024, 8, vocabulary, step)
        for kind, model in models.items():
            model.step(upload_labels(gpu, x.ravel()), upload_labels(gpu, labels), 1e-3)
            if step % 60 == 0 or step == steps - 1:
                print(f"step {step}: {kind} products, loss {model.loss():.4f}")
    x, labels = sentences(1024, 8, vocabulary, 10**6)
    print("next token right (a third is what can be known): " +
          ", ".join(f"{kind} {np.mean(model.predict(x) == labels):.3f}" for kind, model in models.items()))


if __name__ == "__main__":
    import sys

    main_tokens() if sys.argv[1:] == ["tokens"] else main()
