"""The residual-block norms (forward and backward) against numpy in 64 bits
and against differences."""
import numpy as np
import pytest

import rgpu_b200
from rgpu_b200 import gpu as G
from tests import ref_mx4 as R

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -24
B = 2.0 ** -8  # unit roundoff of bf16's 8 bits
EPS = 1e-5


@pytest.fixture(scope="module")
def gpu():
    g = rgpu_b200.Gpu(0)
    yield g
    g.close()


class Case:
    """Inputs on the host (as the device holds them) and on the device."""

    def __init__(self, gpu, m, n, dtype, post, pre, gate, scale=0.5, seed=0, pad=0, offset=0, vectors=True):
        self.gpu, self.m, self.n, self.dtype, self.pad, self.offset = gpu, m, n, dtype, pad, offset
        self.scale, self.kinds, self.keep = scale, (post, pre), []
        rng = np.random.default_rng(seed)
        self.host, self.dev = {}, {}
        for name, std, mean in (("y", 0.8, 0.2), ("r", 1.5, -0.1), ("dz", 0.1, 0.0), ("dh", 0.1, 0.02)):
            self._put(name, rng.standard_normal((m, n)) * std + mean, dtype)
        shape = {"none": None, "one": (1, 1), "row": (1, n), "column": (m, 1), "full": (m, n)}[gate]
        if shape:
            self._put("gate", rng.standard_normal(shape) * 0.3 + 0.6, dtype if gate == "full" else "f32")
        self.norms, self.ref = {}, {}
        for name, kind in (("post", post), ("pre", pre)):
            g = b = None
            if vectors and kind != "none":
                g = self._put("gamma_" + name, rng.standard_normal((1, n)) * 0.2 + 1.0, "f32")
                if vectors != "gamma":
                    b = self._put("beta_" + name, rng.standard_normal((1, n)) * 0.1, "f32")
            self.norms[name] = rgpu_b200.Norm(kind, EPS, g, b)
            self.ref[name] = (kind, EPS, self.host.get("gamma_" + name, np.ones((1, n))),
                              self.host.get("beta_" + name, np.zeros((1, n))))
        self.gate_ref = self.host.get("gate", np.ones((1, 1)))

    def _device(self, shape, dtype):
        t = torch.bfloat16 if dtype == "bf16" else torch.float32
        pad = self.pad if shape[1] == self.n and shape[0] > 1 else 0
        ld = shape[1] + pad
        off = self.offset if shape[1] == self.n else 0
        buf = torch.full((off + shape[0] * ld + 8,), float("nan"), dtype=t, device="cuda")
        view = buf[off:off + shape[0] * ld].view(shape[0], ld)[:, :shape[1]]
        torch.cuda.synchronize()
        self.keep.append(buf)
        return self.gpu.wrap(buf.data_ptr() + off * buf.element_size(), shape, dtype, ld), view

    def _put(self, name, x, dtype):
        h, view = self._device(x.shape, dtype)
        view.copy_(torch.from_numpy(x.astype(np.float32)))
        torch.cuda.synchronize()
        self.host[name] = view.double().cpu().numpy()
        self.dev[name] = h
        return h

    def out(self, shape=None, dtype=None):
        return self._device(shape or (self.m, self.n), dtype or self.dtype)


def _near(got, want, tol, what):
    got = got.double().cpu().numpy()
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} outside, worst by {np.max((np.abs(got - want) / tol)[bad]):.2f}x"


def _store(want, tol, dtype):
    return tol + (B * (np.abs(want) + tol) if dtype == "bf16" else 0.0)


def _sum_error(n):
    """Relative error of a sum of n magnitudes taken in at least 32 strands and joined in a tree, and of what follows."""
    return (n / 32 + 40) * U


def _forward_tolerance(c, z, h):
    """First-order error of z and h: the statistics' relative error times the size of what they scale."""
    e = _sum_error(c.n)
    kind, eps, gamma, beta = c.ref["post"]
    mu, rho = R._stat(c.host["y"], kind, eps)
    size_u = (np.abs(c.host["y"]) + np.abs(c.host["y"]).mean(1, keepdims=True)) * rho * np.abs(gamma) * 2 + np.abs(beta)
    tz = e * (np.abs(c.host["r"]) + abs(c.scale) * np.abs(c.gate_ref) * size_u + np.abs(z))
    kind, eps, gamma, beta = c.ref["pre"]
    mu, rho = R._stat(z, kind, eps)
    big = np.abs(z) + np.abs(z).mean(1, keepdims=True) if kind != "none" else np.abs(z)
    th = (tz + tz.mean(1, keepdims=True) + e * big * 2) * rho * np.abs(gamma) * 2 + e * (np.abs(h) + np.abs(beta))
    return tz, th


SHAPES = [(1, 1), (1, 32), (2, 33), (3, 64), (5, 100), (8, 127), (9, 256), (4, 1000), (17, 1024), (3, 2049), (33, 4096),
          (2, 8192), (3, 8200), (2, 16384), (2, 20001), (301, 96), (700, 512)]
KINDS = [("rms", "rms"), ("layer", "layer"), ("none", "rms"), ("layer", "none")]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("post,pre", KINDS)
@pytest.mark.parametrize("m,n", SHAPES)
def test_forward(gpu, m, n, post, pre, dtype):
    gates = ["none", "one", "row", "column", "full"]
    for i, (pad, offset) in enumerate(((0, 0), (3, 1))):
        c = Case(gpu, m, n, dtype, post, pre, gates[(m + n + i) % 5], seed=m * n + i, pad=pad, offset=offset)
        z, zv = c.out()
        h, hv = c.out()
        gpu.block_forward(c.dev["r"], y=c.dev["y"], post=c.norms["post"], gate=c.dev.get("gate"), scale=c.scale, z=z,
                          pre=c.norms["pre"], h=h)
        gpu.sync()
        wz, wh = R.block_forward(c.host["r"], c.host["y"], c.ref["post"], c.gate_ref, c.scale, c.ref["pre"])
        tz, th = _forward_tolerance(c, wz, wh)
        _near(zv, wz, _store(wz, tz, dtype), "z")
        _near(hv, wh, _store(wh, th, dtype), "h")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("m,n", [(9600, 96), (9500, 504), (2400, 1000), (2500, 2048), (1300, 2056), (600, 4104), (601, 8192)])
def test_many_rows(gpu, m, n, kind, dtype):
    for gate in ("row", "column") if n < 4000 else ("full" if kind == "layer" else "one",):
        c = Case(gpu, m, n, dtype, kind, kind, gate, seed=m + n, pad=8)
        z, zv = c.out()
        h, hv = c.out()
        q = gpu.mx4_zeros(m, n)
        gpu.block_forward(c.dev["r"], y=c.dev["y"], post=c.norms["post"], gate=c.dev.get("gate"), scale=c.scale, z=z,
                          pre=c.norms["pre"], h=h, hq=q)
        wz, wh = R.block_forward(c.host["r"], c.host["y"], c.ref["post"], c.gate_ref, c.scale, c.ref["pre"])
        gpu.sync()
        tz, th = _forward_tolerance(c, wz, wh)
        _near(zv, wz, _store(wz, tz, dtype), "z")
        _near(hv, wh, _store(wh, th, dtype), "h")
        a, b = gpu.zeros((m, n)), gpu.zeros((m, n))
        gpu.mx4_dequantize(q, a)
        gpu.mx4_dequantize(gpu.mx4_quantize(h), b)
        assert np.array_equal(gpu.download(a), gpu.download(b))
        if gate != "full":
            _backward_check(c, c.host["r"], _backward(gpu, c, c.dev["r"]), dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n", [(1, 8), (3, 96), (2400, 104), (700, 504), (1000, 1000), (1300, 2048), (700, 4096), (450, 4104),
                                 (299, 8192)])
def test_rms_training_step(gpu, m, n, dtype):
    # two RMS norms without betas and a gate that rows share: rows overlap in the backward pass
    for gate in ("none", "one", "row"):
        c = Case(gpu, m, n, dtype, "rms", "rms", gate, seed=m + n, vectors="gamma" if gate != "none" else False)
        which = ("dr", "dy", "dgamma_post", "dgamma_pre", "dgate")
        got = _backward(gpu, c, c.dev["r"], which=which)
        _backward_check(c, c.host["r"], got, dtype)
        some = _backward(gpu, c, c.dev["r"], which=("dr",))
        assert torch.equal(some["dr"], got["dr"])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind,vectors", [("layer", True), ("rms", "gamma")])
@pytest.mark.parametrize("m,n,pad", [(150, 5001, 0), (3, 8190, 0), (9, 8191, 1), (300, 1003, 0), (5, 12001, 0), (2, 16384, 0)])
def test_wide_and_odd_rows(gpu, m, n, pad, kind, vectors, dtype):
    for gate in ("row", "full") if vectors is True else ("row",):
        c = Case(gpu, m, n, dtype, kind, kind, gate, seed=m + n, vectors=vectors, pad=pad)
        which = None if vectors is True else ("dr", "dy", "dgamma_post", "dgamma_pre", "dgate")
        _backward_check(c, c.host["r"], _backward(gpu, c, c.dev["r"], which=which), dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind,vectors", [("layer", True), ("rms", "gamma"), ("none", False)])
@pytest.mark.parametrize("m,n", [(160, 4104), (76, 8192), (1, 8200), (90, 9000), (150, 16384), (41, 10003), (2, 16392), (3, 20001)])
def test_rows_of_several_thread_blocks(gpu, m, n, kind, vectors, dtype):
    # 4096 or 8192 columns to a thread block in the backward pass
    for gate in ("column", "full") if vectors is True else ("row",):
        c = Case(gpu, m, n, dtype, kind, kind, gate, seed=m + n, vectors=vectors)
        which = None if vectors is True else ("dr", "dy", "dgamma_post", "dgamma_pre", "dgate") if vectors else ("dr", "dy", "dgate")
        _backward_check(c, c.host["r"], _backward(gpu, c, c.dev["r"], which=which), dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("gate", ["none", "one", "row", "column", "full"])
def test_every_gate_and_in_place(gpu, gate, dtype):
    c = Case(gpu, 19, 320, dtype, "layer", "rms", gate, seed=4)
    z, zv = c.out()
    args = dict(y=c.dev["y"], post=c.norms["post"], gate=c.dev.get("gate"), scale=c.scale, pre=c.norms["pre"])
    h, hv = c.out()
    gpu.block_forward(c.dev["r"], z=z, h=h, **args)
    wz, wh = R.block_forward(c.host["r"], c.host["y"], c.ref["post"], c.gate_ref, c.scale, c.ref["pre"])
    gpu.sync()
    tz, th = _forward_tolerance(c, wz, wh)
    _near(zv, wz, _store(wz, tz, dtype), "z")
    _near(hv, wh, _store(wh, th, dtype), "h")
    h2, h2v = c.out()
    gpu.block_forward(c.dev["r"], z=c.dev["r"], h=h2, **args)  # the stream updated in place
    z2, z2v = c.out()
    gpu.cast(c.dev["r"], z2)
    gpu.sync()
    assert torch.equal(z2v, zv) and torch.equal(h2v, hv)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n", [(1, 32), (3, 100), (130, 96), (5, 1000), (2, 8192), (2, 9000)])
def test_quantised_output_is_the_stored_one_quantised(gpu, m, n, dtype):
    for pad in (0, 3):
        c = Case(gpu, m, n, dtype, "rms", "layer", "row", seed=n, pad=pad)
        args = dict(y=c.dev["y"], post=c.norms["post"], gate=c.dev["gate"], scale=c.scale, pre=c.norms["pre"])
        h, hv = c.out()
        z, zv = c.out()
        z2, z2v = c.out()
        q = gpu.mx4_zeros(m, n)
        gpu.block_forward(c.dev["r"], z=z, h=h, **args)
        gpu.block_forward(c.dev["r"], z=z2, hq=q, **args)
        want = gpu.mx4_quantize(h)
        a, b = gpu.zeros((m, n)), gpu.zeros((m, n))
        gpu.mx4_dequantize(q, a)
        gpu.mx4_dequantize(want, b)
        assert np.array_equal(gpu.download(a), gpu.download(b))
        assert torch.equal(zv, z2v)


def test_no_block_before(gpu):
    c = Case(gpu, 6, 200, "f32", "none", "rms", "none", vectors=False)
    h, hv = c.out()
    gpu.block_forward(c.dev["r"], pre=c.norms["pre"], h=h)
    gpu.sync()
    _near(hv, R.norm(c.host["r"], *c.ref["pre"]), 2 * _sum_error(200) * (1 + np.abs(c.host["r"])), "h")
    dr, drv = c.out()
    gpu.block_backward(c.dev["r"], pre=c.norms["pre"], dh=c.dev["dh"], dr=dr)
    gpu.sync()
    want = R.block_backward(c.host["r"], None, None, None, 1.0, c.ref["pre"], 0.0, c.host["dh"])["dr"]
    _near(drv, want, 8 * _sum_error(200) * (1 + np.abs(want)), "dr")


def test_a_row_of_zeros_is_finite(gpu):
    for kind in ("rms", "layer"):
        c = Case(gpu, 4, 96, "f32", kind, kind, "none")
        zero = gpu.zeros((4, 96))
        z, zv = c.out()
        h, hv = c.out()
        gpu.block_forward(zero, y=zero, post=c.norms["post"], scale=1.0, z=z, pre=c.norms["pre"], h=h)
        dr, drv = c.out()
        dy, dyv = c.out()
        gpu.block_backward(z, y=zero, post=c.norms["post"], scale=1.0, pre=c.norms["pre"], dh=c.dev["dh"], dr=dr, dy=dy)
        gpu.sync()
        assert all(torch.isfinite(t).all() for t in (zv, hv, drv, dyv))


def _backward(gpu, c, z, which=None, dz=True, dh=True):
    """Every gradient that the case has, by name."""
    gate = c.dev.get("gate")
    shapes = {"dr": None, "dy": None}
    for v in ("post", "pre"):
        if c.norms[v].kind != "none" and (dh or v == "post"):
            shapes["dgamma_" + v] = shapes["dbeta_" + v] = (1, c.n)
    if gate is not None:
        shapes["dgate"] = gate.shape
    out, views = {}, {}
    for k, s in shapes.items():
        if which is None or k in which:
            t = c.dtype if s is None else "bf16" if k == "dgate" and gate.dtype_code == G.RT_BF16 else "f32"
            out[k], views[k] = c.out(s, t)
    work = gpu.zeros((gpu.block_backward_workspace(c.m, c.n),))
    gpu.block_backward(z, y=c.dev["y"], post=c.norms["post"], gate=gate, scale=c.scale, pre=c.norms["pre"],
                       dz=c.dev["dz"] if dz else None, dh=c.dev["dh"] if dh else None, work=work, **out)
    gpu.sync()
    return views


def _backward_check(c, z, got, dtype, dz=True, dh=True):
    zero = np.zeros((c.m, c.n))
    want = R.block_backward(z, c.host["y"], c.ref["post"], c.gate_ref, c.scale, c.ref["pre"],
                            c.host["dz"] if dz else zero, c.host["dh"] if dh else zero)
    e = 2 * _sum_error(c.n)

    def size_back(x, norm, d):
        """Size of the terms that a norm's gradient adds up, which may cancel: |a| + mean|a| + |x^| mean|a x^|."""
        mu, rho = R._stat(x, *norm[:2])
        hat = (np.abs(x) + np.abs(mu)) * rho
        a = np.abs(d * norm[2])
        if norm[0] == "none":
            return a, hat
        return (a + a.mean(1, keepdims=True) + hat * (a * hat).mean(1, keepdims=True)) * rho, hat

    size_r, hat_z = size_back(z, c.ref["pre"], c.host["dh"] if dh else zero)
    size_r = size_r + (np.abs(c.host["dz"]) if dz else 0)
    dt = abs(c.scale) * size_r
    du = dt * np.abs(c.gate_ref)
    size_y, hat_y = size_back(c.host["y"], c.ref["post"], du)
    size_u = hat_y * np.abs(c.ref["post"][2]) + np.abs(c.ref["post"][3])
    sizes = {"dr": size_r, "dy": size_y, "dgate": dt * size_u}
    rows = e + (c.m + 40) * U  # and a sum over the rows
    sums = {"dgamma_pre": np.abs(c.host["dh"]) * hat_z, "dbeta_pre": np.abs(c.host["dh"]), "dgamma_post": du * hat_y,
            "dbeta_post": du}
    sizes |= {k: v.sum(0, keepdims=True) for k, v in sums.items()}
    for k, v in got.items():
        w, s, t = want[k], sizes[k], e
        if k == "dgate":
            shape = tuple(v.shape)
            axes = tuple(i for i in (0, 1) if shape[i] == 1 and w.shape[i] != 1)
            w, s = w.sum(axes, keepdims=True), s.sum(axes, keepdims=True)
            t = rows + (c.n + 40) * U
        elif k[1] in "bg":
            t = rows
        bf16 = v.dtype == torch.bfloat16
        _near(v, w, _store(w, 4 * t * s + 1e-30, "bf16" if bf16 else "f32"), k)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("post,pre", KINDS)
@pytest.mark.parametrize("m,n", SHAPES)
def test_backward(gpu, m, n, post, pre, dtype):
    gates = ["none", "one", "row", "column", "full"]
    for i, (pad, offset) in enumerate(((0, 0), (3, 1))):
        c = Case(gpu, m, n, dtype, post, pre, gates[(m + n + i) % 5], seed=m + n + i, pad=pad, offset=offset)
        _backward_check(c, c.host["r"], _backward(gpu, c, c.dev["r"]), dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("gate", ["none", "one", "row", "column", "full"])
def test_backward_of_every_gate(gpu, gate, kind, dtype):
    for vectors in (True, False):
        c = Case(gpu, 37, 264, dtype, kind, kind, gate, seed=9, vectors=vectors)
        _backward_check(c, c.host["r"], _backward(gpu, c, c.dev["r"]), dtype)


def test_each_gradient_alone_and_without_dz_or_dh(gpu):
    c = Case(gpu, 21, 160, "f32", "layer", "rms", "row", seed=3)
    every = _backward(gpu, c, c.dev["r"])
    for k in every:
        assert torch.equal(_backward(gpu, c, c.dev["r"], which=(k,))[k], every[k]), k
    _backward_check(c, c.host["r"], _backward(gpu, c, c.dev["r"], dz=False), "f32", dz=False)
    _backward_check(c, c.host["r"], _backward(gpu, c, c.dev["r"], dh=False), "f32", dh=False)


def test_backward_of_no_rows_gives_zero_vectors(gpu):
    c = Case(gpu, 0, 64, "f32", "layer", "layer", "row")
    got = _backward(gpu, c, c.dev["r"], which=("dgamma_post", "dbeta_post", "dgamma_pre", "dbeta_pre", "dgate"))
    assert len(got) == 5 and all(not v.any() for v in got.values())


def test_backward_in_place_and_the_same_every_time(gpu):
    c = Case(gpu, 333, 520, "bf16", "rms", "rms", "one", seed=6)
    first, again = _backward(gpu, c, c.dev["r"]), _backward(gpu, c, c.dev["r"])
    assert all(torch.equal(first[k], again[k]) for k in first)
    gpu.block_backward(c.dev["r"], y=c.dev["y"], post=c.norms["post"], gate=c.dev["gate"], scale=c.scale,
                       pre=c.norms["pre"], dz=c.dev["dz"], dh=c.dev["dh"], dr=c.dev["dz"])
    back, bv = c.out()
    gpu.cast(c.dev["dz"], back)
    gpu.sync()
    assert torch.equal(bv, first["dr"])


@pytest.mark.parametrize("gate", ["one", "row", "column", "full"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_backward_against_differences(gpu, kind, gate):
    # d/dt of sum(z cz + h ch) along a random direction of every input, by central differences in 64 bits
    c = Case(gpu, 5, 72, "f32", kind, kind, gate, seed=11)
    host = {k: v.copy() for k, v in c.host.items()}

    def forward(h):
        post = (kind, EPS, h["gamma_post"], h["beta_post"])
        pre = (kind, EPS, h["gamma_pre"], h["beta_pre"])
        return R.block_forward(h["r"], h["y"], post, h["gate"], c.scale, pre)

    def loss(h):
        z, out = forward(h)
        return (z * host["dz"]).sum() + (out * host["dh"]).sum()

    z = c._put("z", forward(host)[0], "f32")
    got = {k: v.double().cpu().numpy() for k, v in _backward(gpu, c, z).items()}
    rng = np.random.default_rng(5)
    for name, grad in (("r", "dr"), ("y", "dy"), ("gate", "dgate"), ("gamma_post", "dgamma_post"),
                       ("beta_post", "dbeta_post"), ("gamma_pre", "dgamma_pre"), ("beta_pre", "dbeta_pre")):
        way = rng.standard_normal(host[name].shape)
        t = 1e-5
        lo, hi = dict(host), dict(host)
        lo[name], hi[name] = host[name] - t * way, host[name] + t * way
        slope = (loss(hi) - loss(lo)) / (2 * t)
        dot = (got[grad] * way).sum()
        # differences err by t^2 of a third derivative of order 1 and by 1e-16 / t; the gradient by f32 sums, and by
        # z rounded to f32 once
        tol = 1e-8 + 100 * U * np.abs(got[grad] * way).sum() + 100 * U
        assert abs(slope - dot) <= tol, f"{name}: {slope} against {dot}"


def test_refusals(gpu):
    f, b = gpu.zeros((4, 64)), gpu.zeros((4, 64), "bf16")
    v, rms = gpu.zeros((1, 64)), rgpu_b200.Norm("rms")
    work = gpu.zeros((gpu.block_backward_workspace(4, 64),))

    def refused(word, call, *a, **k):
        with pytest.raises(rgpu_b200.RtError) as e:
            call(*a, **k)
        assert e.value.code == G.RT_ERR_INVALID and word in str(e.value), str(e.value)

    fw, bw = gpu.block_forward, gpu.block_backward
    refused("no output", fw, f, pre=rms)
    refused("y must have r's type", fw, f, y=b, z=f)
    refused("h must have r's type", fw, f, pre=rms, h=b)
    refused("not 4x64", fw, f, pre=rms, h=gpu.zeros((4, 65)))
    refused("f32 or bf16", fw, gpu.zeros((4, 64), "u32"), pre=rms, h=f)
    refused("no y", fw, f, post=rms, h=f)
    refused("no y", fw, f, gate=v, h=f)
    refused("gamma must be f32", fw, f, pre=rgpu_b200.Norm("rms", 1e-5, gpu.zeros((1, 64), "bf16")), h=f)
    refused("not 1x64", fw, f, pre=rgpu_b200.Norm("rms", 1e-5, gpu.zeros((1, 63))), h=f)
    refused("eps", fw, f, pre=rgpu_b200.Norm("rms", -1.0), h=f)
    refused("no norm", fw, f, pre=rgpu_b200.Norm("none", 0.0, v), h=f)
    refused("it must be 1x1", fw, f, y=f, gate=gpu.zeros((2, 64)), z=f)
    refused("broadcast gate must be f32", fw, f, y=f, gate=b, z=f)
    refused("hq is", fw, f, pre=rms, hq=gpu.mx4_zeros(4, 32))
    refused("neither dz nor dh", bw, f, dr=f)
    refused("has no y", bw, f, dz=f, dy=f)
    refused("without a gate", bw, f, y=f, dz=f, dgate=v)
    refused("the gate's type and shape", bw, f, y=f, gate=v, dz=f, dgate=gpu.zeros((1, 1)), work=work)
    refused("not there", bw, f, y=f, dz=f, dgamma_post=v, work=work)
    refused("without dh", bw, f, y=f, pre=rms, dz=f, dgamma_pre=v, work=work)
    refused("work must be", bw, f, y=f, post=rms, dz=f, dgamma_post=v)
    refused("work must be", bw, f, y=f, post=rms, dz=f, dgamma_post=v, work=gpu.zeros((8,)))
    other = rgpu_b200.Gpu(0)
    refused("another context", fw, f, pre=rms, h=other.zeros((4, 64)))
    refused("another context", fw, f, pre=rms, hq=other.mx4_zeros(4, 64))
    refused("another context", bw, f, dz=f, dr=other.zeros((4, 64)))
    y = gpu.zeros((4, 64))
    y.free()
    refused("after free", fw, f, y=y, z=f)
