"""The residual-block norms where they could go wrong unseen: no columns, values
that no norm touches, every row in the sums over rows, outputs in place, wide
rows in 4 bits."""
import numpy as np
import pytest

import rgpu_b200
from rgpu_b200 import gpu as G
from tests import ref_mx4 as R
from tests.test_gpu_block import Case, U, _backward, _near, _store, _sum_error

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def gpu():
    g = rgpu_b200.Gpu(0)
    yield g
    g.close()


@pytest.mark.parametrize("shape", [(1, 1), (3, 1)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradient_of_a_gate_over_no_columns_is_zero(gpu, dtype, shape):
    e = gpu.zeros((3, 0), dtype)
    gate, dgate = gpu.upload(np.ones(shape, np.float32)), gpu.upload(np.full(shape, 9.0, np.float32))
    work = gpu.zeros((max(1, gpu.block_backward_workspace(3, 0)),))
    gpu.block_backward(e, y=e, gate=gate, dz=e, dr=gpu.zeros((3, 0), dtype), dy=gpu.zeros((3, 0), dtype), dgate=dgate, work=work)
    assert not gpu.download(dgate).any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("gate", ["row", "column", "full"])
@pytest.mark.parametrize("post,pre", [("none", "rms"), ("rms", "none"), ("none", "layer"), ("none", "none")])
@pytest.mark.parametrize("m,n", [(5, 96), (5, 100), (4, 1000), (3, 8192), (3, 8200), (2, 12001), (2, 16400)])
def test_infinities_where_there_is_no_norm(gpu, m, n, post, pre, gate, dtype):
    # without a norm the gradient does not depend on the value: dr = dz + dh, dy = s g dr, whatever z and y are
    c = Case(gpu, m, n, dtype, post, pre, gate, seed=m + n)
    for name, kind in (("r", pre), ("y", post)):
        if kind == "none":
            x = c.host[name].copy()
            x[1, 3], x[0, n - 1], x[m - 1, n // 2] = np.inf, -np.inf, np.nan
            c._put(name, x, dtype)
    got = _backward(gpu, c, c.dev["r"], which=("dr", "dy"))
    with np.errstate(invalid="ignore"):
        want = R.block_backward(c.host["r"], c.host["y"], c.ref["post"], c.gate_ref, c.scale, c.ref["pre"], c.host["dz"],
                                c.host["dh"])
    e = 4 * _sum_error(n)
    if pre == "none":
        _near(got["dr"], want["dr"], _store(want["dr"], e * (np.abs(c.host["dz"]) + np.abs(c.host["dh"])), dtype), "dr")
    if post == "none":
        # dy is s g dr of dr before it is rounded: here against the reference's dr
        finite = np.isfinite(want["dy"])
        assert finite.all() and torch.isfinite(got["dy"]).all()
        if pre == "none":
            size = np.abs(c.scale * c.gate_ref) * (np.abs(c.host["dz"]) + np.abs(c.host["dh"]))
            _near(got["dy"], want["dy"], _store(want["dy"], e * size, dtype), "dy")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind,vectors", [("rms", "gamma"), ("layer", True)])
@pytest.mark.parametrize("m,n", [(9600, 96), (9601, 97), (9500, 504), (2400, 1000), (2401, 1001), (2500, 2048), (1300, 4096),
                                 (700, 8192), (301, 8200), (160, 12001), (301, 16400)])
def test_every_row_is_in_the_sums(gpu, m, n, kind, vectors, dtype):
    # A gradient of few rows a column: row r has nonzero entries in the columns j with (r + j) % step = 0, at least
    # three to a row and `terms` to a column: 64, or 3 m / n where that is more.  Zeros add without rounding, so a sum is
    # off by the roundings of its terms, and a row left out or taken twice is as much as one of them.
    step = max(1, min(n // 3, -(-m // 64)))
    here = (np.arange(m)[:, None] + np.arange(n)[None, :]) % step == 0
    terms = -(-m // step)
    rng = np.random.default_rng(m)
    sparse = np.where(here, np.where(rng.random((m, n)) < 0.5, -1.0, 1.0) * (0.5 + rng.random((m, n)) / 2), 0.0)
    for live, sums in (("dz", ["dgamma_post", "dgate"]), ("dh", ["dgamma_pre"])):
        c = Case(gpu, m, n, dtype, kind, kind, "row", seed=m + n, vectors=vectors)
        for name in ("dz", "dh"):
            c._put(name, sparse if name == live else np.zeros((m, n)), dtype)
        which = sums + (["dbeta" + sums[0][6:]] if vectors is True else [])
        got = _backward(gpu, c, c.dev["r"], which=which)
        want = R.block_backward(c.host["r"], c.host["y"], c.ref["post"], c.gate_ref, c.scale, c.ref["pre"], c.host["dz"],
                                c.host["dh"])
        want["dgate"] = want["dgate"].sum(0, keepdims=True)

        def hat(x, norm):
            mu, rho = R._stat(x, *norm[:2])
            return (np.abs(x) + np.abs(mu)) * rho

        d = np.abs(c.host[live])
        s, g = abs(c.scale), np.abs(c.gate_ref)
        size = {"dgamma_pre": d * hat(c.host["r"], c.ref["pre"]), "dbeta_pre": d,
                "dgamma_post": s * g * d * hat(c.host["y"], c.ref["post"]), "dbeta_post": s * g * d,
                "dgate": s * d * (hat(c.host["y"], c.ref["post"]) * np.abs(c.ref["post"][2]) + np.abs(c.ref["post"][3]))}
        for k in which:
            tol = 4 * (2 * _sum_error(n) + (terms + 40) * U) * size[k].sum(0, keepdims=True) + 1e-30
            if k.startswith("dbeta"):  # no y^ that may be small: each row's part is far above the tolerance
                assert (tol < np.where(here, size[k], np.inf).min(0) / 4).all()
            _near(got[k], want[k], tol, k)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind,vectors,gate", [("layer", True, "full"), ("rms", "gamma", "row"), ("layer", True, "column")])
@pytest.mark.parametrize("m,n", [(5, 320), (9, 321), (150, 4104), (3, 8191), (40, 8200), (3, 16384), (3, 16400), (2, 20001)])
def test_gradient_of_the_stream_in_place(gpu, m, n, kind, vectors, gate, dtype):
    # dr written over dz is the dr written elsewhere, on every kernel; so are the others beside it
    c = Case(gpu, m, n, dtype, kind, kind, gate, seed=m + n, vectors=vectors)
    apart = _backward(gpu, c, c.dev["r"], which=("dr", "dy", "dgamma_pre"))
    dy, dyv = c.out()
    dgamma, dgv = c.out((1, n), "f32")
    gpu.block_backward(c.dev["r"], y=c.dev["y"], post=c.norms["post"], gate=c.dev["gate"], scale=c.scale, pre=c.norms["pre"],
                       dz=c.dev["dz"], dh=c.dev["dh"], dr=c.dev["dz"], dy=dy, dgamma_pre=dgamma,
                       work=gpu.zeros((gpu.block_backward_workspace(m, n),)))
    back, bv = c.out()
    gpu.cast(c.dev["dz"], back)
    gpu.sync()
    assert torch.equal(bv, apart["dr"]) and torch.equal(dyv, apart["dy"]) and torch.equal(dgv, apart["dgamma_pre"])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n", [(1, 16385), (3, 16416), (130, 16400), (2, 20001), (1, 33000)])
def test_wide_rows_in_4_bits_are_the_stored_ones_quantised(gpu, m, n, dtype):
    c = Case(gpu, m, n, dtype, "rms", "layer", "row", seed=n)
    args = dict(y=c.dev["y"], post=c.norms["post"], gate=c.dev["gate"], scale=c.scale, pre=c.norms["pre"])
    h, hv = c.out()
    q = gpu.mx4_zeros(m, n)
    cb, sb = rgpu_b200.Mx4Tensor.nbytes(m, n)
    codes = torch.full((cb,), 0xA5, dtype=torch.uint8, device="cuda")
    scales = torch.full((sb,), 0xFF, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    held = gpu.mx4_wrap(codes.data_ptr(), scales.data_ptr(), m, n)
    gpu.block_forward(c.dev["r"], h=h, hq=held, **args)
    gpu.mx4_quantize(h, q)
    a, b = gpu.zeros((m, n)), gpu.zeros((m, n))
    gpu.mx4_dequantize(held, a)
    gpu.mx4_dequantize(q, b)
    assert np.array_equal(gpu.download(a), gpu.download(b))
    # what the format fixes past the row's end: zero codes, no NaN scale
    blocks, groups = -(-n // 32), -(-n // 128)
    two = codes.cpu().numpy().reshape(m, -1)
    every = np.stack([two & 15, two >> 4], 2).reshape(m, -1)
    assert not np.any(every[:, n:] & 7)
    assert not np.any(R.untile_scales(scales.cpu().numpy(), m, groups * 4)[:, blocks:] == 255)


def test_a_vector_freed_after_the_norm_was_made_is_refused(gpu):
    # on the host, before any launch
    f, gamma, beta = gpu.zeros((4, 64)), gpu.zeros((1, 64)), gpu.zeros((1, 64))
    for vector in (gamma, beta):
        norm = rgpu_b200.Norm("layer", 1e-5, gamma if vector is gamma else None, beta if vector is beta else None)
        vector.free()
        before = gpu.launch_count()
        for call in (lambda: gpu.block_forward(f, pre=norm, h=f), lambda: gpu.block_backward(f, pre=norm, dh=f, dr=f)):
            with pytest.raises(rgpu_b200.RtError) as e:
                call()
            assert e.value.code == G.RT_ERR_INVALID and "after free" in str(e.value)
        assert gpu.launch_count() == before
