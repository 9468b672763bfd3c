"""The residual-block norms at their edges."""
import numpy as np
import pytest

import rgpu_b200
from tests import ref_mx4 as R
from tests.test_gpu_block import Case, _backward, _near, _store, _sum_error

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
