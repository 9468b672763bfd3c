"""Host-side rules of the 4-bit matrices and residual-block norms: sizes,
struct layouts, refusals that come before any device call."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import rgpu_b200
from rgpu_b200 import gpu as G
from tests import ref_mx4 as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("rows,k,codes,scales", [(0, 0, 0, 0), (1, 1, 16, 512), (128, 128, 128 * 64, 512),
                                                 (129, 129, 129 * 80, 4 * 512), (3, 32, 48, 512)])
def test_sizes(rows, k, codes, scales):
    assert rgpu_b200.Mx4Tensor.nbytes(rows, k) == (codes, scales)


def test_sizes_of_large_matrices_do_not_wrap():
    rows = k = (1 << 31) - 257
    codes, scales = rgpu_b200.Mx4Tensor.nbytes(rows, k)
    assert codes == rows * (-(-k // 32) * 16) and scales == -(-rows // 128) * -(-k // 128) * 512
    assert rgpu_b200.Mx4Tensor.nbytes(rows + 1, 1) == (-1, -1)
    assert rgpu_b200.Mx4Tensor.nbytes(-1, 1) == (-1, -1)


def test_structs_match_the_header(tmp_path):
    structs = {"rt_norm": G.NormArgs, "rt_block_args": G.BlockArgs, "rt_block_grads": G.BlockGrads}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "rtgpu.h"', "int main(void) {"]
    for name, py in structs.items():
        lines.append(f'printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in py._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["return 0; }"]))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "layout.c"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()
    got = {tuple(line.split()[:2]): int(line.split()[2]) for line in out}
    for name, py in structs.items():
        assert got[(name, "size")] == C.sizeof(py)
        assert all(got[(name, f)] == getattr(py, f).offset for f, _ in py._fields_)


def test_null_handles_are_refused():
    L = G.lib()
    assert L.rt_block_forward(None, None) == G.RT_ERR_INVALID
    assert L.rt_block_backward(None, None, None) == G.RT_ERR_INVALID
    assert L.rt_block_backward_workspace(None, 1, 1) == -1
    assert L.rt_mx4_matmul(None, None, None, None, None, 0) == G.RT_ERR_INVALID
    assert L.rt_mx4_quantize(None, None, 1, None) == G.RT_ERR_INVALID
    assert L.rt_mx4_dequantize(None, None, None) == G.RT_ERR_INVALID
    assert L.rt_mx4_zeros(None, 1, 1, None) == G.RT_ERR_INVALID
    assert L.rt_mx4_free(None) == G.RT_OK and L.rt_mx4_codes(None) is None


def test_reference_rounds_half_way_to_the_even_code():
    x = np.array([[4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.75, 7.9]])
    codes, scales = R.quantize(x)
    assert scales.tolist() == [[127]]
    assert R.values(codes, scales, 10).tolist() == [[4, 0, 1, 1, 2, 2, 4, 4, -1, 6]]
    assert np.array_equal(R.untile_scales(R.tile_scales(np.arange(130 * 5).reshape(130, 5) % 200), 130, 5),
                          np.arange(130 * 5).reshape(130, 5) % 200)


def test_reference_gradient_is_the_difference_quotient():
    # the formulas that the GPU is held to, against differences, on the CPU
    rng = np.random.default_rng(1)
    m, n, t = 3, 10, 1e-6
    r, y, cz, ch = (rng.standard_normal((m, n)) for _ in range(4))
    gate, gp, bp, gn, bn = (rng.standard_normal((1, n)) for _ in range(5))

    def loss(**v):
        w = dict(r=r, y=y, gate=gate, gp=gp, bp=bp, gn=gn, bn=bn) | v
        z, h = R.block_forward(w["r"], w["y"], ("layer", 1e-5, w["gp"], w["bp"]), w["gate"], 0.7, ("rms", 1e-5, w["gn"], w["bn"]))
        return (z * cz).sum() + (h * ch).sum()

    z, _ = R.block_forward(r, y, ("layer", 1e-5, gp, bp), gate, 0.7, ("rms", 1e-5, gn, bn))
    g = R.block_backward(z, y, ("layer", 1e-5, gp, bp), gate, 0.7, ("rms", 1e-5, gn, bn), cz, ch)
    g["dgate"] = g["dgate"].sum(0, keepdims=True)
    for name, grad, x in (("r", "dr", r), ("y", "dy", y), ("gate", "dgate", gate), ("gp", "dgamma_post", gp),
                          ("bp", "dbeta_post", bp), ("gn", "dgamma_pre", gn), ("bn", "dbeta_pre", bn)):
        way = rng.standard_normal(x.shape)
        slope = (loss(**{name: x + t * way}) - loss(**{name: x - t * way})) / (2 * t)
        assert abs(slope - (g[grad] * way).sum()) <= 1e-7 * (1 + np.abs(g[grad] * way).sum()), name
