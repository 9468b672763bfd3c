"""Host-side rules of the 8-bit matrices, the embedding and dropout: sizes, struct
layouts, refusals that come before any device call, and the references that the GPU is
held to."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import rgpu_b200
from rgpu_b200 import gpu as G
from tests import ref_tokens as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("rows,k,codes,scales", [(0, 0, 0, 0), (1, 1, 16, 512), (128, 512, 128 * 512, 512),
                                                 (129, 513, 129 * 528, 4 * 512), (3, 128, 3 * 128, 512)])
def test_sizes(rows, k, codes, scales):
    assert rgpu_b200.Fp8Tensor.nbytes(rows, k) == (codes, scales)


def test_sizes_of_large_matrices_do_not_wrap():
    rows = k = (1 << 31) - 257
    codes, scales = rgpu_b200.Fp8Tensor.nbytes(rows, k)
    assert codes == rows * (-(-k // 16) * 16) and scales == -(-rows // 128) * -(-k // 512) * 512
    assert rgpu_b200.Fp8Tensor.nbytes(rows + 1, 1) == (-1, -1)
    assert rgpu_b200.Fp8Tensor.nbytes(1, -1) == (-1, -1)


def test_workspace():
    f = rgpu_b200.Gpu.embedding_backward_workspace
    assert f(0, 1, 1) > 0
    # two rows of partial sums for each 64 positions, four words a position, one a token
    assert f(1 << 20, 50257, 1024) >= (1 << 20) // 64 * 2 * 1024 + 4 * (1 << 20) + 50257
    for bad in ((-1, 1, 1), (1, -1, 1), (1, 1, -1), (1 << 31, 1, 1), (1, 1 << 31, 1)):
        with pytest.raises(rgpu_b200.RtError):
            f(*bad)
    assert f((1 << 31) - 1, (1 << 31) - 1, 8192) > 1 << 32


def test_struct_matches_the_header(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "rtgpu.h"', "int main(void) {",
             'printf("%zu\\n", sizeof(rt_dropout_mask));']
    lines += [f'printf("%zu\\n", offsetof(rt_dropout_mask, {f}));' for f, _ in G.DropoutMask._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["return 0; }"]))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "layout.c"), "-o", str(exe)], check=True)
    out = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert out == [C.sizeof(G.DropoutMask)] + [getattr(G.DropoutMask, f).offset for f, _ in G.DropoutMask._fields_]


def test_null_handles_are_refused():
    L = G.lib()
    assert L.rt_fp8_matmul(None, None, None, None, None, 0) == G.RT_ERR_INVALID
    assert L.rt_fp8_quantize(None, None, 1, None) == G.RT_ERR_INVALID
    assert L.rt_fp8_dequantize(None, None, None) == G.RT_ERR_INVALID
    assert L.rt_fp8_zeros(None, 1, 1, None) == G.RT_ERR_INVALID
    assert L.rt_fp8_wrap(None, None, None, 1, 1, None) == G.RT_ERR_INVALID
    assert L.rt_fp8_free(None) == G.RT_OK and L.rt_fp8_codes(None) is None and L.rt_fp8_scales(None) is None
    assert L.rt_embedding_forward(None, None, None, 1.0, None) == G.RT_ERR_INVALID
    assert L.rt_embedding_backward(None, None, None, 1.0, 0, None, None) == G.RT_ERR_INVALID
    assert L.rt_dropout(None, None, None, None, None) == G.RT_ERR_INVALID


def test_a_mask_is_held_to_its_fields_widths():
    assert rgpu_b200.Dropout(0.5, 2 ** 64 - 1, site=2 ** 32 - 1, step=2 ** 32 - 1, first_row=2 ** 32).seed == 2 ** 64 - 1
    for bad in (dict(seed=-1), dict(seed=1 << 64), dict(site=1 << 32), dict(step=-1), dict(step=1 << 32), dict(first_row=-1)):
        with pytest.raises(rgpu_b200.RtError):
            rgpu_b200.Dropout(**({"p": 0.5, "seed": 1} | bad))


def test_reference_generator_gives_the_published_answers():
    # the known answers that are published with the generator
    assert R.philox((0, 0, 0, 0), (0, 0)) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    assert R.philox((0xffffffff,) * 4, (0xffffffff,) * 2) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    assert R.philox((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0)) == \
        [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]


def test_reference_mask_drops_its_share():
    kept, share = R.keep(64, 200, 0.3, 0x1234567890abcdef, 3, 9)
    n = kept.size
    assert abs(kept.mean() - share) <= 5 * np.sqrt(share * (1 - share) / n)  # five standard deviations
    assert R.keep(2, 9, 0.0, 1)[0].all() and not R.keep(2, 9, 1.0, 1)[0].any()


def test_reference_rounds_half_way_to_the_even_code():
    # a block whose largest is 448 has scale 1
    x = np.zeros((1, 8))
    x[0] = [448.0, 17.0, 19.0, 1.0625, -1.1875, 2.0 ** -10, 3 * 2.0 ** -10, 432.0]
    codes, scales = R.quantize(x)
    assert scales.tolist() == [[127]]
    assert R.values(codes, scales, 8).tolist() == [[448, 16, 20, 1, -1.25, 0, 2 * 2.0 ** -9, 448]]
    assert R.quantize(np.array([[448.0001]]))[1].tolist() == [[128]]
    assert R.quantize(np.zeros((1, 1)))[1].tolist() == [[0]]
    assert R.quantize(np.array([[np.inf]]))[1].tolist() == [[255]]
    assert R.VALUES[126] == 448 and np.isnan(R.VALUES[127]) and R.VALUES[1] == 2.0 ** -9


def test_reference_gradient_is_the_difference_quotient():
    rng = np.random.default_rng(2)
    tokens = np.array([1, 3, 1, 7, 0, 3, 1])
    table, c = rng.standard_normal((5, 4)), rng.standard_normal((7, 4))
    way = rng.standard_normal(table.shape)
    t = 1e-6
    slope = ((R.embedding(table + t * way, tokens, 1.5) - R.embedding(table - t * way, tokens, 1.5)) * c).sum() / (2 * t)
    d, size, count = R.embedding_backward(5, tokens, c, 1.5)
    assert abs(slope - (d * way).sum()) <= 1e-8 * (size * np.abs(way)).sum()
    assert count.tolist() == [1, 3, 0, 2, 0]


def test_reference_model_gradient_is_the_difference_quotient():
    rng = np.random.default_rng(5)
    vocabulary, context, embed, width, hidden, batch = 6, 3, 4, 8, 10, 9
    shapes = {"embedding": (vocabulary, embed), "w_in": (context * embed, width), "b_in": (1, width),
              "w1_0": (width, hidden), "b1_0": (1, hidden), "w2_0": (hidden, width), "b2_0": (1, width),
              "post_0": (1, width), "gate_0": (1, width), "pre_0": (1, width), "pre_1": (1, width),
              "w_out": (width, 5), "b_out": (1, 5)}
    p = {k: rng.standard_normal(s) for k, s in shapes.items()}
    tokens, labels = rng.integers(0, vocabulary + 2, (batch, context)), rng.integers(0, 5, batch)
    masks = [(rng.random(s) < 0.7) / 0.7 for s in ((batch, context * embed), (batch, hidden))]
    _, g = R.token_model(p, tokens, labels, 1, 0.5, masks)
    assert sorted(g) == sorted(p)
    t = 1e-6
    for k in p:
        way = rng.standard_normal(p[k].shape)
        up, down = (R.token_model(p | {k: p[k] + s * t * way}, tokens, labels, 1, 0.5, masks)[0] for s in (1, -1))
        assert abs((up - down) / (2 * t) - (g[k] * way).sum()) <= 1e-6 * (1 + np.abs(g[k] * way).sum()), k
