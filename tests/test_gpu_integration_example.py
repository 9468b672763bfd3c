"""The integration guide's example of a window of tokens, run as it is written."""
import os
import re

import numpy as np
import pytest

import rgpu_b200
from tests import ref_tokens as R
from tests.test_gpu_fp8 import gpu  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu

GUIDE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "INTEGRATION.md")


@pytest.mark.parametrize("embed", [32, 30, 7])
def test_a_window_of_tokens(gpu, embed):
    code, = [c for c in re.findall(r"```python\n(.*?)```", open(GUIDE).read(), re.S) if "embedding_forward" in c]
    batch, context, vocabulary, units, seed, step = 5, 3, 20, 16, 12, 4
    rng = np.random.default_rng(embed)
    e = rng.standard_normal((vocabulary, embed)).astype(np.float32)
    tokens = rng.integers(0, vocabulary + 3, batch * context).astype(np.uint32)
    w = rng.standard_normal((context * embed, units)).astype(np.float32)
    names = dict(gpu=gpu, rgpu_b200=rgpu_b200, batch=batch, context=context, embed=embed, seed=seed, step=step,
                 table=gpu.upload(e), tokens=rgpu_b200.upload_labels(gpu, tokens), w=gpu.upload(w), b=gpu.zeros((1, units)),
                 out=gpu.zeros((batch, units)))
    exec(code, names)
    # each step rounded once, as the operators state it
    looked_up = R.embedding(e.astype(np.float64), tokens, np.float64(np.float32(embed ** 0.5))).astype(np.float32)
    kept, share = R.keep(batch, context * embed, 0.1, seed, site=0, step=step)
    x = np.where(kept, looked_up.reshape(batch, -1) * np.float32(1 / share), np.float32(0))
    assert np.array_equal(gpu.download(names["x"]), x)
    qx, qw = (R.values(*R.quantize(a), context * embed) for a in (x, w.T))
    want = np.maximum(qx @ qw.T, 0)
    # an f32 sum of context * embed products, in any order
    assert np.all(np.abs(gpu.download(names["out"]) - want) <= (context * embed + 1) * 2.0 ** -24 * (np.abs(qx) @ np.abs(qw.T)))
