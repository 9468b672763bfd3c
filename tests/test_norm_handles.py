"""A Norm holds tensors, not their handles: what a block call passes on is looked
up when the call is made.  No device is needed: the library is a stand-in that
records its arguments, the tensors carry made-up handles."""
import ctypes as C
import types

import pytest

from rgpu_b200 import gpu as G


class Tensor:
    def __init__(self, handle):
        self.handle = C.c_void_p(handle)

    def free(self):
        self.handle = C.c_void_p(0)  # as GpuTensor.free leaves it


@pytest.fixture
def calls(monkeypatch):
    seen = []

    def record(ctx, args, *rest):
        a = args._obj
        seen.append({n: (getattr(a, n).gamma, getattr(a, n).beta) for n in ("post", "pre")})
        return G.RT_OK

    fake = types.SimpleNamespace(rt_block_forward=record, rt_block_backward=record)
    monkeypatch.setattr(G, "lib", lambda: fake)
    return seen


def _forward(**norms):
    me = types.SimpleNamespace(handle=C.c_void_p(1))
    G.Gpu.block_forward(me, Tensor(2), y=Tensor(3), z=Tensor(4), h=Tensor(5), **norms)


def _backward(**norms):
    me = types.SimpleNamespace(handle=C.c_void_p(1))
    G.Gpu.block_backward(me, Tensor(2), y=Tensor(3), dz=Tensor(4), dh=Tensor(5), dr=Tensor(6), **norms)


@pytest.mark.parametrize("call", [_forward, _backward])
@pytest.mark.parametrize("which", ["gamma", "beta"])
@pytest.mark.parametrize("place", ["post", "pre"])
def test_a_vector_freed_after_the_norm_was_made_is_refused(calls, place, which, call):
    norm = G.Norm("layer", 1e-5, Tensor(16), Tensor(32))
    call(**{place: norm})
    assert calls == [{place: (16, 32), ("pre" if place == "post" else "post"): (None, None)}]
    getattr(norm, which).free()
    with pytest.raises(G.RtError) as e:
        call(**{place: norm})
    assert e.value.code == G.RT_ERR_INVALID and "after free" in str(e.value)
    assert len(calls) == 1, "nothing was handed to the library"


def test_a_vector_put_in_later_is_the_one_that_is_passed(calls):
    norm = G.Norm("rms", 1e-5, Tensor(16))
    norm.gamma, norm.beta = Tensor(48), Tensor(64)
    _forward(pre=norm)
    norm.beta = None
    _forward(pre=norm)
    assert [c["pre"] for c in calls] == [(48, 64), (48, None)]


def test_a_vector_freed_before_the_norm_is_made_is_refused():
    gamma = Tensor(16)
    gamma.free()
    with pytest.raises(G.RtError):
        G.Norm("rms", 1e-5, gamma)
