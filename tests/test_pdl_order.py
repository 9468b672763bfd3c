"""Kernels that launch as programmatic dependents start while the kernel before them still
runs.  What that one, and those before it, wrote is visible only behind the wait, and what they
still read may be written only there.  So every thread of every such kernel of the token, 8-bit and
4-bit operators waits before it can return, and before it lets the kernel behind it launch."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rgpu_b200", "csrc")


UNCHANGING = r"__ldg|\.nc\b|const [\w:]+\s*\*\s*__restrict__"


def kernels(name, heads=False):
    """(name, body), with heads the text between the two too, of each __global__ function of a source file, comments taken out."""
    text = open(os.path.join(CSRC, name)).read()
    text = re.sub(r"//[^\n]*", "", text)
    for m in re.finditer(r"__global__", text):
        begin = text.index("{", m.end())
        # the parameters hold no braces
        what = re.findall(r"(\w+)\s*\(", re.sub(r"__launch_bounds__\((?:[^()]|\([^()]*\))*\)", "", text[m.end():begin]))[0]
        depth, end = 0, begin
        while True:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
            if depth == 0:
                break
        yield (what, text[begin + 1:end - 1]) + ((text[m.end():begin],) if heads else ())


@pytest.mark.parametrize("name,count", [("embedding.cu", 8), ("dropout.cu", 1), ("fp8.cu", 3), ("mx4.cu", 3), ("gemm_mx4.cu", 3)])
def test_every_kernel_waits_first(name, count):
    found = list(kernels(name))
    assert len(found) >= count, [k for k, _ in found]
    for what, body in found:
        at = body.find("pdl_wait();")
        assert at >= 0, f"{name}: {what} does not wait"
        before = body[:at]
        assert before.count("{") == before.count("}"), f"{name}: {what} waits on one of its paths only"
        assert "return" not in before and "launch_dependents" not in before, f"{name}: {what} waits too late"


@pytest.mark.parametrize("name", ["embedding.cu", "dropout.cu", "fp8.cu", "row_piece.cuh", "scaled.cuh", "mx4.cu", "mx4.cuh", "gemm_mx4.cu",
                                  "block_norm.cu", "gemm_simt.cu", "gemm_skinny.cu", "gemm_x3.cu", "gemm_tc2.cu", "tc_common.cuh"])
def test_no_load_needs_memory_that_never_changes(name):
    # ld.global.nc, which __ldg is and which a compiler may make of a restricted pointer to const, is for memory that
    # is not written for as long as the grid runs.  A dependent grid runs while the one before it writes what it reads.
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
    assert not re.findall(UNCHANGING, text)


def test_no_such_load_in_the_dependent_kernels_among_others():
    waiting = [(what, head, body) for what, body, head in kernels("elementwise.cu", heads=True) if "pdl_wait();" in body]
    assert {"xent_reg_kernel", "xent_kernel", "opt_step_begin_kernel"} <= {what for what, _, _ in waiting}
    for what, head, body in waiting:
        assert not re.findall(UNCHANGING, head + body), what
