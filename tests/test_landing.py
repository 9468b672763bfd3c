"""A kernel whose wait ran out waits for the copies that it still has on their way.
The rules of csrc/landing.cuh are held, on the host, to every order of issue and
every place to give up that the ring kernels and the two-CTA product have; how
the kernels call them is read from their source.  Nothing here runs on a GPU."""
import os
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rgpu_b200", "csrc")

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "landing.cuh"

// A ring's barriers as the thread that issues sees them.  A copy counts as landed only
// when a wait has waited for it.
struct Ring {
    std::vector<int> issued, landed;
    explicit Ring(int depth) : issued(depth), landed(depth) {}
    void wait(int slot, unsigned phase) {
        if ((landed[slot] & 1) != (int)phase) return;  // that phase is complete
        if (landed[slot] < issued[slot]) ++landed[slot];  // else: nothing issued, the limit ends it
    }
    int left() const {
        int n = 0;
        for (size_t i = 0; i < issued.size(); ++i) n += issued[i] - landed[i];
        return n;
    }
};

// forward_ring_kernel, backward_ring_kernel: gives up at its `stop`th wait.
int one_ring(int depth, int rows, int stop, int count) {
    Ring full(depth);
    for (int d = 0; d < depth && d < rows; ++d) ++full.issued[d];
    bool ok = true;
    int slot = 0, waits = 0, at = 0;
    unsigned phase = 0;
    for (int row = 0; row < rows; ++row) {
        if (waits++ == stop) {
            ok = false;
            at = slot * 2 + phase;
        } else if (ok) {
            full.wait(slot, phase);
        }
        if (ok && row + depth < rows) ++full.issued[slot];
        if (++slot == depth) slot = 0, phase ^= 1;
    }
    if (!ok) rt::land_ring(depth, count, at >> 1, at & 1, [&](int s, unsigned p) { full.wait(s, p); });
    return full.left();
}

// backward_pipe_kernel: z, y and dh in one ring, dz in another.
int two_rings(int depth, int rows, int stop, int count, int count_dz) {
    Ring full(depth), dz(depth);
    for (int d = 0; d < depth && d < rows; ++d) ++full.issued[d], ++dz.issued[d];
    bool ok = true;
    int slot = 0, waits = 0, at = 0;
    unsigned phase = 0;
    auto wait = [&](Ring& r, int s, unsigned p) {
        if (waits++ == stop) {
            ok = false;
            at = s * 2 + p;
        } else if (ok) {
            r.wait(s, p);
        }
    };
    wait(full, 0, 0);
    if (ok && depth < rows) ++full.issued[0];
    for (int row = 0; row < rows; ++row) {
        wait(dz, slot, phase);
        const int next = slot + 1 == depth ? 0 : slot + 1;
        const unsigned next_phase = next ? phase : phase ^ 1;
        if (row + 1 < rows) wait(full, next, next_phase);
        if (ok) {
            if (row + depth < rows) ++dz.issued[slot];
            if (row + depth + 1 < rows) ++full.issued[next];
        }
        slot = next;
        phase = next_phase;
    }
    if (!ok) {
        rt::land_ring(depth, count, at >> 1, at & 1, [&](int s, unsigned p) { full.wait(s, p); });
        rt::land_ring(depth, count_dz, at >> 1, at & 1, [&](int s, unsigned p) { dz.wait(s, p); });
    }
    return full.left() + dz.left();
}

// mx4_pair_kernel: a leader that issued `own` stages and a peer that issued `peer`; every
// copy lands.  Bytes count in halves of a stage.
int pair(int slots, int own, int peer) {
    const int last = own > peer ? own : peer;
    std::vector<int> arrived(last), bytes(last), waited(last);
    for (int i = 0; i < last; ++i) {
        if (i < own) ++arrived[i], bytes[i] += 2 - 1;  // announces both halves, brings its own
        if (i < peer) bytes[i] -= 1;
    }
    std::vector<int> phase(slots);  // of each barrier: the first stage not known to be complete
    auto current = [&](int slot) { return slot + phase[slot] * slots; };
    for (int s = 0; s < slots; ++s)
        while (current(s) < last - slots) ++phase[s];  // read by the MMAs, so complete
    rt::land_pair(slots, own, peer, [&](int s) { ++arrived[current(s)], bytes[current(s)] += 1; },
                  [&](int s) { bytes[current(s)] -= 1; },
                  [&](int s, unsigned p) {
                      const int i = current(s);
                      if ((unsigned)(phase[s] & 1) != p) return;
                      if (arrived[i] == 1 && bytes[i] == 0) ++waited[i], ++phase[s];
                  });
    int left = 0;
    for (int i = last > slots ? last - slots : 0; i < last; ++i) left += waited[i] != 1;
    return left;
}

int main(int, char** v) {
    const int extra = atoi(v[1]), extra_dz = atoi(v[2]);
    int bad = 0;
    for (int depth = 1; depth <= 4; ++depth)
        for (int rows = 0; rows < 20; ++rows)
            for (int stop = -1; stop <= 2 * rows; ++stop) {
                bad += one_ring(depth, rows, stop, depth) != 0;
                if (depth >= 2 && rows) bad += two_rings(depth, rows, stop, depth + extra, depth + extra_dz) != 0;
            }
    for (int slots : {4, 6})
        for (int own = 0; own < 25; ++own)
            for (int peer = own > slots ? own - slots : 0; peer <= own + slots; ++peer) bad += pair(slots, own, peer) != 0;
    printf("%d\n", bad);
}
"""


def _body(source, name):
    """Text of the kernel `name`."""
    text = open(os.path.join(CSRC, source)).read()
    start = re.search(r"__global__[^;{]*\b" + name + r"\(", text).start()
    return text[start:text.index("\n}\n", start)]


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("landing")
    (tmp / "landing.cc").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-I", CSRC, str(tmp / "landing.cc"), "-o", str(tmp / "landing")], check=True)
    return lambda *extra: int(subprocess.run([str(tmp / "landing"), *map(str, extra)], check=True, capture_output=True, text=True).stdout)


def _count(argument):
    """`depth + 1` as 1, `depth` as 0."""
    extra = argument.replace("r.depth", "depth").replace("depth", "0")
    assert re.fullmatch(r"0( \+ \d)?", extra), argument
    return int(extra.split("+")[-1])


def test_every_copy_of_a_run_that_gave_up_is_waited_for(check):
    calls = dict(re.findall(r"land_copies\((\w+), depth, ([^,]+),", _body("block_norm.cu", "backward_pipe_kernel")))
    assert sorted(calls) == ["full", "full_dz"]
    assert check(_count(calls["full"]), _count(calls["full_dz"])) == 0
    assert check(0, 0) > 0, "one round of each ring leaves the copy that follows the slot just read"
    for kernel in ("forward_ring_kernel", "backward_ring_kernel"):
        (count,) = re.findall(r"land_copies\(full, r\.depth, ([^,]+),", _body("block_norm.cu", kernel))
        assert _count(count) == 0


@pytest.mark.parametrize("kernel,barriers", [("mx4_kernel", ["done"]), ("mx4_pair_kernel", ["drain", "told"])])
def test_a_product_that_gave_up_waits_for_its_mmas_and_copies(kernel, barriers):
    body = _body("gemm_mx4.cu", kernel)
    for barrier in barriers:  # by a flag that nothing sets: the abort flag would end the wait at once
        flags = re.findall(r"mbar_wait\(smem_u32\(" + barrier + r"\), 0, ([^)]+)\)", body)
        assert flags and flags[-1] == "&never", (barrier, flags)
    assert body.rindex("&never") < body.rindex("tcgen05.dealloc")
    if kernel == "mx4_pair_kernel":
        assert "abort_flag" not in re.findall(r"mbar_wait\(smem_u32\(drain\), 0, ([^)]+)\)", body)
        assert re.search(r"land_pair\(\s*S, \*issued_all, both \? \*issued_peer : \*issued_all", body)
