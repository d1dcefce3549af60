"""What delta_step's kernel for many rows leaves behind where a wait runs out. Without a GPU: the branch as it stands in the source, compiled
for the host."""
import ctypes
import re
import shutil
import subprocess

import numpy as np
import pytest

from flyguy_b200 import native

SOURCE = (native.PKG / "csrc" / "fg_delta.cu").read_text()


def _block(opening):
    """The text between the braces that `opening` opens."""
    at = SOURCE.index(opening) + len(opening)
    depth, end = 1, at
    while depth:
        depth += {"{": 1, "}": -1}.get(SOURCE[end], 0)
        end += 1
    return SOURCE[at:end - 1]


HARNESS = """
#include <cstdint>
#include <cstring>
static int g_step_error;
static float __int_as_float(int x) { float f; memcpy(&f, &x, 4); return f; }
template <class T> T from_f(float x) { return x; }
static void atomicExch(int* to, int v) { *to = v; }
template <class T> void give_up(T* rows, int block, int blocks, int items, uint32_t i, int E) {
    constexpr int kWideThreads = 512;
    struct { int E; } s{E};
    const auto nth = [&](uint32_t i) { return block + i * blocks; };
    const auto out_of = [&](uint32_t item) { return rows + item * E; };
    for (int tid = 0; tid < kWideThreads; ++tid) {
        T* o = out_of(nth(i));
        (void)o;
        do { BRANCH } while (0);
    }
}
extern "C" int run(float* rows, int block, int blocks, int items, int i, int E) { give_up(rows, block, blocks, items, i, E); return g_step_error; }
"""


@pytest.mark.skipif(not shutil.which("g++"), reason="needs a host compiler")
def test_no_row_behind_a_wait_that_ran_out_looks_like_a_result(tmp_path):
    """The row that waited and all later ones of its block hold NaN; those of other blocks and earlier ones are left alone."""
    (tmp_path / "t.cpp").write_text(HARNESS.replace("BRANCH", _block("if (!workers(there)) {")))
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-o", str(tmp_path / "t.so"), str(tmp_path / "t.cpp")], check=True)
    lib = ctypes.CDLL(str(tmp_path / "t.so"))
    items, blocks, block, first, E = 23, 4, 2, 2, 600
    rows = np.zeros((items, E), np.float32)
    assert lib.run(ctypes.c_void_p(rows.ctypes.data), block, blocks, items, first, E) == 1
    gone = np.zeros(items, bool)
    gone[block + first * blocks::blocks] = True
    assert np.isnan(rows[gone]).all() and not rows[~gone].any()


def test_states_are_sent_off_for_longer_than_they_are_waited_for():
    """The warp that copies waits longer for the workers than they wait for a state: what they have worked on is stored."""
    tries = r"phase_of\(%s \+ 8 \* place, \(phases >> place\) & 1(?:, (\d+))?\)"
    workers = re.search("const bool there = " + tries % "full", SOURCE).group(1)
    copies = re.search(r"if \(!" + tries % "done", SOURCE).group(1)
    assert int(copies or 1) > int(workers or 1)
