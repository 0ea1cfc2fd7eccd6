"""The plan of a product's tiles (csrc/nt_plan.hpp) from Python: the header compiled by itself, for tests that have to
know which tile, splits and cut their sizes take."""
import ctypes as C
import functools
import os
import subprocess
import tempfile

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SMALL, MEDIUM, LARGE = range(3)
SOURCE = """
#include "nt_plan.hpp"
using namespace nt::tile;
extern "C" void plan_of(int64_t m, int64_t n, int64_t kb, int split, int64_t *out) {
    const Plan p = plan(m, n, kb, split != 0);
    out[0] = int64_t(p.size), out[1] = p.per, out[2] = p.splits;
}
extern "C" int64_t whole(int64_t m, int64_t n, int64_t kb) { return whole_rounds(m, n, kb); }
"""


@functools.lru_cache(None)
def _lib():
    folder = tempfile.mkdtemp()
    src, so = os.path.join(folder, "plan.cpp"), os.path.join(folder, "plan.so")
    with open(src, "w") as f:
        f.write(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, "noetic-tensor_amd", "csrc"), src,
                    "-o", so], check=True)
    lib = C.CDLL(so)
    lib.plan_of.argtypes = [C.c_int64, C.c_int64, C.c_int64, C.c_int, C.POINTER(C.c_int64)]
    lib.plan_of.restype = None
    lib.whole.argtypes, lib.whole.restype = [C.c_int64] * 3, C.c_int64
    return lib


def plan(m, n, kb, split):
    """(tile, bytes of k of a split, splits) of [m, k] x [n, k], kb bytes of k."""
    out = (C.c_int64 * 3)()
    _lib().plan_of(m, n, kb, int(split), out)
    return tuple(out)


def whole_rounds(m, n, kb):
    return _lib().whole(m, n, kb)


def int8_product(m, n, k):
    """How the 8-bit product of more than four rows goes."""
    size, _, splits = plan(m, n, (k + 15) // 16 * 16, True)
    return size, splits


def readout(rows, V, d, layout):
    """How the readout's products go, for operands read in place and a G in one piece: (pass over the logits, its columns in
    whole rounds; dH's tile and splits; dW's tile, splits and columns in whole rounds)."""
    kp = (d + 7) // 8 * 8
    wide = (V + 7) // 8 * 8
    assert (V + 255) // 256 * 256 * rows <= 1 << 28
    logits = plan(rows, V, kp * 2, False)[0], whole_rounds(rows, V, kp * 2)
    hidden = plan(rows, d, wide * 2, True)
    shape = (d, V) if layout == "dv" else (V, d)
    weight = plan(*shape, rows * 2, True)
    cut = 0 if weight[2] > 1 else whole_rounds(d, V, rows * 2)
    return logits, (hidden[0], hidden[2]), (weight[0], weight[2], cut)
