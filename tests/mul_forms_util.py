"""The choice between the int8 product's forms (aubier_amd/csrc/mul_i8_forms.h), compiled for the host."""
import ctypes
import functools
import shutil
import subprocess
import tempfile
from pathlib import Path

from aubier_amd import build as B

NAMES = "DIRECT8 DIRECT8_2 SPLIT11 SPLIT12 SPLIT22 SPLIT32 SPLIT128 TILE128 TILE192 TILE256".split()
SHIM = """
#include "mul_i8_forms.h"
using namespace mla::rows;
static_assert(TILE256 == %d && sizeof(FORMS) / sizeof(FORMS[0]) == %d, "the names that the tests use");
extern "C" int form_of(int rows, int n, int k, int may_cut, int * parts, int64_t * work) {
    const Choice c = choose(n, k, rows, may_cut != 0);
    *parts = c.n_split;
    *work = c.work;
    return c.kind;
}
extern "C" int form(int i, int * bn, int * bm, int * cuts) {
    *bn = FORMS[i].bn;
    *bm = FORMS[i].bm;
    *cuts = FORMS[i].cut != 0.f;
    return FORMS[i].kind;
}
""" % (len(NAMES) - 1, len(NAMES))

there = shutil.which("g++") is not None


@functools.lru_cache(None)
def _lib():
    with tempfile.TemporaryDirectory() as d:
        src, so = Path(d) / "forms.cpp", Path(d) / "forms.so"
        src.write_text(SHIM)
        subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-I", str(B.CSRC), str(src), "-o", str(so)], check=True)
        return ctypes.CDLL(str(so))


def form_of(rows, n, k, may_cut=True):
    """(name, parts of k, bytes of the workspace) for a shape."""
    parts, work = ctypes.c_int(), ctypes.c_int64()
    kind = _lib().form_of(rows, n, k, int(may_cut), ctypes.byref(parts), ctypes.byref(work))
    return NAMES[kind], parts.value, work.value


def forms():
    """{name: (channels and rows of a tile, whether it may cut k)}"""
    out = {}
    for i in range(len(NAMES)):
        bn, bm, cuts = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
        kind = _lib().form(i, ctypes.byref(bn), ctypes.byref(bm), ctypes.byref(cuts))
        out[NAMES[kind]] = (bn.value, bm.value, bool(cuts.value))
    return out
