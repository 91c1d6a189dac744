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

# (form, whether k is cut): shapes that it is given -- rows, channels, k -- at its edges: one row and channel past whole tiles, results at
# places that are and are not aligned to four values, k of one step, of an odd number of steps, ending with 16 bytes of a step
# or in parts of unequal lengths
SHAPES = {
    ("DIRECT8", False): [(1, 4, 256), (1, 1, 272), (17, 1, 208), (17, 577, 1040), (1, 575, 7184)],
    ("DIRECT8_2", False): [(1, 4, 128), (1, 1, 16), (35, 1547, 272), (17, 1, 16), (3, 24575, 1552)],
    ("SPLIT11", False): [(49, 4, 128), (49, 1, 16), (49, 1, 272), (65, 1, 16)],
    ("SPLIT11", True): [(1, 4, 9216), (1, 1, 9488), (33, 1, 4592), (1, 1, 9456), (8, 576, 7168)],
    ("SPLIT12", False): [(8193, 4, 128), (8193, 1, 16), (385, 609, 272), (64, 7150, 4112)],
    ("SPLIT12", True): [(263, 148, 4608), (136, 286, 4496), (129, 257, 4576), (264, 161, 4160)],
    ("SPLIT22", False): [(66, 5480, 128), (8289, 33, 16), (897, 545, 272), (65, 5569, 16)],
    ("SPLIT22", True): [(262, 396, 8064), (199, 391, 8976), (257, 385, 6624)],
    ("SPLIT32", False): [(66, 8240, 128), (65, 8289, 16), (65, 8257, 272), (65, 8353, 16)],
    ("SPLIT32", True): [(647, 260, 9856), (193, 769, 9488), (193, 769, 8896), (641, 257, 8800)],
    ("SPLIT128", False): [(65, 16572, 128), (65, 16449, 16), (65, 16705, 272), (1025, 1921, 672)],
    ("SPLIT128", True): [(604, 780, 15232), (705, 705, 14352), (385, 1153, 13376), (130, 4090, 16400), (200, 2100, 16400)],
    ("TILE128", False): [(8209, 100, 128), (8233, 97, 16), (8705, 97, 272), (129, 8193, 16)],
    ("TILE192", False): [(129, 17096, 128), (129, 16385, 16), (129, 17025, 288), (257, 10945, 32), (1401, 7100, 2064)],
    ("TILE256", False): [(392, 24748, 128), (385, 25089, 16), (257, 24833, 528), (513, 20737, 16), (2001, 7101, 144), (4001, 4090, 4112)],
}


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
