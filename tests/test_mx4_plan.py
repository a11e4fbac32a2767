"""The MX4 kernels' host-side choices (csrc/exl3_mx4_plan.h), compiled here and checked without a GPU."""
import ctypes
import os
import random
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "b70-inference_amd", "csrc")

SHIM = """
#define __host__
#define __device__
#define _Float16 short
#include "exl3_mx4_plan.h"
using namespace exl3;
extern "C" void plan(int64_t m, int64_t n, int64_t k, int both, int cus, int* out) {
    const Mx4Plan p = both ? mx4_gemm_plan(m, n, k, cus) : mx4_linear_plan(m, n, k, cus);
    out[0] = p.tile;
    out[1] = p.P;
    out[2] = p.bps;
}
extern "C" int moe_rows(int64_t npairs, int64_t E) { return mx4_moe_rows(npairs, E); }
extern "C" int64_t max_blocks(int64_t npairs, int64_t E, int rows) { return mx4_max_blocks(npairs, E, rows); }
// blocks of an expert with c rows by count(), by walking locate() over every row as the align kernels do; largest block
extern "C" void cut(int rows, int c, int* out) {
    const BlockCut b = mx4_cut(rows);
    out[0] = b.count(c);
    out[1] = out[2] = 0;
    for (int f = 0; f < c;) {
        int first, cnt;
        b.locate(c, f, first, cnt);
        if (first != f || cnt < 1) { out[1] = -1; return; }
        for (int i = f; i < f + cnt; ++i) {
            int g, n;
            b.locate(c, i, g, n);
            if (g != first || n != cnt) { out[1] = -1; return; }
        }
        ++out[1];
        if (cnt > out[2]) out[2] = cnt;
        f = first + cnt;
    }
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("clang++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    d = tmp_path_factory.mktemp("mx4plan")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.check_call([cxx, "-std=c++20", "-O1", "-shared", "-fPIC", f"-I{CSRC}", "-o", str(d / "plan.so"),
                           str(d / "shim.cpp")])
    L = ctypes.CDLL(str(d / "plan.so"))
    L.max_blocks.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int]
    L.max_blocks.restype = ctypes.c_int64
    L.plan.argtypes = [ctypes.c_int64] * 3 + [ctypes.c_int, ctypes.c_int, ctypes.c_void_p]
    L.plan.restype = None
    L.moe_rows.argtypes = [ctypes.c_int64] * 2
    return L


def cut(lib, rows, c):
    out = (ctypes.c_int * 3)()
    lib.cut(rows, c, out)
    return tuple(out)


@pytest.mark.parametrize("rows", [16, 32, 64, 128])
def test_blocks_of_a_call_fit_their_table(lib, rows):
    for c in range(0, 3 * rows + 2):
        n, walked, largest = cut(lib, rows, c)
        assert n == walked == -(-c // rows) and largest <= rows, (rows, c)
    rng = random.Random(rows)
    for _ in range(300):
        E = rng.choice((1, 2, 5, 40, 300))
        counts = [rng.choice((0, 1, rng.randrange(3 * rows), rows, rows + 1, 2 * rows - 1)) for _ in range(E)]
        npairs = sum(counts)
        assert sum(cut(lib, rows, c)[0] for c in counts) <= lib.max_blocks(npairs, E, rows)
    for npairs in range(1, 200):                         # as many blocks as can be: one row in all experts but one
        for E in (1, 2, 7, 64):
            lone = min(E, npairs) - 1
            worst = lone + cut(lib, rows, npairs - lone)[0]
            assert worst <= lib.max_blocks(npairs, E, rows)


def plan(lib, m, n, k, both, cus=256):
    out = (ctypes.c_int * 3)()
    lib.plan(m, n, k, both, cus, out)
    return tuple(out)


def test_plans_cover_k_and_stay_within_bounds(lib):
    rng = random.Random(3)
    for _ in range(3000):
        m, n, k = rng.randrange(1, 5000), rng.randrange(1, 30000), 32 * rng.randrange(1, 700)
        for both in (0, 1):
            tile, P, bps = plan(lib, m, n, k, both, rng.choice((64, 256, 304)))
            nst = -(-k // 128)
            assert 0 <= tile < 3 and 1 <= P <= 16
            assert (P - 1) * bps < nst <= P * bps        # every split has work, together they cover k


def test_shapes_of_the_tile_tests(lib):
    """The shapes that the GPU tests take for every tile, without and with splits."""
    want = {(0, 3000, 160, 2601): (1, False), (0, 2001, 8224, 70): (1, True), (0, 1001, 160, 12301): (2, False),
            (0, 1501, 4128, 2602): (2, True), (1, 97, 544, 16401): (1, False), (1, 1501, 8224, 70): (1, True),
            (1, 1001, 160, 12301): (2, False), (1, 201, 8224, 16402): (2, True), (0, 520, 1024, 520): (0, False),
            (0, 31, 4096, 48): (0, True), (1, 520, 1024, 520): (0, False), (1, 100, 4096, 128): (0, True)}
    for (both, m, k, n), (tile, split) in want.items():
        p = plan(lib, m, n, k, both)
        assert (p[0], p[1] > 1) == (tile, split), (both, m, k, n, p)


def test_rows_per_block(lib):
    assert [lib.moe_rows(p, 4) for p in (1, 104, 105, 384, 385, 100000)] == [32, 32, 64, 64, 128, 128]
