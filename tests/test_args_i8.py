"""Which calls of the 8-bit operators are refused: the host checks of csrc/args_i8.hpp, compiled with g++ and called here with addresses that nothing reads."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
CSRC = ROOT / "tile-rs_b200" / "csrc"
SOURCE = """
#include "args_i8.hpp"
using namespace tsm100::args;
extern "C" const char* rows(const tsm100_quantise_rows_desc* d, void* x, void* up, void* y, float* s, int* nothing) {
  bool n; const char* r = quantise_rows(d, x, up, y, s, &n); *nothing = n; return r;
}
extern "C" const char* product(const tsm100_gemm_i8_desc* d, void* a, float* as, void* w, float* ws, void* c, int* nothing) {
  bool n; const char* r = gemm_i8(d, a, as, w, ws, c, &n); *nothing = n; return r;
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = tmp_path_factory.mktemp("args") / "libargs.so"
    src = out.with_suffix(".cpp")
    src.write_text(SOURCE)
    subprocess.run(["/usr/bin/g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", str(src), "-o", str(out)], check=True)
    handle = C.CDLL(str(out))
    for f in (handle.rows, handle.product):
        f.restype = C.c_char_p
    return handle


def rows(lib, pkg, dtype=2, rows=4, cols=64, pitch=0, x=0x1000, up=0, y=0x3000, scales=0x4000, desc=True):
    d, nothing = pkg.capi.QuantiseRowsDesc(dtype, rows, cols, pitch), C.c_int(-1)
    r = lib.rows(C.byref(d) if desc else None, *(C.c_void_p(p) for p in (x, up, y, scales)), C.byref(nothing))
    return (r or b"").decode(), nothing.value


def product(lib, pkg, dtype=2, m=4, n=64, k=64, lda=0, ldw=0, ldc=0, a=0x1000, a_scales=0x2000, w=0x3000, w_scales=0x4000, c=0x5000, desc=True):
    d, nothing = pkg.capi.GemmI8Desc(dtype, m, n, k, lda, ldw, ldc), C.c_int(-1)
    r = lib.product(C.byref(d) if desc else None, *(C.c_void_p(p) for p in (a, a_scales, w, w_scales, c)), C.byref(nothing))
    return (r or b"").decode(), nothing.value


@pytest.mark.parametrize("change,words", [
    ({"desc": False}, "null descriptor"), ({"dtype": 3}, "dtype"), ({"dtype": -1}, "dtype"), ({"rows": -1}, "shape"), ({"cols": 1 << 31}, "shape"), ({"pitch": -8}, "shape"),
    ({"pitch": 63}, "less than cols"), ({"rows": 1 << 30, "pitch": 1 << 40}, "shape"), ({"x": 0}, "null buffer"), ({"y": 0}, "null buffer"), ({"scales": 0}, "null buffer"),
    ({"x": 0x1001}, "boundary"), ({"up": 0x1001}, "boundary"), ({"dtype": 0, "x": 0x1002}, "boundary"), ({"scales": 0x4002}, "boundary")])
def test_rows_that_are_refused(lib, pkg, change, words):
    assert words in rows(lib, pkg, **change)[0]


@pytest.mark.parametrize("change,nothing", [({}, 0), ({"up": 0x2000, "pitch": 128}, 0), ({"x": 0x1002, "y": 0x3001}, 0), ({"rows": 0, "x": 0}, 1), ({"cols": 0, "y": 0}, 1)])
def test_rows_that_are_taken(lib, pkg, change, nothing):
    assert rows(lib, pkg, **change) == ("", nothing)


@pytest.mark.parametrize("change,words", [
    ({"desc": False}, "null descriptor"), ({"dtype": 3}, "dtype"), ({"m": -1}, "shape"), ({"n": 1 << 31}, "shape"), ({"k": -1}, "shape"), ({"k": 131072}, "131072"),
    ({"lda": -1}, "shape"), ({"lda": 63}, "pitch"), ({"ldw": 63}, "pitch"), ({"ldc": 63}, "pitch"), ({"ldc": 1 << 40}, "shape"), ({"a": 0}, "null buffer"),
    ({"a_scales": 0}, "null buffer"), ({"w": 0}, "null buffer"), ({"w_scales": 0}, "null buffer"), ({"c": 0}, "null buffer"), ({"c": 0x5001}, "boundary"),
    ({"dtype": 0, "c": 0x5002}, "boundary"), ({"a_scales": 0x2002}, "boundary"), ({"w_scales": 0x4001}, "boundary"),
    ({"m": 1 << 30, "n": 1 << 20}, "too many rows")])
def test_products_that_are_refused(lib, pkg, change, words):
    assert words in product(lib, pkg, **change)[0]


@pytest.mark.parametrize("change,nothing", [({}, 0), ({"a": 0x1001, "w": 0x3003, "c": 0x5002}, 0), ({"k": 131071}, 0), ({"m": 0, "a": 0}, 1), ({"n": 0, "c": 0}, 1),
                                            ({"k": 0, "a": 0, "w": 0, "a_scales": 0, "w_scales": 0}, 0), ({"lda": 80, "ldw": 96, "ldc": 100}, 0)])
def test_products_that_are_taken(lib, pkg, change, nothing):
    assert product(lib, pkg, **change) == ("", nothing)


def test_the_largest_sums_fit_32_bits():
    assert 128 * 128 * 131071 < 2 ** 31
