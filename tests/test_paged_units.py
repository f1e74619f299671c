"""Host functions of the paged operators' sources, compiled by themselves and called without a GPU."""
import ctypes
import os
import random
import subprocess

import pytest

from conftest import REPO
from fftsparse_b200 import build

SOURCE = r"""
#include "paged_common.cuh"

namespace ffts { void set_error(int, const char *, ...) {} }

extern "C" int unit_rows_apart(const long long *sizes, const long long *strides, int n, long long inner) {
  int64_t a[3], b[3];
  for (int i = 0; i < n; ++i) { a[i] = sizes[i]; b[i] = strides[i]; }
  return ffts::rows_apart(a, b, n, inner);
}
"""


@pytest.fixture(scope="module")
def units(tmp_path_factory):
    d = tmp_path_factory.mktemp("units")
    src, lib = d / "units.cu", d / "units.so"
    src.write_text(SOURCE)
    flags = [f for f in build.NVCC_FLAGS if f not in ("-Xcompiler", "-fvisibility=hidden", "-fPIC", "-O3")]
    subprocess.run([build.nvcc(), *flags, "-O1", "-Xcompiler", "-fPIC", "-shared", "-I", build.INCLUDE, "-I", build.CSRC,
                    str(src), "-o", str(lib)], check=True, cwd=REPO)
    return ctypes.CDLL(os.fspath(lib))


def longs(values):
    return (ctypes.c_longlong * len(values))(*values)


# ------------------------------------------------------------------ rows of a written tensor
def apart(units, sizes, strides, inner):
    return bool(units.unit_rows_apart(longs(sizes), longs(strides), len(sizes), ctypes.c_longlong(inner)))


@pytest.mark.parametrize("sizes,strides,inner,want", [
    ((3, 4), (256, 64), 64, True), ((3, 4), (64, 192), 64, True), ((3, 4), (72, 288), 64, True),
    ((3, 4), (0, 64), 64, False), ((1, 4), (0, 64), 64, True), ((3, 4), (256, 0), 64, False), ((3, 1), (64, 0), 64, True),
    ((3, 4), (248, 64), 64, False), ((3, 4), (256, 56), 64, False), ((1, 1), (0, 0), 64, True), ((0, 4), (0, 64), 64, True),
    ((2, 2, 16), (2048, 1024, 64), 64, True), ((2, 2, 16), (2048, 64, 128), 64, True), ((2, 2, 16), (1024, 1024, 64), 64, False),
    ((2, 2, 16), (2048, 0, 128), 64, False), ((2, 2, 16), (0, 64, 128), 64, False),
    ((40000, 8, 64), (65536, 8192, 128), 128, True), ((1 << 30, 8, 2), (2048, 256, 128), 128, True)])
def test_rows_apart(units, sizes, strides, inner, want):
    assert apart(units, sizes, strides, inner) is want


def test_rows_apart_never_passes_rows_that_overlap(units):
    rng = random.Random(1)
    passed = 0
    for _ in range(20000):
        sizes = [rng.randrange(1, 4) for _ in range(3)]
        strides = [rng.randrange(0, 20) for _ in range(3)]
        inner = rng.randrange(1, 4)
        if apart(units, sizes, strides, inner):
            seen = [i * strides[0] + j * strides[1] + k * strides[2] + e for i in range(sizes[0]) for j in range(sizes[1])
                    for k in range(sizes[2]) for e in range(inner)]
            assert len(set(seen)) == len(seen), (sizes, strides, inner)
            passed += 1
    assert passed > 1000
