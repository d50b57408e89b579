"""The attention's arithmetic on sizes (csrc/attend_plan.h), compiled for the host: what its kernels read lies within
their operands. No GPU."""
import ctypes
import os
import shutil
import subprocess

import pytest

from conftest import PKG, ROOT

SOURCE = r"""
#include "attend_plan.h"
extern "C" int q_dim(int j, int g, int d) { return trellis::att_q_dim(j, g, d); }
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    cxx = shutil.which(os.environ.get("CXX", "g++"))
    if not cxx:
        pytest.skip("no C++ compiler")
    where = tmp_path_factory.mktemp("plan")
    (where / "plan.cpp").write_text(SOURCE)
    subprocess.run([cxx, "-std=c++17", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, PKG, "csrc"),
                    str(where / "plan.cpp"), "-o", str(where / "plan.so")], check=True)
    return ctypes.CDLL(str(where / "plan.so"))


def test_queries_are_read_within_their_rows(plan):
    """Every lane group's 8 dims of every k-step lie in the head's row, and are the step's own where the row has them."""
    for d in range(8, 257, 8):
        padded = 64 if d <= 64 else 128 if d <= 128 else 256
        for j in range(padded // 32):
            for g in range(4):
                at = plan.q_dim(j, g, d)
                assert 0 <= at <= d - 8, (d, j, g, at)
                assert 32 * j + 8 * g >= d or at == 32 * j + 8 * g, (d, j, g, at)
