"""The arithmetic on sizes of the attention of several new tokens (csrc/tree_plan.h), compiled for the host: the chunks
that its kernels make of any rows fit the workgroups and the workspace that the host has planned without seeing the
rows. No GPU."""
import ctypes
import os
import random
import shutil
import subprocess

import pytest

from conftest import PKG, ROOT

SOURCE = r"""
#include "tree_plan.h"
using namespace trellis;
extern "C" void plan(int rows, int heads, int q_heads, int d, int tokens, int n, int exact, int cus, int64_t* out) {
  const TreeChunks p = tree_chunks(rows, heads, q_heads, d, tokens, n, exact, cus);
  out[0] = p.aim, out[1] = p.blocks, out[2] = p.items, out[3] = 32 * tree_waves(exact);
}
// blocks and chunks of rows of these lengths and new tokens, as tree_find counts them
extern "C" void made(const int* lens, const int* fresh, int rows, int heads, int group, int qr, int aim, int64_t* out) {
  int work = 0, all = 0, most = 0;
  for (int b = 0; b < rows; ++b) {
    const int blocks = tree_blocks(static_cast<int64_t>(fresh[b]) * group, qr), own = tree_units(lens[b]) > 1 ? tree_units(lens[b]) : 1;
    work += blocks * own, all += blocks;
    if (blocks && own > most) most = own;
  }
  const int units = aim ? tree_chunk_units(work, all, most, heads, aim) : 0;
  out[0] = static_cast<int64_t>(all) * heads, out[1] = 0, out[2] = 1;
  for (int b = 0; b < rows; ++b) {
    const int blocks = tree_blocks(static_cast<int64_t>(fresh[b]) * group, qr), own = tree_units(lens[b]) > 1 ? tree_units(lens[b]) : 1;
    const int chunks = aim ? (own + units - 1) / units : 1;
    out[1] += static_cast<int64_t>(blocks) * chunks * heads;
    // its chunks alike, and the last one not past the row
    const int each = (own + chunks - 1) / chunks;
    if (static_cast<int64_t>(each) * chunks < own || (aim && each > units)) out[2] = 0;
  }
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    cxx = shutil.which(os.environ.get("CXX", "g++"))
    if not cxx:
        pytest.skip("no C++ compiler")
    where = tmp_path_factory.mktemp("tree_plan")
    (where / "plan.cpp").write_text(SOURCE)
    subprocess.run([cxx, "-std=c++17", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, PKG, "csrc"),
                    str(where / "plan.cpp"), "-o", str(where / "plan.so")], check=True)
    return ctypes.CDLL(str(where / "plan.so"))


def _plan(lib, rows, heads, group, d, tokens, n, exact, cus=256):
    out = (ctypes.c_int64 * 4)()
    lib.plan(rows, heads, heads * group, d, tokens, n, exact, cus, out)
    return out[:]


def test_every_chunk_has_its_place(lib):
    rng, cut = random.Random(3), 0
    out = (ctypes.c_int64 * 3)()
    for trial in range(6000):
        rows, heads = rng.choice([1, 1, 2, 3, 16, 65, 200, 512, 513, 700]), rng.choice([1, 1, 2, 3, 8, 32])
        group, d, exact = rng.choice([1, 2, 4, 7, 16, 64, 65, 128, 129, 1000]), rng.choice([8, 64, 128, 136, 256]), rng.random() < 0.5
        n, tokens = int(2 ** rng.uniform(0, 17)), int(2 ** rng.uniform(0, 12))
        aim, blocks, items, qr = _plan(lib, rows, heads, group, d, tokens, n, exact)
        cut += aim > 0
        for kind in range(4):
            # every token in one row; spread; in the first rows; some in no row
            some = [0] * rows
            for _ in range(min(tokens, 300)) if kind else ():
                some[rng.randrange(rows) if kind != 2 else 0] += 1
            if kind == 0:
                some[rng.randrange(rows)] = tokens
            lens = [n if kind < 2 else rng.randint(0, n) for _ in range(rows)]
            lib.made((ctypes.c_int * rows)(*lens), (ctypes.c_int * rows)(*some), rows, heads, group, qr, aim, out)
            where = rows, heads, group, d, tokens, n, exact, kind, aim, blocks, items, out[:]
            assert out[0] <= blocks and out[1] <= items and out[2], where
    assert cut > 500


def test_rows_that_are_not_cut(lib):
    """Short rows, very many rows, and calls that fill the GPU with blocks alone."""
    assert _plan(lib, 4, 8, 4, 128, 40, 256, False)[0] == 0
    assert _plan(lib, 513, 1, 1, 64, 513, 4000, False)[0] == 0
    assert _plan(lib, 1, 8, 4, 128, 20000, 20000, False)[0] == 0
    assert _plan(lib, 4, 8, 4, 128, 40, 257, False)[0] > 0
    assert _plan(lib, 0, 8, 4, 128, 0, 257, False)[:3] == [0, 0, 0]
