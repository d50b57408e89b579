"""The attention's arithmetic on sizes (csrc/attend_plan.h), compiled for the host: what its kernels read lies within
their operands. No GPU."""
import ctypes
import os
import random
import shutil
import subprocess

import pytest

from conftest import PKG, ROOT

SOURCE = r"""
#include "attend_plan.h"
extern "C" int chunks(int rows, int heads, int q_heads, int d, int n, int cus, int64_t* out) {
  const trellis::AttChunks p = trellis::att_chunks(rows, heads, q_heads, d, n, cus);
  out[0] = p.aim, out[1] = p.chunk, out[2] = p.items;
  return p.row_blocks;
}
// the chunks that rows of these lengths are cut into, and the most of one row and head
extern "C" int64_t made(const int* lens, int rows, int heads, int aim, int64_t* most) {
  int units = 0;
  for (int b = 0; b < rows; ++b) units += trellis::att_units(lens[b]);
  const int size = trellis::att_chunk_units(units * heads, aim);
  int64_t all = 0;
  for (int b = *most = 0; b < rows; ++b) {
    const int64_t own = (trellis::att_units(lens[b]) + size - 1) / size;
    all += own * heads;
    if (own > *most) *most = own;
  }
  return all;
}
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
    lib = ctypes.CDLL(str(where / "plan.so"))
    lib.made.restype = ctypes.c_int64
    return lib


def test_queries_are_read_within_their_rows(plan):
    """Every lane group's 8 dims of every k-step lie in the head's row, and are the step's own where the row has them."""
    for d in range(8, 257, 8):
        padded = 64 if d <= 64 else 128 if d <= 128 else 256
        for j in range(padded // 32):
            for g in range(4):
                at = plan.q_dim(j, g, d)
                assert 0 <= at <= d - 8, (d, j, g, at)
                assert 32 * j + 8 * g >= d or at == 32 * j + 8 * g, (d, j, g, at)


def _chunks(plan, rows, heads, group, d, n, cus=256):
    out = (ctypes.c_int64 * 3)()
    plan.chunks(rows, heads, heads * group, d, n, cus, out)
    return out[:]


def test_every_chunk_has_its_place(plan):
    """The chunks that rows of any lengths make are no more than the plan's workgroups and partial sums, also where a
    group has more blocks of 16 query heads than there are workgroups to aim at; no row has more than the join takes."""
    rng = random.Random(1)
    most = ctypes.c_int64(0)
    for trial in range(4000):
        rows = rng.choice([2, 2, 3, 5, 16, 64, 65, 200, 512])
        heads = rng.choice([1, 1, 2, 3, 8, 32])
        group = rng.choice([1, 4, 16, 17, 40, 1000, 4096, 4097, 8192, 8193, 8208, 9000, 20000])
        d, n = rng.choice([64, 128, 136, 256]), int(2 ** rng.uniform(9.01, 17))
        aim, _, items = _chunks(plan, rows, heads, group, d, n)
        assert aim >= 1
        for lens in ([n] * rows, [n] + [0] * (rows - 1), [rng.randint(0, n) for _ in range(rows)], [n] + [1] * (rows - 1)):
            made = plan.made((ctypes.c_int * rows)(*lens), rows, heads, aim, ctypes.byref(most))
            assert made <= items and most.value <= 1024, (rows, heads, group, d, n, lens[:8], made, items, most.value)


def test_one_rows_chunks_cover_it(plan):
    rng = random.Random(2)
    for trial in range(4000):
        heads, group = rng.choice([1, 2, 3, 8, 32]), rng.choice([1, 4, 17, 8193, 20000])
        d, n = rng.choice([64, 128, 136, 256]), int(2 ** rng.uniform(9.01, 30))
        aim, chunk, items = _chunks(plan, 1, heads, group, d, n)
        assert aim >= 1 and chunk % 128 == 0 and items % heads == 0
        assert (items // heads - 1) * chunk < n <= items // heads * chunk and items // heads <= 1024, (heads, group, d, n)


def test_workspace_holds_every_chunk_of_a_huge_group(te):
    """Two rows of 13000 tokens under 8208 query heads of one key-value head make 4 chunks of 64 dims and 2 numbers."""
    size = ctypes.c_size_t(0)
    cache = te._capi.TrellisKVCache(k=256, v=256, table=256, lens=512, page_stride=1024, head_stride=1024, slot_stride=64, table_stride=1000,
                                    pages=9, heads=1, page_size=16, head_dim=64, dtype=1, rows=2, width=1000, max_len=13000)
    assert te.library().trellis_attention_workspace_bytes(cache, 8208, 0, size) == 0
    assert size.value >= 4 * 8208 * (64 + 2) * 4
