"""The key/value pool without a GPU: the sizes of its pages, what is refused before a device is needed, and how the work of chunks is counted,
which the host compiles from the header that the kernel uses."""

import ctypes as C
import os
import shutil
import subprocess

import pytest

from bobcat_b200 import F16, I8, errors

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bobcat_b200", "csrc")


@pytest.mark.parametrize("page_size", [16, 64, 256])
@pytest.mark.parametrize("kv, hd", [(1, 64), (8, 128), (1024, 256)])
def test_bytes_of_pages(lib, page_size, kv, hd):
    for n in (0, 1, 70000, 0xFFFFFFFF):
        assert lib.bc_kv_pool_bytes(F16, n, page_size, kv, hd) == n * page_size * kv * hd * 2
        assert lib.bc_kv_pool_bytes(I8, n, page_size, kv, hd) == n * page_size * kv * (hd + 4)


def test_shapes_that_pages_cannot_have(lib):
    for fmt, page_size, kv, hd in [(0, 16, 1, 64), (8, 16, 1, 64), (F16, 0, 1, 64), (F16, 8, 1, 64), (I8, 24, 1, 64), (I8, 512, 1, 64), (F16, 16, 0, 64),
                                   (F16, 16, 1025, 64), (F16, 16, 1, 0), (I8, 16, 1, 80), (I8, 16, 1, 512)]:
        assert lib.bc_kv_pool_bytes(fmt, 4, page_size, kv, hd) == 0


def test_no_backend_is_an_error(lib):
    assert lib.bc_op_kv_write(None, None, None, None, 0, None, 0, 64, 64) == errors.Argument.status
    assert lib.bc_op_kv_read(None, None, None, None, 0, None, 0, 0, 64, 64) == errors.Argument.status
    assert lib.bc_op_attention_paged(None, None, None, None, 0, None, 0, None, 0, 8, 512, 64) == errors.Argument.status
    out = C.c_void_p()
    assert lib.bc_buffer_at(None, 256, 16, C.byref(out)) == errors.Argument.status and not out.value


def test_scratch_does_not_follow_the_lengths(lib):
    sizes = [lib.bc_attention_paged_scratch_floats(heads, kv, 128) for heads, kv in ((8, 8), (32, 4), (64, 64))]
    assert len(set(sizes)) == 1 and 0 < sizes[0] < lib.bc_attention_paged_scratch_floats(8, 8, 256)


@pytest.fixture(scope="module")
def schedule(tmp_path_factory):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no host compiler")
    folder = tmp_path_factory.mktemp("schedule")
    source, binary = folder / "schedule.cpp", folder / "schedule.so"
    source.write_text("""
#include "chunk_schedule.h"
using namespace bc::k;
extern "C" uint64_t sums(uint32_t n, uint32_t m, uint32_t a, uint32_t b) { return floor_sum(n, m, a, b); }
extern "C" uint32_t sequence(uint32_t start, uint32_t end, uint32_t len, uint64_t capacity, uint32_t n_rows, uint32_t fewest, uint32_t per_tile, uint32_t key_tile,
                             uint32_t* tiles, uint64_t* before, uint64_t* counted, uint64_t* per_head) {
    const ChunkSeq s = chunk_seq(start, end, len, capacity, n_rows, fewest, per_tile, key_tile);
    for (uint32_t r = 0; r < s.row_tiles; ++r) tiles[r] = s.tiles(r), before[r] = s.tiles_before(r), counted[r] = s.counted_before(r);
    *per_head = s.tiles_per_head();
    return s.row_tiles;
}
extern "C" uint32_t cost() { return kRowTileCost; }
""")
    subprocess.run([compiler, "-O1", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, "-I", "/usr/local/cuda/include", "-o", str(binary), str(source)], check=True)
    library = C.CDLL(str(binary))
    library.sums.restype = C.c_uint64
    library.sums.argtypes = [C.c_uint32] * 4
    library.sequence.argtypes = [C.c_uint32] * 3 + [C.c_uint64] + [C.c_uint32] * 4 + [C.c_void_p] * 4
    return library


def test_sums_of_quotients(schedule):
    for n in (0, 1, 2, 7, 100, 5000):
        for m in (1, 3, 64, 128):
            for a in (0, 1, 16, 127, 300):
                for b in (0, 5, 127, 1 << 31):
                    assert schedule.sums(n, m, a, b) == sum((a * i + b) // m for i in range(n))


@pytest.mark.parametrize("per_tile", [16, 18, 42, 128])  # 8, 7, 3 and 1 query heads a KV head
@pytest.mark.parametrize("key_tile", [64, 128])
@pytest.mark.parametrize("n, length, capacity, n_rows, fewest", [
    (1, 1, 256, 1000, 0), (1, 0, 256, 1000, 0), (5, 3, 256, 1000, 0), (300, 300, 512, 1000, 0), (300, 5000, 8192, 1000, 0), (300, 5000, 1024, 1000, 0),
    (300, 100, 64, 1000, 0), (300, 700, 1024, 150, 0), (300, 700, 1024, 7, 0), (2, 700, 1024, 1000, 3), (3, 700, 1024, 1000, 3), (0, 700, 1024, 1000, 0),
    (2000, (1 << 32) - 1, 1 << 31, 5000, 0)])
def test_key_tiles_of_row_tiles(schedule, per_tile, key_tile, n, length, capacity, n_rows, fewest):
    """Each row tile has the key tiles that its last row sees, one at least, of those that the table holds; the closed forms add them up."""
    start = 7
    most = n // per_tile + 1
    tiles, before, counted, per_head = (C.c_uint32 * most)(), (C.c_uint64 * most)(), (C.c_uint64 * most)(), C.c_uint64()
    row_tiles = schedule.sequence(start, start + n, length, capacity, n_rows, fewest, per_tile, key_tile, tiles, before, counted, C.byref(per_head))
    rows = max(0, min(n, n_rows - start)) if n >= fewest else 0
    assert row_tiles == -(-rows // per_tile)
    total = 0
    for r in range(row_tiles):
        last = length - n + min((r + 1) * per_tile, rows) - 1  # of the row tile, its position
        needed = -(-min(max(last + 1, 0), capacity, length) // key_tile)
        assert needed <= tiles[r] <= max(needed, 1) + (0 if 0 <= length - n <= capacity - n else -(-n // key_tile) + 1)
        assert before[r] == total and counted[r] == total + schedule.cost() * r
        total += tiles[r]
    assert per_head.value == total
