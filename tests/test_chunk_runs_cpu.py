"""How attention of chunks walks its work, compiled for the host from the header that the kernel uses: the CTAs' runs together take every key tile of every row
tile once, in order, and a walk whose sequences are gone ends."""

import ctypes as C
import os
import random
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bobcat_b200", "csrc")


@pytest.fixture(scope="module")
def runs(tmp_path_factory):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no host compiler")
    folder = tmp_path_factory.mktemp("runs")
    source, binary = folder / "runs.cpp", folder / "runs.so"
    source.write_text("""
#include "chunk_schedule.h"
#include <vector>
using namespace bc::k;
struct Call {
    uint32_t n_seqs; const uint32_t *starts, *lens; uint64_t capacity; uint32_t n_rows, fewest, per_tile, key_tile, kv;
    ChunkSeq at(uint32_t s) const { return chunk_seq(starts[s], starts[s + 1], lens[s], capacity, n_rows, fewest, per_tile, key_tile); }
};
// Places of the call's work, one by one: sequence, head, row tile, place in the row tile.
extern "C" uint64_t places(const Call* c, int whole, uint32_t* out, uint64_t room) {
    uint64_t n = 0;
    for (uint32_t s = 0; s < c->n_seqs; ++s) {
        const ChunkSeq q = c->at(s);
        for (uint32_t h = 0; h < c->kv; ++h)
            for (uint32_t r = 0; r < q.row_tiles; ++r)
                for (uint32_t i = 0; i < (whole ? 1 : q.tiles(r) + kRowTileCost); ++i, ++n)
                    if (n < room) out[4 * n] = s, out[4 * n + 1] = h, out[4 * n + 2] = r, out[4 * n + 3] = i;
    }
    return n;
}
// The units of the run [begin, end) that begins at a place; sequences from `gone` on have no rows any more. Eight numbers each.
extern "C" uint64_t walk(const Call* c, int whole, uint64_t begin, uint64_t end, const uint32_t* place, uint32_t gone, uint64_t* out, uint64_t room) {
    std::vector<uint32_t> starts(c->starts, c->starts + c->n_seqs + 1);
    for (uint32_t s = gone; s < c->n_seqs; ++s) starts[s + 1] = starts[gone];
    ChunkCursor cur{};
    cur.whole = whole;
    cur.s = c->at(place[0]);
    cur.seq = place[0], cur.head = place[1], cur.row_tile = place[2], cur.at = place[3];
    cur.count = cur.s.tiles(cur.row_tile);
    cur.end = end;
    cur.left = end - begin;
    for (uint64_t n = 0; n < room; ++n) {
        ChunkUnit u;
        if (!cur.take(starts.data(), c->lens, c->n_seqs, c->n_rows, c->kv, c->capacity, c->fewest, u)) return n;
        const uint64_t v[8] = {u.seq, u.head, u.row_tile, u.tile0, u.tiles, u.last, u.begins, u.ends};
        for (int i = 0; i < 8; ++i) out[8 * n + i] = v[i];
    }
    return room;
}
extern "C" uint32_t tiles(const Call* c, uint32_t s, uint32_t r) { return c->at(s).tiles(r); }
extern "C" uint32_t cost() { return kRowTileCost; }
""")
    subprocess.run([compiler, "-O1", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, "-I", "/usr/local/cuda/include", "-o", str(binary), str(source)], check=True)
    library = C.CDLL(str(binary))
    library.places.restype = library.walk.restype = C.c_uint64
    library.places.argtypes = [C.c_void_p, C.c_int, C.c_void_p, C.c_uint64]
    library.walk.argtypes = [C.c_void_p, C.c_int, C.c_uint64, C.c_uint64, C.c_void_p, C.c_uint32, C.c_void_p, C.c_uint64]
    library.tiles.argtypes = [C.c_void_p, C.c_uint32, C.c_uint32]
    return library


class Call(C.Structure):
    _fields_ = [("n_seqs", C.c_uint32), ("starts", C.c_void_p), ("lens", C.c_void_p), ("capacity", C.c_uint64)] + [
        (n, C.c_uint32) for n in ("n_rows", "fewest", "per_tile", "key_tile", "kv")]


def call(news, lens, capacity, fewest, per_tile, key_tile, kv, n_rows=None):
    starts = (C.c_uint32 * (len(news) + 1))(*[sum(news[:i]) for i in range(len(news) + 1)])
    held = (C.c_uint32 * len(news))(*lens)
    c = Call(len(news), C.addressof(starts), C.addressof(held), capacity, sum(news) if n_rows is None else n_rows, fewest, per_tile, key_tile, kv)
    c.keep = (starts, held)
    return c


def all_places(runs, c, whole):
    n = runs.places(C.byref(c), whole, None, 0)
    out = (C.c_uint32 * (4 * max(n, 1)))()
    runs.places(C.byref(c), whole, out, n)
    return n, out


def units_of(runs, c, whole, begin, end, out, gone=0xFFFFFFFF):
    room = 4 * (end - begin) + 4
    units = (C.c_uint64 * (8 * room))()
    n = runs.walk(C.byref(c), whole, begin, end, (C.c_uint32 * 4)(*out[4 * begin:4 * begin + 4]), gone, units, room)
    assert n < room  # the walk ended
    return [tuple(units[8 * i:8 * i + 8]) for i in range(n)]


def cases():
    rng = random.Random(5)
    for i in range(60):
        n = rng.choice([1, 1, 2, 5, 70])
        news = [rng.choice([0, 0, 1, 2, 3, 4, 17, 40, 130, 300]) for _ in range(n)]
        lens = [max(0, m + rng.randint(-3, 900)) for m in news]
        yield news, lens, rng.choice([256, 512, 1 << 20]), rng.choice([0, 4]), rng.choice([16, 18, 42, 128]), rng.choice([64, 128]), rng.choice([1, 2, 5]), rng.choice([1, 3, 7, 148])


@pytest.mark.parametrize("whole", [0, 1])
def test_runs_take_every_tile_once(runs, whole):
    for news, lens, capacity, fewest, per_tile, key_tile, kv, ctas in cases():
        c = call(news, lens, capacity, fewest, per_tile, key_tile, kv)
        n, out = all_places(runs, c, whole)
        want, got, ends = [], [], {}
        for i in range(n):
            s, h, r, at = out[4 * i:4 * i + 4]
            ends[s, h, r] = i
            tile = range(runs.tiles(C.byref(c), s, r)) if whole else [at - runs.cost()] if at >= runs.cost() else []
            want += [(s, h, r, t) for t in tile]
        count = min(ctas, n)
        for cta in range(count):
            begin, end = n * cta // count, n * (cta + 1) // count
            for s, h, r, tile0, tiles, last, begins, ends_here in units_of(runs, c, whole, begin, end, out):
                got += [(s, h, r, t) for t in range(tile0, tile0 + tiles)]
                assert last == ends[s, h, r]
                assert begins == (tile0 == 0) and ends_here == (tile0 + tiles == runs.tiles(C.byref(c), s, r))
        assert got == want


@pytest.mark.parametrize("whole", [0, 1])
def test_a_walk_whose_sequences_are_gone_ends(runs, whole):
    """Words that change under a call: nothing is taken twice, and nothing of what is no longer there."""
    news, lens = [40, 0, 20, 300, 1, 9], [50, 0, 20, 700, 900, 9]
    c = call(news, lens, 1 << 20, 0, 16, 64, 2)
    n, out = all_places(runs, c, whole)
    for gone in range(1, 7):
        units = units_of(runs, c, whole, 0, n, out, gone)
        assert len(set(units)) == len(units) and {u[0] for u in units} == {s for s in range(gone) if news[s]}
