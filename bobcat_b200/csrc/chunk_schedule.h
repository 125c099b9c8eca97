// The work of attention over pages for sequences of several new rows, as equal runs: plain arithmetic, the same on
// the host, which checks it, and in the kernel.
//
// A row tile is the query heads of `per_tile` neighbouring rows of one sequence and KV head. Row tile r sees the key tiles up to its last row's
// position; the tiles of a head, summed over its row tiles, are a sum of floor((a r + b) / m), which has a closed form by Euclid's steps, so a CTA
// finds its place without walking through them.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace bc {
namespace k {

// Sum over i = 0 .. n - 1 of floor((a i + b) / m), of numbers with (a mod m) n + m below 2^32: divisions of 64 bits are most of a search's instructions.
__host__ __device__ inline uint64_t floor_sum(uint32_t n, uint32_t m, uint32_t a, uint32_t b) {
    uint64_t sum = 0;
    while (n > 0) {
        const uint32_t of_a = a / m, of_b = b / m;
        sum += of_a * ((uint64_t)n * (n - 1) / 2) + (uint64_t)of_b * n;
        a -= of_a * m;
        b -= of_b * m;
        const uint32_t last = a * n + b, other = a;
        n = last / m;
        b = last - n * m;
        a = m;
        m = other;
        if (m == 0) break;
    }
    return sum;
}

// What a row tile counts beside its key tiles, ahead of them: its queries, its sums and the pipeline's start take about as long as two.
constexpr uint32_t kRowTileCost = 2;

struct ChunkSeq {
    uint32_t row0, n, end;   // rows row0 .. row0 + n - 1 are the sequence's; row `end` would be the position behind its last
    uint32_t len, held;      // positions, and those that its table can name
    uint32_t per_tile, row_tiles, key_tile;
    // Position of the first row, for counting: within what the table holds.
    __host__ __device__ uint32_t first() const {
        const uint32_t rows = end - row0;
        const uint32_t at = len > rows ? len - rows : 0;
        return at < held ? at : held;
    }
    // Key tiles of row tile r, one at least.
    __host__ __device__ uint32_t tiles(uint32_t r) const {
        const uint32_t rows = (r + 1) * per_tile;
        return (first() + (rows < n ? rows : n) - 1) / key_tile + 1;
    }
    // Key tiles of row tiles 0 .. r - 1, r < row_tiles.
    __host__ __device__ uint64_t tiles_before(uint32_t r) const { return r + floor_sum(r, key_tile, per_tile, first() + per_tile - 1); }
    __host__ __device__ uint64_t tiles_per_head() const { return row_tiles == 0 ? 0 : tiles_before(row_tiles - 1) + tiles(row_tiles - 1); }
    // What row tiles 0 .. r - 1 count as.
    __host__ __device__ uint64_t counted_before(uint32_t r) const { return tiles_before(r) + (uint64_t)kRowTileCost * r; }
};

// n_rows: rows of the whole call; fewest: sequences of fewer rows are not these kernels' work.
__host__ __device__ inline ChunkSeq chunk_seq(uint32_t start, uint32_t end, uint32_t len, uint64_t capacity, uint32_t n_rows, uint32_t fewest, uint32_t per_tile, uint32_t key_tile) {
    ChunkSeq s;
    s.row0 = start;
    s.end = end;
    s.n = start < n_rows && end > start ? (end < n_rows ? end : n_rows) - start : 0;
    if (end - start < fewest) s.n = 0;
    s.len = len;
    s.held = len < capacity ? len : (uint32_t)capacity;
    s.per_tile = per_tile;
    s.row_tiles = (s.n + per_tile - 1) / per_tile;
    s.key_tile = key_tile;
    return s;
}

// A stretch of key tiles of one row tile.
struct ChunkUnit {
    uint32_t seq, head, row_tile, tile0, tiles;
    uint64_t last;  // where the row tile ends in the call's work: its last place
    bool begins, ends;
};

// Walks a run: of row tiles that count as their key tiles and kRowTileCost, or of whole ones that count as one.
struct ChunkCursor {
    uint32_t seq, head, row_tile, count;
    uint64_t at, left, end;  // in the row tile; of the run; the run's end
    bool whole;
    ChunkSeq s;
    __host__ __device__ uint64_t all() const { return whole ? 1 : (uint64_t)count + kRowTileCost; }
    // The next stretch; false where the run has none, as where it ends ahead of a row tile's first key tile, or the sequences have ended before it.
    __host__ __device__ bool take(const uint32_t* starts, const uint32_t* lens, uint32_t n_seqs, uint32_t n_rows, uint32_t n_kv_heads, uint64_t capacity, uint32_t fewest, ChunkUnit& u) {
        if (left == 0) return false;
        if (at == all()) {  // on to the next row tile
            at = 0;
            if (++row_tile >= s.row_tiles) {
                row_tile = 0;
                if (++head >= n_kv_heads) {
                    head = 0;
                    do {
                        if (++seq >= n_seqs) {
                            left = 0;
                            return false;
                        }
                        s = chunk_seq(starts[seq], starts[seq + 1], lens[seq], capacity, n_rows, fewest, s.per_tile, s.key_tile);
                    } while (s.row_tiles == 0);
                }
            }
            count = s.tiles(row_tile);
        }
        u.seq = seq;
        u.head = head;
        u.row_tile = row_tile;
        u.last = end - left - at + all() - 1;
        const uint64_t upto = at + left < all() ? at + left : all();
        u.tile0 = whole || at < kRowTileCost ? 0 : (uint32_t)(at - kRowTileCost);
        const uint32_t tile1 = whole ? count : upto < kRowTileCost ? 0 : (uint32_t)(upto - kRowTileCost);
        u.tiles = tile1 - u.tile0;
        u.begins = u.tile0 == 0;
        u.ends = tile1 == count;
        left -= upto - at;
        at = upto;
        return u.tiles > 0;
    }
};

}  // namespace k
}  // namespace bc
