// Attention of sequences' new rows over a pool of key/value pages on the tensor cores: the form for several rows of a sequence, whose time
// is multiplies.
//
// Arithmetic: that of kernels_attention_paged.cu. Elements are exact halves (8-bit ones as whole numbers, their scales multiply scores and
// probabilities in f32), a query element and a probability (times the value's scale) are two halves, sums are f32. tcgen05 cuts a sum off instead of
// rounding it, so what it sums stays short: scores over a head, values over one key tile; the tiles' sums are added up in registers.
//
// Shape. Persistent CTAs over equal runs (chunk_schedule.h) of row tiles: 128 rows, the query heads of neighbouring rows that share a KV head, against
// key tiles of 128 positions (64 for heads of 256). One warp walks the run, looks the pages up and brings a tile's bytes into shared memory by bulk
// copies, a page's share each. Four warps unpack them and, of values, transpose them, into the no-swizzle K-major operand layout; its 128-byte core matrices
// lie 144 bytes apart, so that what neighbouring lanes store falls in distinct banks. One warp issues the multiplies. Eight warps own the rows, a thread
// half of a row's scores and half of its sums: they exchange the rows' maxima through shared memory, turn scores into probabilities in place in
// tensor memory, and add the previous tile's product to their sums, while the scores of the next tile run. Tiles that every row sees whole have a loop of
// their own (2048 rows behind 30 001 positions: 2.12 ms, 2.37 in one loop with the masks and with weights by row).
// Queries and probabilities are A operands in tensor memory: both operands in shared memory would take its 128 bytes a cycle whole. (Heads of 256
// leave room for the queries' upper halves alone.)
//
// Measured: 2048 rows of 32 heads of 128 behind 30 001 8-bit positions, 2.12 ms: 490 TFLOP/s of attention, twice that in half products (multiplies alone would take
// 1.26 ms). A key tile takes 4300 cycles, its multiplies 2100 of them; the rest is the rows' warps, whose instructions bound it: 58 % of the issue slots
// are used. Tried and left, against 2.31 ms then: four threads to a row (2.48: the instructions grow by a quarter), scores held in registers between
// maximum and exponential (2.61). 512 rows from position 0, 32 heads of 64, take 19 us, most of it one CTA's way through two tiles.

#include <type_traits>

#include "async_utils.cuh"
#include "chunk_schedule.h"
#include "kv_pool.cuh"

#include "../../include/bobcat_cuda.h"

namespace bc {
namespace k {

namespace {

using namespace async;

constexpr uint32_t kRows = 128;                    // rows of a tile
constexpr uint32_t kParts = 2;                     // threads of a row
constexpr uint32_t kRowWarps = 4 * kParts, kUnpackWarps = 4, kMmaWarp = kRowWarps + kUnpackWarps, kCopyWarp = kMmaWarp + 1, kThreads = 32 * (kMmaWarp + 4);
constexpr uint32_t kRowThreads = 32 * kRowWarps, kUnpackThreads = 32 * kUnpackWarps;
// Registers of a thread after the split, 128 before: 256 threads x 184 + 128 x 96 + 128 x 48 = 512 x 128.
constexpr int kRowRegisters = 184, kUnpackRegisters = 96, kOtherRegisters = 48;
constexpr uint32_t kCore = 144;                    // bytes from one core matrix to the next
constexpr uint32_t kTmemColumns = 512;
constexpr uint32_t kMostCtas = kChunkMostCtas;
constexpr uint32_t kJoinCtas = 8;                  // of the joining launch, to a cut row tile
constexpr uint32_t kSpinLimit = 1u << 22;
constexpr uint32_t kRing = 4, kDescRing = 8;       // tiles whose scales and masks are kept; whose descriptions are

template <int HD>
constexpr uint32_t key_tile() { return HD == 256 ? 64 : 128; }
// Operand tiles and tiles of bytes on their way, as many as shared memory holds.
template <int FMT, int HD>
constexpr uint32_t stages() { return HD == 256 || (HD == 128 && FMT == BC_F16) ? 1 : 2; }
template <int FMT, int HD>
constexpr uint32_t raw_tiles() { return HD == 256 && FMT == BC_F16 ? 1 : 2; }

__device__ int* g_wait_word;  // where a wait that ran out leaves its code (kernels.h), null until set

struct ChunkParams {
    KvPool pool;
    KvRows rows;
    const float* q;
    float* out;
    float* parts;  // [2 * CTA + which][kRows][HD] sums, then [2 * CTA + which][kRows] (maximum, sum), then a ChunkHead per CTA, then a ChunkSpan
    uint64_t q_stride, q_head_stride;
    uint32_t n_heads, group, fewest;
};
// What a CTA leaves the joining launch: the unit that begins in its run and goes on behind it, `last` the CTA that this ends in, 0 when there is none; and whether
// sums of a row that it has written whole are no number (kOdd).
struct ChunkHead {
    uint32_t row0, n, head, last;  // rows of the call from row0, n of them (and kOdd); KV head
};
constexpr uint32_t kOdd = 1u << 31;
// Its first unit and its last.
struct ChunkSpan {
    uint32_t seq[2], head[2], row_tile[2], unused[2];
};
__device__ __forceinline__ ChunkHead* chunk_heads(float* parts, uint32_t head_dim) { return reinterpret_cast<ChunkHead*>(parts + (uint64_t)2 * kMostCtas * kRows * (head_dim + 2)); }
__device__ __forceinline__ ChunkSpan* chunk_spans(float* parts, uint32_t head_dim) { return reinterpret_cast<ChunkSpan*>(chunk_heads(parts, head_dim) + kMostCtas); }

// Where the first loading warp is in the run.
struct Place {
    ChunkCursor cursor;
    ChunkUnit unit;
    uint32_t in_unit, unit_number;
    ChunkHead cut;
    ChunkSpan span;
};
// What a tile is, for every role.
struct TileDesc {
    uint32_t key0, end;       // the first position, and the position behind the sequence's last that its table can name
    uint32_t groups;          // of 16 positions, a bit each: in a page of the pool
    uint32_t row0, n, head;   // the row tile's first row of the call, its rows, the KV head
    int32_t pos0;             // the position of its first row
    uint32_t unit;            // number within the run
    uint32_t first, last;     // of the unit
    uint32_t begins, ends;    // the unit: whether the row tile's first and last key tiles are its
};
// What the unpacking warps leave behind for a tile.
template <uint32_t KT, int FMT>
struct TileInfo {
    uint32_t valid[KT / 32];
    uint32_t masked;          // whether some row does not see some of its positions
    alignas(16) uint32_t top_scale[kUnpackWarps], low_scale[kUnpackWarps];  // the values' largest and smallest finite scale, by warp
    alignas(16) float dk[FMT == BC_I8 ? KT : 4];
    alignas(16) float dv[FMT == BC_I8 ? KT : 4];
};
// A tile's bytes as they lie in the pages: its keys with both scales, which the scores' warps want first, and its values.
template <uint32_t KT, int FMT, int HD>
struct RawKeys {
    static constexpr uint32_t kRowBytes = FMT == BC_F16 ? 2 * HD : HD;
    uint8_t keys[KT * kRowBytes];
    float dk[FMT == BC_I8 ? KT : 4], dv[FMT == BC_I8 ? KT : 4];
};

__device__ __forceinline__ void give_up(volatile int* dead, int code) {
    *dead = 1;
    if (g_wait_word) *reinterpret_cast<volatile int*>(g_wait_word) = code;
}
__device__ __forceinline__ bool wait_on(uint32_t bar, uint32_t parity, volatile int* dead, int code) {
    if (__all_sync(0xffffffffu, mbar_wait(bar, parity, kSpinLimit, dead))) return true;
    if ((threadIdx.x & 31) == 0) give_up(dead, code);
    return false;
}
// A whole warp's wait. One that runs out takes the warp out of its loop, and the others with it: all that warps wait for are mbarriers, so nobody
// waits for it for good. It touches nothing after that: what it would go by may not be there.
__device__ __forceinline__ void await(bool& alive, uint32_t bar, uint32_t parity, volatile int* dead, int code) {
    if (alive) alive = __all_sync(0xffffffffu, mbar_test(bar, parity)) || wait_on(bar, parity, dead, code);
}

__device__ __forceinline__ void umma_f16_a_tmem(uint32_t tmem_d, uint32_t tmem_a, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Loads and stores of memory may move across these; tcgen05.wait::st keeps what follows behind.
__device__ __forceinline__ void tmem_store_8(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
                 "r"(v[6]), "r"(v[7]));
}
// Pairs of f32 in one instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(r)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(r)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return r;
}
__device__ __forceinline__ float log2_fast(float x) {  // of zero, minus infinity
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// (x, y) as halves of the upper 11 bits, cut off, and of what they leave over.
__device__ __forceinline__ void cut_half2(float2 x, uint32_t& hi, uint32_t& lo) {
    const float2 upper = make_float2(__uint_as_float(__float_as_uint(x.x) & 0xffffe000u), __uint_as_float(__float_as_uint(x.y) & 0xffffe000u));
    const __half2 h = __floats2half2_rn(upper.x, upper.y);
    const float2 rest = fma2(upper, make_float2(-1.f, -1.f), x);
    const __half2 l = __floats2half2_rn(rest.x, rest.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}
// Which of 16 scores a row sees: those of positions that exist, up to the last it may.
template <uint32_t KT, int FMT>
__device__ __forceinline__ uint32_t seen_bits(const TileInfo<KT, FMT>& info, uint32_t score, int32_t upto) {
    const uint32_t there = info.valid[score / 32] >> (score % 32), n = (uint32_t)max(upto + 1, 0);  // scores up to the limit
    return there & (n >= 16 ? 0xffffu : (1u << n) - 1);
}

// Four lanes' four pieces each: piece i of lane j becomes piece j of lane i. A row's memory is read and written four lanes at a time, 64 bytes, while a
// thread works on a row of its own.
__device__ __forceinline__ void quad_transpose(float4 (&v)[4], uint32_t lane) {
#pragma unroll
    for (int bit = 1; bit <= 2; bit <<= 1) {
        const bool upper = lane & bit;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i & bit) continue;
            float4 &a = v[i], &b = v[i | bit], give = upper ? a : b;
            give.x = __shfl_xor_sync(0xffffffffu, give.x, bit);
            give.y = __shfl_xor_sync(0xffffffffu, give.y, bit);
            give.z = __shfl_xor_sync(0xffffffffu, give.z, bit);
            give.w = __shfl_xor_sync(0xffffffffu, give.w, bit);
            (upper ? a : b) = give;
        }
    }
}

// A barrier of several warps that a warp may leave: an mbarrier with an arrival of each.
struct WarpsBarrier {
    uint32_t bar, phase;
    int code;
    __device__ __forceinline__ void sync(bool& alive, volatile int* dead) {
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
        await(alive, bar, phase, dead, code);
        phase ^= 1;
    }
};

template <int FMT, int HD>
struct Shared {
    static constexpr uint32_t KT = key_tile<HD>(), kStages = stages<FMT, HD>(), kRaw = raw_tiles<FMT, HD>(), kUnits = 8;
    static constexpr uint32_t kTileBytes = KT / 8 * (HD / 8) * kCore;
    uint8_t q_lo[HD == 256 ? kRows / 8 * (HD / 8) * kCore : 16];
    uint8_t keys[kStages][kTileBytes], values[kStages][kTileBytes];
    alignas(16) RawKeys<KT, FMT, HD> raw_keys[kRaw];
    alignas(16) uint8_t raw_values[kRaw][KT * RawKeys<KT, FMT, HD>::kRowBytes];
    TileInfo<KT, FMT> info[kRing];
    TileDesc desc[kDescRing];
    float heaviest[2][kParts][FMT == BC_I8 ? kRows : 1];  // [parity][part]: of the parts of a row's weights, their logarithms
    float most[2][kParts][kRows];  // [parity][part]: maxima of the parts of a row's scores; at a unit's ends, other exchanges
    uint32_t not_finite[FMT == BC_F16 ? kUnits : 1][FMT == BC_F16 ? HD : 1];  // by unit: the first position with such a value, of each element
    uint32_t any_not_finite[kUnits];
    uint64_t bars[4 * kStages + 4 * kRaw + 13 + kDescRing];
    uint64_t counted, ahead[2];  // the call's work; key tiles ahead of the run's beginning, and of its end
    Place place;
    uint32_t tmem;
    int dead, never;            // whether a wait has run out; a flag that nobody raises
    int odd;                    // whether sums of a row that was written whole are no number
};

template <int FMT, int HD>
__global__ void __launch_bounds__(kThreads, 1) attention_chunk_paged_kernel(const __grid_constant__ ChunkParams p) {
    using S = Shared<FMT, HD>;
    constexpr uint32_t KT = S::KT, ST = S::kStages, RAW = S::kRaw, kUnits = S::kUnits;
    constexpr uint32_t kKeyStep = HD / 8 * kCore;  // between groups of 8 rows of a K-major operand over a head's elements
    // Tensor memory: two tiles of scores, the product with the values, the queries' halves.
    constexpr uint32_t kPv = 2 * KT, kQHi = kPv + HD, kQLo = kQHi + HD / 2;
    constexpr bool kQLoShared = HD == 256;
    static_assert(kQLo + (kQLoShared ? 0 : HD / 2) <= kTmemColumns, "tensor memory");
    constexpr float kLift = FMT == BC_F16 ? 15.f : 14.f;  // probabilities times 2^15; weights times scales of up to two units
    extern __shared__ __align__(128) uint8_t smem_raw[];
    S& sh = *reinterpret_cast<S*>(smem_raw);
    volatile int* dead = &sh.dead;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const KvPool& pool = p.pool;
    const uint64_t capacity = (uint64_t)p.rows.max_pages << pool.page_shift;
    const uint32_t per_tile = kRows / p.group;
    const uint32_t bars = smem_u32(sh.bars);
    const uint32_t k_full = bars, k_free = k_full + 8 * ST, v_full = k_free + 8 * ST, v_free = v_full + 8 * ST, rk_full = v_free + 8 * ST, rk_free = rk_full + 8 * RAW;
    const uint32_t rv_full = rk_free + 8 * RAW, rv_free = rv_full + 8 * RAW, s_full = rv_free + 8 * RAW, p_ready = s_full + 16, pv_full = p_ready + 16, pv_free = pv_full + 16, q_ready = pv_free + 8;
    const uint32_t rows_bar = q_ready + 8, unpack_bar = rows_bar + 8 * 4, described = unpack_bar + 8;

    pdl_launch_dependents();
    if (tid == 0) {
        for (uint32_t s = 0; s < ST; ++s) {
            mbar_init(k_full + 8 * s, kUnpackWarps);
            mbar_init(k_free + 8 * s, 1);
            mbar_init(v_full + 8 * s, kUnpackWarps);
            mbar_init(v_free + 8 * s, 1);
        }
        for (uint32_t r = 0; r < RAW; ++r) {
            mbar_init(rk_full + 8 * r, 1);
            mbar_init(rk_free + 8 * r, kUnpackWarps);
            mbar_init(rv_full + 8 * r, 1);
            mbar_init(rv_free + 8 * r, kUnpackWarps);
        }
        mbar_init(s_full, 1);
        mbar_init(s_full + 8, 1);
        mbar_init(p_ready, kRowWarps);
        mbar_init(p_ready + 8, kRowWarps);
        mbar_init(pv_full, 1);
        mbar_init(pv_full + 8, 1);
        mbar_init(pv_free, kRowWarps);
        mbar_init(q_ready, kRowWarps);
        for (uint32_t w = 0; w < 4; ++w) mbar_init(rows_bar + 8 * w, kParts);
        mbar_init(unpack_bar, kUnpackWarps);
        for (uint32_t d = 0; d < kDescRing; ++d) mbar_init(described + 8 * d, 1);
        sh.dead = sh.never = sh.odd = 0;
        mbar_init_fence();
    }
    if (warp == kMmaWarp) tmem_alloc(smem_u32(&sh.tmem), kTmemColumns);
    pdl_wait();
    if (warp == kCopyWarp || warp == kCopyWarp + 1) {
        // The run, and where it begins and ends.
        auto seq_at = [&](uint32_t s) {
            return chunk_seq(p.rows.starts[s], p.rows.starts[s + 1], p.rows.lens[s], capacity, p.rows.n_rows, p.fewest, per_tile, KT);
        };
        uint64_t total = 0, units = 0;
        uint32_t longest = 0;
        uint64_t my_tiles = 0, my_units = 0;  // of the lane's first sequence
        for (uint32_t s = lane; s < p.rows.n_seqs; s += 32) {
            const ChunkSeq sq = seq_at(s);
            const uint64_t tiles = pool.n_kv_heads * sq.tiles_per_head(), row_tiles = (uint64_t)pool.n_kv_heads * sq.row_tiles;
            if (s == lane) my_tiles = tiles, my_units = row_tiles;
            total += tiles;
            units += row_tiles;
            if (row_tiles > 0) longest = max(longest, sq.tiles(sq.row_tiles - 1));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            total += __shfl_xor_sync(0xffffffffu, total, o);
            units += __shfl_xor_sync(0xffffffffu, units, o);
        }
        longest = __reduce_max_sync(0xffffffffu, longest);
        // Equal runs cut row tiles; runs of whole ones are not equal, but nothing is cut, which saves a row tile's cost and a part to join. (512 rows of 8
        // heads from position 0, 128 row tiles of 1 to 4 key tiles: 23 us cut, 19 whole.)
        const uint64_t ctas = gridDim.x, units_each = (units + ctas - 1) / ctas;
        const bool whole = units_each * (longest + kRowTileCost) <= (total + kRowTileCost * units) / ctas + kRowTileCost + 1;
        const uint64_t counted = whole ? units : total + kRowTileCost * units, runs = min(ctas, counted);
        // Where the run begins, and the key tiles ahead of it; the other warp, where it ends.
        const bool begin = warp == kCopyWarp;
        const uint64_t place = blockIdx.x < runs ? counted * (blockIdx.x + (begin ? 0 : 1)) / runs : counted;
        uint64_t ahead = place < counted ? 0 : total;
        ChunkCursor cur{};
        cur.whole = whole;
        if (place < counted) {
            uint64_t base = 0;
            for (uint32_t s0 = 0; s0 < p.rows.n_seqs; s0 += 32) {
                uint64_t tiles = my_tiles, row_tiles = my_units;
                if (s0 > 0) {
                    tiles = row_tiles = 0;
                    if (s0 + lane < p.rows.n_seqs) {
                        const ChunkSeq sq = seq_at(s0 + lane);
                        tiles = pool.n_kv_heads * sq.tiles_per_head();
                        row_tiles = (uint64_t)pool.n_kv_heads * sq.row_tiles;
                    }
                }
                const uint64_t mine = whole ? row_tiles : tiles + kRowTileCost * row_tiles;
                uint64_t upto = mine, tiles_upto = tiles;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint64_t other = __shfl_up_sync(0xffffffffu, upto, o), other_tiles = __shfl_up_sync(0xffffffffu, tiles_upto, o);
                    if (lane >= (uint32_t)o) upto += other, tiles_upto += other_tiles;
                }
                const uint32_t beyond = __ballot_sync(0xffffffffu, base + upto > place);
                const int who = beyond ? __ffs(beyond) - 1 : 31;
                base += __shfl_sync(0xffffffffu, beyond ? upto - mine : upto, who);
                ahead += __shfl_sync(0xffffffffu, beyond ? tiles_upto - tiles : tiles_upto, who);
                if (beyond) {
                    cur.seq = s0 + who;
                    break;
                }
            }
            cur.s = seq_at(cur.seq);
            const uint64_t tiles_per_head = cur.s.tiles_per_head(), per_head = whole ? cur.s.row_tiles : tiles_per_head + (uint64_t)kRowTileCost * cur.s.row_tiles;
            const uint64_t in_seq = place - base, in_head = in_seq % per_head;
            cur.head = (uint32_t)(in_seq / per_head);
            if (whole) {
                cur.row_tile = (uint32_t)in_head;
                cur.at = 0;
            } else {
                // The last row tile that begins at or before in_head: 32 candidates at a time.
                uint32_t lo = 0, span = cur.s.row_tiles;
                while (span > 1) {
                    const uint32_t step = (span + 31) / 32, r = lo + lane * step;
                    const uint32_t below = __ballot_sync(0xffffffffu, lane * step < span && cur.s.counted_before(r) <= in_head);
                    const uint32_t who = 31 - __clz(below);  // lane 0's holds
                    lo += who * step;
                    span = min(step, span - who * step);
                }
                cur.row_tile = lo;
                cur.at = in_head - cur.s.counted_before(lo);
            }
            cur.count = cur.s.tiles(cur.row_tile);
            ahead += cur.head * tiles_per_head + cur.s.tiles_before(cur.row_tile);
            if (cur.at > kRowTileCost) ahead += cur.at - kRowTileCost;
            cur.end = counted * (blockIdx.x + 1) / runs;
            cur.left = cur.end - place;
        }
        if (lane == 0) sh.ahead[begin ? 0 : 1] = ahead;
        if (lane == 0 && begin) {
            sh.counted = counted;
            sh.place.cut = ChunkHead{};
            sh.place.cursor = cur;
            sh.place.unit.tiles = sh.place.in_unit = 0;
            sh.place.unit_number = ~0u;
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = sh.tmem;
    const uint32_t n_tiles = (uint32_t)(sh.ahead[1] - sh.ahead[0]);
    bool alive = true;

    if (warp < kRowWarps) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRowRegisters));
        const uint32_t part = warp >> 2, row = (warp & 3) * 32 + lane;
        constexpr uint32_t kScores = KT / kParts, kSums = HD / kParts;  // of a thread
        const uint32_t first_score = part * kScores, first_sum = part * kSums;
        const uint32_t lanes = tmem + ((warp & 3) << 21);
        const float scale = 1.4426950408889634f / sqrtf((float)HD) / 16384.f;
        float factor = 0.f;
        // The warps that share 32 rows wait for one another, and for nobody else's.
        WarpsBarrier sharers{rows_bar + 8 * (warp & 3), 0, 13};
        auto rows_sync = [&]() { sharers.sync(alive, dead); };

        // The next unit's queries, a thread half of a row: its largest element goes to 2^14 (see kernels_attention_paged.cu). The other half's
        // largest comes through shared memory.
        auto load_queries = [&](uint32_t tile) {
            await(alive, described + 8 * (tile % kDescRing), (tile / kDescRing) & 1, dead, 9);
            if (!alive) return;
            const TileDesc& d = sh.desc[tile % kDescRing];
            const uint32_t query = row / p.group;
            const bool there = query < d.n;
            const uint64_t mine = there ? (uint64_t)(d.row0 + query) * p.q_stride + (uint64_t)(d.head * p.group + row % p.group) * p.q_head_stride : ~0ull;
            uint64_t from[4];  // of the quad's rows
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) {
                from[r] = __shfl_sync(0xffffffffu, mine, (lane & ~3u) + r);
                if (from[r] != ~0ull) from[r] += part * kSums + 4 * (lane & 3);
            }
            // 32 elements at a time, in loops: twice the memory costs less than a thousand instructions in a line (heads of 256: 27000 cycles so, 8000 in loops).
            using Block = float4[2][4];
            auto load = [&](uint32_t block, Block& v) {
#pragma unroll
                for (uint32_t i = 0; i < 2; ++i)
#pragma unroll
                    for (uint32_t r = 0; r < 4; ++r)
                        v[i][r] = from[r] != ~0ull ? *reinterpret_cast<const float4*>(p.q + from[r] + 32 * block + 16 * i) : make_float4(0.f, 0.f, 0.f, 0.f);
            };
            auto larger = [](uint32_t most, const float4& x) {
                return max(max(most, __float_as_uint(x.x) & 0x7fffffffu), max(__float_as_uint(x.y) & 0x7fffffffu, max(__float_as_uint(x.z) & 0x7fffffffu, __float_as_uint(x.w) & 0x7fffffffu)));
            };
            Block v;
            uint32_t tops[4] = {0, 0, 0, 0};  // of the quad's rows, this lane's elements
#pragma unroll 1
            for (uint32_t block = 0; block < kSums / 32; ++block) {
                load(block, v);
#pragma unroll
                for (uint32_t i = 0; i < 2; ++i)
#pragma unroll
                    for (uint32_t r = 0; r < 4; ++r) tops[r] = larger(tops[r], v[i][r]);
            }
            uint32_t top = 0;
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) {
                tops[r] = max(tops[r], __shfl_xor_sync(0xffffffffu, tops[r], 1));
                tops[r] = max(tops[r], __shfl_xor_sync(0xffffffffu, tops[r], 2));
                if ((lane & 3) == r) top = tops[r];
            }
            if (kSums > 32) load(0, v);
            sh.most[0][part][row] = __uint_as_float(top);
            rows_sync();
#pragma unroll
            for (uint32_t i = 0; i < kParts; ++i) top = max(top, __float_as_uint(sh.most[0][i][row]));
            rows_sync();
            if (!alive) return;
            const uint32_t exponent = min(max(top >> 23, 1u), 253u);
            const float up = __uint_as_float((254u - exponent) << 23);
            factor = __uint_as_float(exponent << 23) * scale;
#pragma unroll 1
            for (uint32_t block = 0; block < kSums / 32; ++block) {
#pragma unroll
                for (uint32_t i = 0; i < 2; ++i) {  // 16 elements: 8 columns
                    quad_transpose(v[i], lane);
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) {
                        const float4 x = v[i][e];
                        split_half2(x.x * up * 16384.f, x.y * up * 16384.f, hi[2 * e], lo[2 * e]);
                        split_half2(x.z * up * 16384.f, x.w * up * 16384.f, hi[2 * e + 1], lo[2 * e + 1]);
                    }
                    const uint32_t sixteen = 2 * block + i;
                    tmem_store_8(lanes + kQHi + part * (kSums / 2) + 8 * sixteen, hi);
                    if constexpr (kQLoShared) {
                        uint8_t* to = sh.q_lo + (row >> 3) * kKeyStep + (part * (kSums / 8) + 2 * sixteen) * kCore + (row & 7) * 16;
                        *reinterpret_cast<uint4*>(to) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                        *reinterpret_cast<uint4*>(to + kCore) = make_uint4(lo[4], lo[5], lo[6], lo[7]);
                    } else {
                        tmem_store_8(lanes + kQLo + part * (kSums / 2) + 8 * sixteen, lo);
                    }
                }
                if (block + 1 < kSums / 32) load(block + 1, v);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            if (kQLoShared) fence_proxy_async();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_ready);
        };
        float2 o[kSums / 2];
        float top = 0.f, total = 0.f, unit = 0.f;
        uint32_t lowest = 0;   // 8-bit values: the smallest scale so far
        float heaviest = 0.f;  // of the row's largest exponential times scale so far, no more than the logarithm (where scales differ)
        int32_t limit = 0;  // the last position that the row sees, negative for none
        // Sums become o keep + product grow.
        auto add_product = [&](uint32_t tile, float keep, float grow) {
            await(alive, pv_full + 8 * (tile & 1), (tile >> 1) & 1, dead, 1);
            if (!alive) return;
            tc_fence_after_sync();
            const float2 keep2 = make_float2(keep, keep), grow2 = make_float2(grow, grow);
#pragma unroll
            for (uint32_t c = 0; c < kSums; c += 16) {
                float v[16];
                tmem_load_16(lanes + kPv + first_sum + c, v);
#pragma unroll
                for (uint32_t i = 0; i < 16; i += 2) {
                    float2 add = make_float2(v[i], v[i + 1]);
                    if (FMT == BC_I8) add = mul2(add, grow2);
                    o[(c + i) / 2] = fma2(o[(c + i) / 2], keep2, add);
                }
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(pv_free);
        };
        // 16 scores of a tile from score c on, scaled and masked.
        // The scales are asked for ahead of the scores: nothing moves across a wait for tensor memory.
        auto load_scores = [&](uint32_t scores_at, const TileInfo<KT, FMT>& info, bool masked, int32_t see, uint32_t c, float2 (&x)[8]) {
            float4 d[4];
            if constexpr (FMT == BC_I8) {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) d[i] = *reinterpret_cast<const float4*>(info.dk + first_score + c + 4 * i);
            }
            tmem_load_16(scores_at + c, reinterpret_cast<float(&)[16]>(x));
            if constexpr (FMT == BC_I8) {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    x[2 * i] = mul2(x[2 * i], make_float2(d[i].x, d[i].y));
                    x[2 * i + 1] = mul2(x[2 * i + 1], make_float2(d[i].z, d[i].w));
                }
            }
            if (masked) {
                const uint32_t bits = seen_bits(info, first_score + c, see - (int32_t)c);
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {
                    if (!(bits >> (2 * i) & 1)) x[i].x = -INFINITY;
                    if (!(bits >> (2 * i + 1) & 1)) x[i].y = -INFINITY;
                }
            }
        };
        // The tile's scores to probabilities, in place: of each 16 the upper halves, then the lower. 16 at a time, twice (for their maximum, then again), in loops of 16 and not
        // more: roles run side by side, and what bounds all of them is that they fetch each other's instructions away (2048 rows over 10000 positions: 672 us; 730
        // with two of them in a line, 950 with all four; scores kept in registers between the two, 10 % slower than read twice).
        // PLAIN: every row sees all of the tile, and 8-bit values' weights are counted by tile (`differ`).
        auto take = [&](auto plain, bool by_row, uint32_t tile, float& keep, float& grow) {
            constexpr bool PLAIN = decltype(plain)::value, MAY_BY_ROW = !PLAIN && FMT == BC_I8;
            const uint32_t scores_at = lanes + (tile & 1) * KT + first_score;
            const TileInfo<KT, FMT>& info = sh.info[tile % kRing];
            const int32_t see = (int32_t)max(min((int64_t)limit - sh.desc[tile % kDescRing].key0 - first_score, (int64_t)KT), (int64_t)-1);  // the last score seen
            const bool masked = !PLAIN && info.masked;
            float most[2] = {-INFINITY, -INFINITY};
#pragma unroll 1
            for (uint32_t c = 0; c < kScores; c += 16) {
                float2 x[8];
                load_scores(scores_at, info, masked, see, c, x);
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) most[i & 1] = fmaxf(most[i & 1], fmaxf(x[i].x, x[i].y));
            }
            float tile_top = fmaxf(most[0], most[1]) * factor;
            sh.most[tile & 1][part][row] = tile_top;
            rows_sync();
            if (!alive) return;
            tile_top = fmaxf(tile_top, sh.most[tile & 1][part ^ 1][row]);
            const float now = fmaxf(top, tile_top);
            const float shift = now == -INFINITY ? 0.f : now;
            const float fall = exp2_fast(top - shift), before = top;
            top = now;
            float down = kLift - shift, tile_unit = 1.f;
            if constexpr (FMT == BC_I8) {
                const uint4 tops = *reinterpret_cast<const uint4*>(info.top_scale);
                int exponent = (int)(max(max(tops.x, tops.y), max(tops.z, tops.w)) >> 23) - 127;
                if constexpr (MAY_BY_ROW) {
                    if (by_row) {
                        const uint4 lows = *reinterpret_cast<const uint4*>(info.low_scale);
                        auto exponent_of = [](uint32_t bits) { return bits ? (float)(int)(bits >> 23) - 127.f : -INFINITY; };
                        heaviest = fmaxf(heaviest, fmaxf(before + exponent_of(lowest), tile_top + exponent_of(min(min(lows.x, lows.y), min(lows.z, lows.w)))));
                        // The same for both threads of a row, so for both warps.
                        if (__any_sync(0xffffffffu, now + (float)(exponent - 6) > heaviest || exponent >= 100)) {
                            float mine = -INFINITY;
#pragma unroll 1
                            for (uint32_t c = 0; c < kScores; c += 16) {
                                float2 x[8];
                                load_scores(scores_at, info, masked, see, c, x);
#pragma unroll
                                for (uint32_t i = 0; i < 8; ++i) {
                                    const float2 d = *reinterpret_cast<const float2*>(info.dv + first_score + c + 2 * i);
                                    mine = fmaxf(mine, fmaxf(fmaf(x[i].x, factor, log2_fast(d.x)), fmaf(x[i].y, factor, log2_fast(d.y))));
                                }
                            }
                            sh.heaviest[tile & 1][part][row] = mine;
                            rows_sync();
                            if (!alive) return;
                            mine = floorf(fmaxf(mine, sh.heaviest[tile & 1][part ^ 1][row]) - shift);
                            heaviest = fmaxf(heaviest, mine + shift);
                            exponent = (int)fmaxf(mine, -128.f);
                        }
                    }
                }
                exponent = min(max(exponent, -100), 100);
                tile_unit = __uint_as_float((uint32_t)(exponent + 127) << 23);
                down -= (float)exponent;
            }
            const float2 factor2 = make_float2(factor, factor), down2 = make_float2(down, down);
            float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll 1
            for (uint32_t c = 0; c < kScores; c += 16) {
                float2 x[8];
                load_scores(scores_at, info, masked, see, c, x);
                uint32_t hi[8], lo[8];
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {
                    x[i] = fma2(x[i], factor2, down2);
                    x[i].x = exp2_fast(x[i].x);
                    x[i].y = exp2_fast(x[i].y);
                    sum[i & 1] = add2(sum[i & 1], x[i]);
                }
                if constexpr (FMT == BC_I8) {
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) {
                        const float4 d = *reinterpret_cast<const float4*>(info.dv + first_score + c + 4 * i);
                        x[2 * i] = mul2(x[2 * i], make_float2(d.x, d.y));
                        x[2 * i + 1] = mul2(x[2 * i + 1], make_float2(d.z, d.w));
                    }
                    if (masked) {  // a scale may be no number
                        const uint32_t bits = seen_bits(info, first_score + c, see - (int32_t)c);
#pragma unroll
                        for (uint32_t i = 0; i < 8; ++i) {
                            if (!(bits >> (2 * i) & 1)) x[i].x = 0.f;
                            if (!(bits >> (2 * i + 1) & 1)) x[i].y = 0.f;
                        }
                    }
                }
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) cut_half2(x[i], hi[i], lo[i]);
                tmem_store_8(scores_at + c, hi);
                tmem_store_8(scores_at + c + 8, lo);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            total = total * fall + ((sum[0].x + sum[1].x) + (sum[0].y + sum[1].y)) * tile_unit;
            if constexpr (FMT == BC_I8) {
                // The sums' unit follows the larger of what they were and what this tile brings.
                const float target = fmaxf(unit * fall, tile_unit);
                const uint32_t exponent = min(max(__float_as_uint(target) >> 23, 1u), 253u);
                const float next = __uint_as_float(exponent << 23), inverse = __uint_as_float((254u - exponent) << 23);
                keep = fall * (unit * inverse);
                grow = tile_unit * inverse;
                unit = next;
            } else {
                keep = fall;
                grow = 1.f;
                unit = 1.f;
            }
        };
        // 8-bit values: weights, probabilities times scales, are counted in the power of two below the tile's largest scale, 2^14 to one, and are exact to
        // 2^-25 of these. A row's largest weight is the unit's smallest scale so far at the least. From where that is less than 2^-7 of a tile's largest scale,
        // which may be of a position that a row does not see, or hardly, rows look closer: the largest weight is at least a tile's largest probability times its
        // smallest scale; where 32 rows find one for which that is too little, too, each counts in the power of two below its own largest weight.
        // So a weight keeps 22 bits, or 2^-32 of its row's largest.
        auto differ = [&](uint32_t tile) {
            if constexpr (FMT == BC_I8) {
                const TileInfo<KT, FMT>& info = sh.info[tile % kRing];
                const uint4 tops = *reinterpret_cast<const uint4*>(info.top_scale), lows = *reinterpret_cast<const uint4*>(info.low_scale);
                lowest = min(lowest, min(min(lows.x, lows.y), min(lows.z, lows.w)));
                return (max(max(tops.x, tops.y), max(tops.z, tops.w)) >> 23) > min(lowest >> 23, 220u) + 6;
            } else {
                return false;
            }
        };
        auto publish = [&](uint32_t tile) {
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_ready + 8 * (tile & 1));
        };
        // A row's results: whole, or a part for the joining launch. `sums` are those of the row's elements from first_element on.
        auto store = [&](const TileDesc& desc, uint32_t first_element, const float2 (&sums)[HD / kParts / 2], float times, bool stats) {
            const bool whole = desc.begins && desc.ends;
            const uint32_t slot = 2 * blockIdx.x + (desc.begins ? 1 : 0);
            if (whole) times *= top == -INFINITY && total == 0.f ? 0.f : 1.f / total;
            const uint64_t mine = row / p.group >= desc.n ? ~0ull
                                  : whole ? (uint64_t)(desc.row0 + row / p.group) * p.n_heads * HD + (desc.head * p.group + row % p.group) * HD
                                          : ((uint64_t)slot * kRows + row) * HD;
            float* const to = (whole ? p.out : p.parts) + first_element + 4 * (lane & 3);
            const bool any = FMT == BC_F16 && sh.any_not_finite[desc.unit % kUnits];
#pragma unroll
            for (uint32_t i = 0; i < HD / kParts / 16; ++i) {
                float4 v[4];
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) {
                    const float2 a = sums[8 * i + 2 * k], b = sums[8 * i + 2 * k + 1];
                    v[k] = make_float4(a.x * times, a.y * times, b.x * times, b.y * times);
                }
                quad_transpose(v, lane);
#pragma unroll
                for (uint32_t r = 0; r < 4; ++r) {
                    const uint64_t at = __shfl_sync(0xffffffffu, mine, (lane & ~3u) + r);
                    if (at != ~0ull) *reinterpret_cast<float4*>(to + at + 16 * i) = v[r];
                }
            }
            if (any) {  // after the quad's stores
                __syncwarp();
                const uint32_t* at = sh.not_finite[desc.unit % kUnits] + first_element;
                if (mine != ~0ull)
#pragma unroll 1
                    for (uint32_t e = 0; e < HD / kParts; ++e)
                        if ((int64_t)at[FMT == BC_F16 ? e : 0] <= limit) (whole ? p.out : p.parts)[mine + first_element + e] = __uint_as_float(0x7fc00000u);
            }
            if (FMT == BC_F16 && whole && mine != ~0ull && total != total) sh.odd = 1;
            if (!whole && stats)
                *reinterpret_cast<float2*>(p.parts + (uint64_t)2 * kMostCtas * kRows * HD + ((uint64_t)slot * kRows + row) * 2) = make_float2(top, total);
        };
        auto start_unit = [&](uint32_t tile) {
            // (Rows that are nobody's see all there is: no tile is masked for them.)
            const TileDesc& desc = sh.desc[tile % kDescRing];
            const uint32_t query = row / p.group;
            limit = (int32_t)min((int64_t)desc.pos0 + (query < desc.n ? query : 0x40000000u), (int64_t)desc.end - 1);
#pragma unroll
            for (uint32_t i = 0; i < kSums / 2; ++i) o[i] = make_float2(0.f, 0.f);
            top = -INFINITY;
            total = unit = 0.f;
            lowest = 0x7f7fffff;
            heaviest = -INFINITY;
        };
        // All rows' threads take every tile; the last product is added to the sums when the next tile's probabilities are there.
        uint32_t tile = 0;
        float keep = 0.f, grow = 0.f;
        bool begins = true;  // the tile is its unit's first
        // Tiles up to the unit's last; PLAIN: false at one that is not. Most of a long unit's are, and a loop for these alone is the shorter one.
        auto take_tiles = [&](auto plain) {
            while (true) {
                await(alive, s_full + 8 * (tile & 1), (tile >> 1) & 1, dead, 2);
                if (!alive) return true;
                tc_fence_after_sync();
                const bool by_row = differ(tile);
                if (decltype(plain)::value && (by_row || sh.info[tile % kRing].masked)) return false;
                float next_keep, next_grow;
                take(plain, by_row, tile, next_keep, next_grow);
                if (!begins && alive) add_product(tile - 1, keep, grow);  // before the next one may take its place
                if (!alive) return true;
                keep = next_keep;
                grow = next_grow;
                begins = false;
                publish(tile);
                if (sh.desc[tile++ % kDescRing].last) return true;
            }
        };
        while (n_tiles > 0) {
            // The next unit's queries go ahead of the last one's end, whose scores are done, where registers hold both.
            if (tile > 0) rows_sync();  // the maxima have been read
            if (HD < 256 && tile < n_tiles && alive) load_queries(tile);
            if (tile > 0 && alive) {
                add_product(tile - 1, keep, grow);
                // A row's sums of probabilities meet.
                sh.most[0][part][row] = total;
                rows_sync();
                total = sh.most[0][0][row] + sh.most[0][1][row];
                rows_sync();  // the next unit writes there
                if (!alive) break;
                store(sh.desc[(tile - 1) % kDescRing], first_sum, o, unit, part == 0);
            }
            if (HD == 256 && tile < n_tiles && alive) load_queries(tile);
            if (tile == n_tiles || !alive) break;
            start_unit(tile);
            begins = true;
            if (!take_tiles(std::true_type{})) take_tiles(std::false_type{});
            if (!alive) break;
        }
    } else if (warp < kMmaWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kUnpackRegisters));
        // ---- bytes to operands
        const uint32_t utid = tid - kRowThreads, uwarp = utid >> 5;
        constexpr uint32_t kPieces = KT * (HD / 8) / kUnpackThreads;           // pieces of 8 elements of a key that a thread unpacks
        constexpr uint32_t kBlocks = KT / 8 * (HD / 8) / kUnpackThreads;       // blocks of 8 positions x 8 elements of values
        constexpr uint32_t kPiece = FMT == BC_F16 ? 16 : 8, kWords = kPiece / 4, kRowBytes = RawKeys<KT, FMT, HD>::kRowBytes;
        WarpsBarrier everyone{unpack_bar, 0, 14};
        // Keys one tile ahead of values: the next scores need no more, while the values' place waits for a product.
        for (uint32_t i = 0; i <= n_tiles && n_tiles > 0; ++i) {
            if (i < n_tiles) {
                const uint32_t j = i, st = j % ST;
                TileInfo<KT, FMT>& info = sh.info[j % kRing];
                const RawKeys<KT, FMT, HD>& raw = sh.raw_keys[j % RAW];
                await(alive, rk_full + 8 * (j % RAW), (j / RAW) & 1, dead, 10);
                if (!alive) break;
                const TileDesc& desc = sh.desc[j % kDescRing];
                const uint32_t key0 = desc.key0, end = desc.end, groups = desc.groups;
                auto key_there = [&](uint32_t key) { return (groups >> (key >> 4) & 1) && key0 + key < end; };
                const bool whole = groups == (1u << KT / 16) - 1 && end - key0 >= KT;  // every position is there
                // Free keys: their scores are done, so the rows' warps are done with the tile before those, and the ring's fourth is nobody's.
                await(alive, k_free + 8 * st, ((j / ST) & 1) ^ 1, dead, 3);
                if (!alive) break;
                if constexpr (FMT == BC_F16) {
                    if (desc.first) {
                        const uint32_t slot = desc.unit % kUnits;
                        for (uint32_t e = utid; e < HD; e += kUnpackThreads) sh.not_finite[slot][e] = 0xffffffffu;
                        if (utid == 0) sh.any_not_finite[slot] = 0;
                        everyone.sync(alive, dead);  // before any of them finds one
                        if (!alive) break;
                    }
                }
                // Masks and scales of the tile's positions.
                const bool there = utid < KT && key_there(utid);
                const uint32_t votes = __ballot_sync(0xffffffffu, there);
                if (lane == 0 && uwarp < KT / 32) info.valid[uwarp] = votes;
                if (utid == 0) info.masked = !whole || (int64_t)key0 + KT - 1 > desc.pos0;
                if constexpr (FMT == BC_I8) {
                    const float dv = there ? raw.dv[utid] : 0.f;
                    if (utid < KT) {
                        info.dk[utid] = there ? raw.dk[utid] : 0.f;
                        info.dv[utid] = dv;
                    }
                    const uint32_t bits = __float_as_uint(dv) & 0x7fffffffu;
                    const uint32_t largest = __reduce_max_sync(0xffffffffu, bits < 0x7f800000u ? bits : 0u);
                    const uint32_t smallest = __reduce_min_sync(0xffffffffu, there && bits < 0x7f800000u ? bits : 0x7f7fffffu);
                    if (lane == 0) info.top_scale[uwarp] = largest, info.low_scale[uwarp] = smallest;
                }
                {  // What is there of positions that are not is masked in the scores, whatever it is.
                    const uint8_t* from = raw.keys + utid * kPiece;
                    uint8_t* const to = sh.keys[st];
#pragma unroll 4
                    for (uint32_t n = 0; n < kPieces; ++n) {
                        const uint32_t at = utid + n * kUnpackThreads, piece = at % (HD / 8), key = at / (HD / 8);
                        uint4 w;
                        if constexpr (FMT == BC_F16) {
                            w = *reinterpret_cast<const uint4*>(from + n * kUnpackThreads * kPiece);
                        } else {
                            const uint2 b = *reinterpret_cast<const uint2*>(from + n * kUnpackThreads * kPiece);
                            unpack_i8(b.x, w.x, w.y);
                            unpack_i8(b.y, w.z, w.w);
                        }
                        *reinterpret_cast<uint4*>(to + (key >> 3) * kKeyStep + piece * kCore + (key & 7) * 16) = w;
                    }
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(k_full + 8 * st);
                    mbar_arrive(rk_free + 8 * (j % RAW));
                }
            }
            if (i == 0) continue;
            const uint32_t j = i - 1, st = j % ST;
            const TileDesc& desc = sh.desc[j % kDescRing];
            const uint32_t key0 = desc.key0, end = desc.end, groups = desc.groups;
            auto key_there = [&](uint32_t key) { return (groups >> (key >> 4) & 1) && key0 + key < end; };
            const bool whole = groups == (1u << KT / 16) - 1 && end - key0 >= KT;
            await(alive, rv_full + 8 * (j % RAW), (j / RAW) & 1, dead, 15);
            await(alive, v_free + 8 * st, ((j / ST) & 1) ^ 1, dead, 4);
            if (!alive) break;
            uint8_t* const to = sh.values[st];
            // A value that is not finite would reach rows that do not see it: zero times it is no number. Tiles that end behind the row tile's
            // first row keep such values apart.
            const bool apart = FMT == BC_F16 && (int64_t)key0 + KT - 1 > desc.pos0;
#pragma unroll 1
            for (uint32_t n = 0; n < kBlocks; ++n) {
                const uint32_t at = utid + n * kUnpackThreads, piece = at % (HD / 8), key = at / (HD / 8) * 8;
                const uint8_t* from = sh.raw_values[j % RAW] + key * kRowBytes + piece * kPiece;
                uint4* const core = reinterpret_cast<uint4*>(to + piece * kCore + (key >> 3) * kKeyStep);  // 8 elements x 8 positions
                uint32_t v[8][kWords];
#pragma unroll
                for (uint32_t r = 0; r < 8; ++r) {
                    if constexpr (FMT == BC_F16) {
                        const uint4 w = *reinterpret_cast<const uint4*>(from + r * kRowBytes);
                        v[r][0] = w.x, v[r][1] = w.y, v[r][2] = w.z, v[r][3] = w.w;
                    } else {
                        const uint2 w = *reinterpret_cast<const uint2*>(from + r * kRowBytes);
                        v[r][0] = w.x, v[r][1] = w.y;
                    }
                }
                if (!whole) {
#pragma unroll
                    for (uint32_t r = 0; r < 8; ++r)
                        if (!key_there(key + r))
#pragma unroll
                            for (uint32_t w = 0; w < kWords; ++w) v[r][w] = FMT == BC_F16 ? 0u : 0x80808080u;
                }
                if constexpr (FMT == BC_F16) {
                    if (apart) {
                        uint32_t any = 0;
#pragma unroll
                        for (uint32_t r = 0; r < 8; ++r)
#pragma unroll
                            for (uint32_t w = 0; w < kWords; ++w) any |= (v[r][w] & 0x7c007c00u) + 0x04000400u;  // exponents of all ones carry
                        if (any & 0x80008000u) {
#pragma unroll
                            for (uint32_t r = 0; r < 8; ++r)
#pragma unroll
                                for (uint32_t w = 0; w < kWords; ++w)
#pragma unroll
                                    for (uint32_t e = 0; e < 2; ++e)
                                        if ((v[r][w] >> (16 * e) & 0x7c00u) == 0x7c00u) {
                                            const uint32_t slot = desc.unit % kUnits;
                                            atomicMin(&sh.not_finite[slot][8 * piece + 2 * w + e], key0 + key + r);
                                            sh.any_not_finite[slot] = 1;
                                            v[r][w] &= ~(0xffffu << (16 * e));
                                        }
                        }
                    }
#pragma unroll
                    for (uint32_t w = 0; w < 4; ++w) {
                        uint32_t even[4], odd[4];
#pragma unroll
                        for (uint32_t r = 0; r < 4; ++r) {
                            even[r] = __byte_perm(v[2 * r][w], v[2 * r + 1][w], 0x5410);
                            odd[r] = __byte_perm(v[2 * r][w], v[2 * r + 1][w], 0x7632);
                        }
                        core[2 * w] = make_uint4(even[0], even[1], even[2], even[3]);
                        core[2 * w + 1] = make_uint4(odd[0], odd[1], odd[2], odd[3]);
                    }
                } else {
#pragma unroll
                    for (uint32_t w = 0; w < 2; ++w)
#pragma unroll
                        for (uint32_t h = 0; h < 2; ++h) {  // elements 4w + 2h and the next
                            uint32_t even[4], odd[4];
#pragma unroll
                            for (uint32_t r = 0; r < 4; ++r) unpack_i8(__byte_perm(v[2 * r][w], v[2 * r + 1][w], h ? 0x7362 : 0x5140), even[r], odd[r]);
                            core[4 * w + 2 * h] = make_uint4(even[0], even[1], even[2], even[3]);
                            core[4 * w + 2 * h + 1] = make_uint4(odd[0], odd[1], odd[2], odd[3]);
                        }
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(v_full + 8 * st);
                mbar_arrive(rv_free + 8 * (j % RAW));
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegisters));
        if (warp == kMmaWarp) {
            // ---- the tensor core. Lower halves first: what a sum cuts off grows with what is there already. Every loop and branch goes by a vote: the
            // compiler then keeps the descriptors in uniform registers, where the instruction wants them (without, an instruction took 106 cycles
            // to issue, of the 64 that it runs). In loops too: unrolled, chunks of heads of 256 took 199 us, so 182.
            const uint32_t scores_idesc = umma_idesc_f16(kRows, KT), values_idesc = umma_idesc_f16(kRows, HD);
            const uint64_t q_lo = umma_desc(smem_u32(sh.q_lo), kCore, kKeyStep), keys0 = umma_desc(smem_u32(sh.keys), kCore, kKeyStep),
                           values0 = umma_desc(smem_u32(sh.values), kKeyStep, kCore);
            uint32_t units = 0;
            auto product = [&](uint32_t j) {  // P V of tile j
                await(alive, p_ready + 8 * (j & 1), (j >> 1) & 1, dead, 5);
                if (j > 0) await(alive, pv_free, (j - 1) & 1, dead, 12);
                await(alive, v_full + 8 * (j % ST), (j / ST) & 1, dead, 6);
                if (__any_sync(0xffffffffu, !alive)) return;
                tc_fence_after_sync();
                const uint64_t v = values0 + (j % ST) * (S::kTileBytes >> 4);
                const uint32_t weights = tmem + (j & 1) * KT;
                if (elect_one()) {
#pragma unroll 1
                    for (uint32_t part = 0; part < 2; ++part)
#pragma unroll 1
                        for (uint32_t ks = 0; ks < KT / 16; ++ks)
                            umma_f16_a_tmem(tmem + kPv, weights + ks * 16 + (part ^ 1) * 8, v + (uint64_t)(ks * 2 * kKeyStep >> 4), values_idesc, part | ks);
                }
                __syncwarp();
                if (elect_one()) {
                    umma_commit(v_free + 8 * (j % ST));
                    umma_commit(pv_full + 8 * (j & 1));
                }
                __syncwarp();
            };
            for (uint32_t j = 0; __all_sync(0xffffffffu, j < n_tiles && alive); ++j) {
                await(alive, k_full + 8 * (j % ST), (j / ST) & 1, dead, 7);
                if (__any_sync(0xffffffffu, !alive)) break;
                const bool first = __any_sync(0xffffffffu, sh.desc[j % kDescRing].first != 0);
                if (first) {
                    if (j > 0) product(j - 1);
                    await(alive, q_ready, units & 1, dead, 8);
                    ++units;
                }
                if (__any_sync(0xffffffffu, !alive)) break;
                tc_fence_after_sync();
                const uint64_t keys = keys0 + (j % ST) * (S::kTileBytes >> 4);
                const uint32_t to = tmem + (j & 1) * KT;
                if (elect_one()) {
#pragma unroll 1
                    for (uint32_t ks = 0; ks < HD / 16; ++ks) {
                        if constexpr (kQLoShared)
                            umma_f16(to, q_lo + (uint64_t)(ks * 2 * kCore >> 4), keys + (uint64_t)(ks * 2 * kCore >> 4), scores_idesc, ks);
                        else
                            umma_f16_a_tmem(to, tmem + kQLo + ks * 8, keys + (uint64_t)(ks * 2 * kCore >> 4), scores_idesc, ks);
                    }
#pragma unroll 1
                    for (uint32_t ks = 0; ks < HD / 16; ++ks) umma_f16_a_tmem(to, tmem + kQHi + ks * 8, keys + (uint64_t)(ks * 2 * kCore >> 4), scores_idesc, 1);
                }
                __syncwarp();
                if (elect_one()) {
                    umma_commit(k_free + 8 * (j % ST));
                    umma_commit(s_full + 8 * (j & 1));
                }
                __syncwarp();
                if (!first) product(j - 1);
            }
            if (__all_sync(0xffffffffu, n_tiles > 0 && alive)) product(n_tiles - 1);
        } else if (warp == kCopyWarp) {
            // ---- the walk through the run, and the pages' bytes: a lane per 16 positions of keys, values, and either's scales. What lies in one page
            // is one copy, the first of its lanes': copies' number, not their bytes, is what the copying engine's time goes by (tiles of 128 positions
            // in 32 copies kept everyone waiting).
            Place& at = sh.place;
            constexpr uint32_t kGroups = KT / 16, kRowBytes = RawKeys<KT, FMT, HD>::kRowBytes;
            const uint32_t page_slots = (1u << pool.page_shift) - 1;
            uint32_t keys_issued = 0, values_issued = 0;
            const uint32_t group = lane % kGroups, what = lane / kGroups;
            const uint32_t segment = min(page_slots + 1, KT);  // positions of a copy
            const bool leads = group * 16 % segment == 0;
            uint32_t value_segments = 0;  // of the tile before
            uint64_t value_rows_at = ~0ull;  // of the tile before
            for (uint32_t i = 0; i <= n_tiles && n_tiles > 0; ++i) {
                uint64_t rows_at = ~0ull;
                uint32_t segments = 0;
                if (i < n_tiles) {
                    const uint32_t j = i;
                    TileDesc& d = sh.desc[j % kDescRing];
                    bool some = true;
                    if (lane == 0 && at.in_unit == at.unit.tiles) {
                        some = at.cursor.take(p.rows.starts, p.rows.lens, p.rows.n_seqs, p.rows.n_rows, pool.n_kv_heads, capacity, p.fewest, at.unit);
                        at.in_unit = 0;
                        if (++at.unit_number == 0 && FMT == BC_F16) at.span = ChunkSpan{{at.unit.seq, 0}, {at.unit.head, 0}, {at.unit.row_tile, 0}, {}};
                    }
                    // The run's tiles have been counted. One that ends before, since the call's words have changed since, is given up here: what the cursor holds then
                    // describes no rows of the call.
                    alive = __all_sync(0xffffffffu, some);
                    if (!alive) {
                        if (lane == 0) give_up(dead, 17);
                        break;
                    }
                    if (lane == 0) {
                        const ChunkUnit& u = at.unit;
                        const ChunkSeq& s = at.cursor.s;
                        const uint32_t query0 = u.row_tile * per_tile;
                        const int64_t pos = (int64_t)s.len - (s.end - s.row0) + query0;
                        d.key0 = (u.tile0 + at.in_unit) * KT;
                        d.end = s.held;
                        d.row0 = s.row0 + query0;
                        d.n = min(per_tile, s.n - query0);
                        d.head = u.head;
                        d.pos0 = (int32_t)max(min(pos, (int64_t)0x7fffffff), -(int64_t)0x7fffffff);
                        d.unit = at.unit_number;
                        d.first = at.in_unit == 0;
                        d.last = at.in_unit + 1 == u.tiles;
                        d.begins = u.begins;
                        d.ends = u.ends;
                        if (s.held < s.len) leave_fault(pool, kFaultTable);
                        if (u.begins && !u.ends && at.in_unit == 0) {
                            // The CTA whose run holds the row tile's end: run c is [total c / runs, total (c + 1) / runs).
                            const uint64_t total = sh.counted, runs = min((uint64_t)gridDim.x, total);
                            uint32_t last = (uint32_t)(u.last * runs / total);
                            while (total * (last + 1) / runs <= u.last) ++last;
                            while (total * last / runs > u.last) --last;
                            at.cut = ChunkHead{d.row0, d.n, d.head, last};
                        }
                        ++at.in_unit;
                        mbar_arrive(described + 8 * (j % kDescRing));  // but for the groups, which the copies' arrival shows
                    }
                    __syncwarp();
                    // Every lane looks up its group's page.
                    const uint32_t key = d.key0 + 16 * group;
                    uint32_t page = ~0u;
                    if (key < d.end) {
                        page = p.rows.table[(uint64_t)at.unit.seq * p.rows.max_pages + (key >> pool.page_shift)];
                        if (page >= pool.n_pages) leave_fault(pool, kFaultPage);
                    }
                    const bool there = page < pool.n_pages;
                    const uint32_t groups = __ballot_sync(0xffffffffu, there) & ((1u << kGroups) - 1);
                    segments = __popc(__ballot_sync(0xffffffffu, there && leads) & ((1u << kGroups) - 1));
                    if (there && leads) rows_at = kv_row_at(pool, page, d.head, key & page_slots);
                    const uint32_t slot = j % RAW, bar = rk_full + 8 * slot;
                    await(alive, rk_free + 8 * slot, ((j / RAW) & 1) ^ 1, dead, 11);
                    if (!alive) break;
                    ++keys_issued;
                    if (lane == 0) {
                        d.groups = groups;
                        mbar_arrive_expect(bar, segments * segment * (kRowBytes + (FMT == BC_I8 ? 8 : 0)));
                    }
                    __syncwarp();
                    if (there && leads) {
                        RawKeys<KT, FMT, HD>& raw = sh.raw_keys[slot];
                        if (what == 0)
                            bulk_load(smem_u32(raw.keys) + group * 16 * kRowBytes, pool.k + rows_at, segment * kRowBytes, bar);
                        else if (FMT == BC_I8 && what < 3)
                            bulk_load(smem_u32(what == 2 ? raw.dv : raw.dk) + group * 64, (what == 2 ? pool.v : pool.k) + kv_scale_at(pool, page, d.head, key & page_slots), segment * 4, bar);
                    }
                    __syncwarp();
                }
                if (i > 0) {
                    const uint32_t j = i - 1, slot = j % RAW, bar = rv_full + 8 * slot;
                    await(alive, rv_free + 8 * slot, ((j / RAW) & 1) ^ 1, dead, 16);
                    if (!alive) break;
                    ++values_issued;
                    if (lane == 0) mbar_arrive_expect(bar, value_segments * segment * kRowBytes);
                    __syncwarp();
                    if (what == 0 && value_rows_at != ~0ull) bulk_load(smem_u32(sh.raw_values[slot]) + group * 16 * kRowBytes, pool.v + value_rows_at, segment * kRowBytes, bar);
                    __syncwarp();
                }
                value_rows_at = rows_at;
                value_segments = segments;
            }
            if (lane == 0) {
                chunk_heads(p.parts, HD)[blockIdx.x] = alive ? at.cut : ChunkHead{};
                if constexpr (FMT == BC_F16) {
                    at.span.seq[1] = at.unit.seq, at.span.head[1] = at.unit.head, at.span.row_tile[1] = at.unit.row_tile;
                    chunk_spans(p.parts, HD)[blockIdx.x] = at.span;
                }
            }
            // Copies in flight end before the CTA does: the unpacking warps wait for them, or this one does when those gave up.
            for (uint32_t r = 0; r < RAW && r < keys_issued && *dead; ++r) {
                const uint32_t j = keys_issued - 1 - r;
                mbar_wait(rk_full + 8 * (j % RAW), (j / RAW) & 1, kSpinLimit, &sh.never);
            }
            for (uint32_t r = 0; r < RAW && r < values_issued && *dead; ++r) {
                const uint32_t j = values_issued - 1 - r;
                mbar_wait(rv_full + 8 * (j % RAW), (j / RAW) & 1, kSpinLimit, &sh.never);
            }
        }
    }
    // Whoever waited for the last product has seen all multiplies end; after a wait that ran out, they get a limited time to.
    tc_fence_before_sync();
    __syncthreads();
    if (FMT == BC_F16 && tid == 0 && sh.odd) chunk_heads(p.parts, HD)[blockIdx.x].n = sh.dead ? 0 : sh.place.cut.n | kOdd;
    if (warp == kMmaWarp) {
        if (sh.dead && n_tiles > 0) {
            if (elect_one()) {
                mbar_init(q_ready, 1);
                mbar_init_fence();
                umma_commit(q_ready);
                for (uint32_t spin = 0; spin < kSpinLimit && !mbar_test(q_ready, 0); ++spin) {}
            }
            __syncwarp();
        }
        tc_fence_after_sync();
        tmem_dealloc(tmem, kTmemColumns);
    }
}

// Attention of one query by a warp, in f32 throughout, with infinities as the formula has them. Rows whose sums are no number are done again by this: a half page may hold
// an infinite key whose score is minus infinity, which weighs nothing, but a query's lower half times it may be plus infinity, or no number.
template <int HD>
__device__ __forceinline__ void attend_in_f32(const ChunkParams& p, uint32_t seq, uint32_t kv_head, const float* q, uint32_t n_keys, float* out) {
    const KvPool& pool = p.pool;
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t* const table = p.rows.table + (uint64_t)seq * p.rows.max_pages;
    float top = -INFINITY, total = 0.f;
    float2 sum[HD / 64];
#pragma unroll
    for (int i = 0; i < HD / 64; ++i) sum[i] = make_float2(0.f, 0.f);
    for (uint32_t key0 = 0; key0 < n_keys; key0 += 32) {
        const uint32_t key = key0 + lane, page = key < n_keys ? table[key >> pool.page_shift] : kNoSlot;
        const bool there = page < pool.n_pages;
        const uint64_t at = there ? kv_row_at(pool, page, kv_head, key & ((1u << pool.page_shift) - 1)) : 0;
        float score = -INFINITY;
        if (there) {
            float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
            for (int e = 0; e < HD; e += 4) {
                const float4 x = *reinterpret_cast<const float4*>(q + e);
                const uint2 w = *reinterpret_cast<const uint2*>(pool.k + at + 2 * e);
                const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
                s[0] = fmaf(x.x, a.x, s[0]);
                s[1] = fmaf(x.y, a.y, s[1]);
                s[2] = fmaf(x.z, b.x, s[2]);
                s[3] = fmaf(x.w, b.y, s[3]);
            }
            score = ((s[0] + s[1]) + (s[2] + s[3])) * (1.4426950408889634f / sqrtf((float)HD));
        }
        if (__any_sync(0xffffffffu, !(score < INFINITY))) {  // so is the row
            for (uint32_t e = lane; e < HD; e += 32) out[e] = __uint_as_float(0x7fc00000u);
            return;
        }
        const float now = fmaxf(top, warp_max(score)), shift = now == -INFINITY ? 0.f : now, fall = exp2f(top - shift), weight = exp2f(score - shift);
        top = now;
        total = total * fall + weight;
#pragma unroll
        for (int i = 0; i < HD / 64; ++i) sum[i] = make_float2(sum[i].x * fall, sum[i].y * fall);
        for (uint32_t left = __ballot_sync(0xffffffffu, there); left; left &= left - 1) {
            const uint32_t who = __ffs(left) - 1;
            const float w = __shfl_sync(0xffffffffu, weight, who);
            const __half2* v = reinterpret_cast<const __half2*>(pool.v + __shfl_sync(0xffffffffu, at, who)) + lane;
#pragma unroll
            for (int i = 0; i < HD / 64; ++i) {
                const float2 x = __half22float2(v[32 * i]);
                sum[i].x = fmaf(w, x.x, sum[i].x);
                sum[i].y = fmaf(w, x.y, sum[i].y);
            }
        }
    }
    total = warp_sum(total);
    const float inverse = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
    for (int i = 0; i < HD / 64; ++i) reinterpret_cast<float2*>(out)[32 * i + lane] = make_float2(sum[i].x * inverse, sum[i].y * inverse);
}

// A row's query head again. (Not in line, nor what follows: the joining launch is short, and most of its time is its beginning.)
template <int HD>
__device__ __noinline__ void again(const ChunkParams& p, uint32_t seq, uint32_t row, uint32_t head) {
    const uint32_t back = p.rows.starts[seq + 1] - row, len = p.rows.lens[seq];
    const uint32_t held = (uint32_t)min((uint64_t)len, (uint64_t)p.rows.max_pages << p.pool.page_shift), n_keys = back <= len ? min(len - back + 1, held) : 0;
    attend_in_f32<HD>(p, seq, head / p.group, p.q + row * p.q_stride + head * p.q_head_stride, n_keys, p.out + ((uint64_t)row * p.n_heads + head) * HD);
}
// The rows of CTA c's units whose sums are no number, by kJoinCtas CTAs; of units that were cut the launch's joining takes care.
template <int HD>
__device__ __noinline__ void again_where_whole(const ChunkParams& p, uint32_t c, uint32_t ctas) {
    const uint32_t lane = threadIdx.x & 31, warp = blockIdx.y * 8 + (threadIdx.x >> 5), per_tile = kRows / p.group;
    const ChunkHead* const heads = chunk_heads(p.parts, HD);
    const ChunkSpan span = chunk_spans(p.parts, HD)[c];
    for (uint32_t seq = span.seq[0]; seq <= span.seq[1]; ++seq) {
        const ChunkSeq s = chunk_seq(p.rows.starts[seq], p.rows.starts[seq + 1], p.rows.lens[seq], (uint64_t)p.rows.max_pages << p.pool.page_shift, p.rows.n_rows, p.fewest, per_tile, 128);
        const bool first = seq == span.seq[0], last = seq == span.seq[1];
        for (uint32_t head = first ? span.head[0] : 0; head <= (last ? span.head[1] : p.pool.n_kv_heads - 1); ++head) {
            const uint32_t tile1 = last && head == span.head[1] ? min(s.row_tiles, span.row_tile[1] + 1) : s.row_tiles;
            for (uint32_t tile = first && head == span.head[0] ? span.row_tile[0] : 0; tile < tile1; ++tile) {
                const uint32_t row0 = s.row0 + tile * per_tile, n = min(per_tile, s.n - tile * per_tile);
                bool joined = false;
                for (uint32_t k = lane; k < ctas; k += 32) joined |= heads[k].last != 0 && heads[k].head == head && heads[k].row0 == row0;
                if (__any_sync(0xffffffffu, joined)) continue;
                for (uint32_t r = warp; r < n * p.group; r += 8 * kJoinCtas) {
                    const uint32_t row = row0 + r / p.group, q_head = head * p.group + r % p.group;
                    const float x = p.out[((uint64_t)row * p.n_heads + q_head) * HD + lane];
                    if (__any_sync(0xffffffffu, x != x)) again<HD>(p, seq, row, q_head);
                }
            }
        }
    }
}

// Joins the parts of a unit that begins in CTA c's run: a warp to a row. Rows of halves whose sums are no number are done again.
template <int FMT, int HD>
__global__ void __launch_bounds__(256, HD == 64 ? 8 : 6) attention_chunk_paged_join_kernel(const __grid_constant__ ChunkParams p, uint32_t ctas) {
    constexpr int kPairs = HD / 64;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x;
    const ChunkHead cut = chunk_heads(p.parts, HD)[c];
    if (cut.last != 0) {
        const float2* stats = reinterpret_cast<const float2*>(p.parts + (uint64_t)2 * kMostCtas * kRows * HD);
        const uint32_t n = cut.last - c + 1;
        auto slot_of = [&](uint32_t i) { return (uint64_t)(2 * (c + i) + (i == 0 ? 1 : 0)); };
        for (uint32_t r = blockIdx.y * 8 + warp; r < (cut.n & ~kOdd) * p.group; r += kJoinCtas * 8) {
            float top = -INFINITY;
            for (uint32_t i = lane; i < n; i += 32) top = fmaxf(top, stats[slot_of(i) * kRows + r].x);
            top = warp_max(top);
            const float shift = top == -INFINITY ? 0.f : top;
            float total = 0.f;
            float2 sum[kPairs];
#pragma unroll
            for (int i = 0; i < kPairs; ++i) sum[i] = make_float2(0.f, 0.f);
            for (uint32_t i0 = 0; i0 < n; i0 += 32) {
                float2 st = make_float2(-INFINITY, 0.f);
                if (i0 + lane < n) st = stats[slot_of(i0 + lane) * kRows + r];
                const float weight = st.x == -INFINITY ? 0.f : exp2f(st.x - shift);
                total += weight * st.y;
                const uint32_t many = min(32u, n - i0);
#pragma unroll 4
                for (uint32_t i = 0; i < many; ++i) {
                    const float w = __shfl_sync(0xffffffffu, weight, i);
                    const bool any = __shfl_sync(0xffffffffu, st.x, i) != -INFINITY;
                    const float2* from = reinterpret_cast<const float2*>(p.parts + (slot_of(i0 + i) * kRows + r) * HD) + lane;
#pragma unroll
                    for (int k = 0; k < kPairs; ++k) {
                        const float2 v = from[32 * k];
                        if (any) {
                            sum[k].x += w * v.x;
                            sum[k].y += w * v.y;
                        }
                    }
                }
            }
            total = warp_sum(total);
            const uint32_t row = cut.row0 + r / p.group, head = cut.head * p.group + r % p.group;
            if (FMT == BC_F16 && total != total) {
                again<HD>(p, seq_of_row(p.rows, row), row, head);
                continue;
            }
            const float inverse = top == -INFINITY && total == 0.f ? 0.f : 1.f / total;
            float2* to = reinterpret_cast<float2*>(p.out + ((uint64_t)row * p.n_heads + head) * HD) + lane;
#pragma unroll
            for (int k = 0; k < kPairs; ++k) to[32 * k] = make_float2(sum[k].x * inverse, sum[k].y * inverse);
        }
    }
    if (FMT == BC_F16 && cut.n & kOdd) again_where_whole<HD>(p, c, ctas);
}

uint32_t chunk_ctas() {
    const uint32_t sms = (uint32_t)sm_count();
    return sms < kMostCtas ? sms : kMostCtas;
}

template <int FMT, int HD>
cudaError_t launch_chunk(cudaStream_t stream, const ChunkParams& p) {
    constexpr size_t smem = sizeof(Shared<FMT, HD>);
    static_assert(smem <= 227 * 1024, "shared memory of a CTA");
    cudaError_t e = ensure_dynamic_smem((const void*)attention_chunk_paged_kernel<FMT, HD>, smem);
    if (e != cudaSuccess) return e;
    const uint32_t ctas = chunk_ctas();
    e = launch_dependent(attention_chunk_paged_kernel<FMT, HD>, dim3(ctas), dim3(kThreads), smem, stream, p);
    if (e != cudaSuccess) return e;
    return launch_dependent(attention_chunk_paged_join_kernel<FMT, HD>, dim3(ctas, kJoinCtas), dim3(256), 0, stream, p, ctas);
}

}  // namespace

uint64_t attention_chunk_scratch_floats(uint32_t head_dim) {
    return (uint64_t)2 * kMostCtas * kRows * (head_dim + 2) + (uint64_t)kMostCtas * (sizeof(ChunkHead) + sizeof(ChunkSpan)) / 4;
}

int attention_chunk_launches() { return 2; }

cudaError_t attention_chunk(cudaStream_t stream, const KvPool& pool, const KvRows& rows, const float* q, uint64_t q_stride, uint64_t q_head_stride, float* scratch,
                            float* out, uint32_t n_heads, uint32_t fewest) {
    const ChunkParams p{pool, rows, q, out, scratch, q_stride, q_head_stride, n_heads, n_heads / pool.n_kv_heads, fewest};
    const bool half = pool.format == BC_F16;
    switch (pool.head_dim) {
        case 64: return half ? launch_chunk<BC_F16, 64>(stream, p) : launch_chunk<BC_I8, 64>(stream, p);
        case 128: return half ? launch_chunk<BC_F16, 128>(stream, p) : launch_chunk<BC_I8, 128>(stream, p);
        default: return half ? launch_chunk<BC_F16, 256>(stream, p) : launch_chunk<BC_I8, 256>(stream, p);
    }
}

cudaError_t attention_chunk_wait_word(int* word) { return cudaMemcpyToSymbol(g_wait_word, &word, sizeof word); }

}  // namespace k
}  // namespace bc
