// Causal grouped-query attention of the new rows of several sequences over a pool of key/value pages, a query at a time: the form for
// single tokens, whose time is the cache's bytes.
//
// Work. A unit is one row of one KV head: the group of up to 8 query heads that share the head, over the positions that the row sees.
// Units are cut into blocks of 128 positions (256 of heads of 64), and the blocks of all units, in order, into equal runs, one to a CTA: however
// the lengths differ, every CTA reads about the same number of positions, a block or two fewer for each unit that it begins, and lengths stay on
// the device (a captured call serves whatever they become).
// (Twice as many runs, half as long: 5 % slower.) A unit that lies in one CTA's run is written out by it; a unit that is cut leaves
// unnormalised sums with their maximum and sum of exponentials, at most two to a CTA, and a second launch joins them in order.
//
// Arithmetic. Elements are exact in half precision (8-bit ones as whole numbers, their scales multiply scores and probabilities in f32).
// A query element, and a probability times the value's scale, is split into two halves, value = hi + lo (about 22 bits), every product is half x
// half summed in f32. So results are those of f32 arithmetic up to the order of the sums. Halves below 2^-14 lose bits, so what is split is brought
// to the upper end of their range by a power of two first: a query row's largest element to 2^14, the largest probability to 2^15, the largest weight of
// 8-bit values to 2^11 or more (`unit` follows it). What is 2^25 times smaller than these still keeps 22 bits or is lost beside them.
//
// A warp takes 16 positions at a time (32 of heads of 64). Their bytes come by cp.async into a ring of the warp's own, rows as far apart as keeps the fragments'
// loads off one another's banks, and go from there into the fragments of mma.m16n8k16 without another arrangement: elements' order within a product is
// free, and a page's rows hold what a lane needs in 8 or 16 neighbouring bytes. Scores: the 16 rows of A are the group's 8 query heads' hi parts,
// then their lo parts, so one multiply gives both sums and a thread adds its two. Values are the A operand (elements x positions), for which
// pairs of positions are woven together by byte permutes; B is the probabilities as the scores left them, hi and lo: up to four query heads share the 8
// columns (hi in the first four, lo in the others, from rows of queries given twice), more take two multiplies. The tensor cores cut sums
// off: what they add up is one step, and steps are added in f32, rounding.
//
// Measured: a token each of 64 sequences, 32 heads over 8 of 128, contexts of 500 to 8200: 8-bit pages, 589 MB, 112 to 120 us by the
// device (5.2 to 4.9 TB/s; 4 more where units do not count two blocks beside their own, kUnitCost), halves, 1.14 GB, 190 to 199 us (6.0 to 5.8 TB/s). One sequence of 131 072 8-bit positions, 4 KV heads of 256: 273 MB in
// 51 to 53 us (5.4 to 5.1 TB/s). Of the 112 us about ten are the launch's beginning and the join; CTAs of equal runs end 86 to 108 us after it. One sequence of 301
// positions: 6 us, all of it latency.

#include "async_utils.cuh"
#include "kv_pool.cuh"

#include "../../include/bobcat_cuda.h"

namespace bc {
namespace k {

namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr uint32_t kHalf = 16;                 // positions in a fragment, always of one page
constexpr float kLift = 15.f;                  // probabilities are taken times 2^15
constexpr uint32_t kRows = 8;                  // query heads of a KV head, at most
constexpr uint32_t kMostCtas = kPagedMostCtas;

struct TokenParams {
    KvPool pool;
    KvRows rows;
    const float* q;
    float* out;
    float* parts;  // [2 * CTA + which][kRows][HD] sums, then [2 * CTA + which][kRows] (maximum, sum), then a PartsHead per CTA
    uint64_t q_stride, q_head_stride;
    uint32_t n_heads, group;
    uint32_t most;  // sequences of more rows are the other kernel's (kernels_attention_chunk.cu)
    bool whole;     // units are not cut: each counts as one block, and there is nothing to join
};
// What the joining launch needs of the unit that begins in a CTA's run and goes on behind it; `last` is the CTA it ends in, 0 when there is none.
struct PartsHead {
    uint32_t row, head, last, unused;
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same from zero.
__device__ __forceinline__ void mma_f16_new(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// Whole numbers: 32 signed bytes a row times 32 unsigned ones a column; from `upper` in rows 0 to 7, `lower` in the others.
__device__ __forceinline__ void mma_i8_new(uint32_t (&c)[4], const uint4& a, uint32_t b0, uint32_t b1, uint32_t upper, uint32_t lower) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%11,%11};"
                 : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
                 : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "r"(upper), "r"(lower));
}
__device__ __forceinline__ void mma_i8(uint32_t (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

// A warp's ring: steps under way, and where a step's keys, values and scales lie in it. Two rows of keys that a load's phase covers fall 64
// bytes apart, four of values (every other one) 32.
template <int FMT, int HD>
struct Ring {
    // Positions of a step: two fragments where registers and shared memory hold them, which halves what a step costs beside its multiplies. A block, the
    // unit that work is counted in, is a step of each warp.
    static constexpr uint32_t kStep = HD == 64 ? 2 * kHalf : kHalf, kBlock = kStep * kWarps, kHalves = kStep / kHalf;
    static constexpr uint32_t kRowBytes = FMT == BC_F16 ? 2 * HD : HD;
    static constexpr uint32_t kKeyPitch = kRowBytes == 64 ? 64 : kRowBytes + 64, kValuePitch = kRowBytes + 16;
    static constexpr uint32_t kValues = kStep * kKeyPitch, kScales = kValues + kStep * kValuePitch, kBytes = kScales + (FMT == BC_I8 ? 8 * kStep : 0);
    static constexpr uint32_t kSteps = kBytes <= 5632 ? 2 : 1;
    // Blocks that a unit counts beside its own, ahead of them: its beginning and end take as long as these.
    static constexpr uint32_t kUnitCost = FMT == BC_F16 ? 1 : 2;
};
// A sequence of the call: its rows, the positions it holds, the blocks its longest row takes.
struct Seq {
    uint32_t row0, n, end, len;
    uint32_t blocks, counted;  // of its longest row; of them, what a unit counts as
};
__device__ __forceinline__ Seq seq_at(const KvPool& pool, const KvRows& rows, uint32_t s, uint32_t most, uint32_t block, uint32_t unit_cost, bool whole) {
    Seq q;
    q.row0 = rows.starts[s];
    q.end = rows.starts[s + 1];
    q.n = q.row0 < rows.n_rows && q.end > q.row0 && q.end - q.row0 <= most ? min(q.end, rows.n_rows) - q.row0 : 0;
    q.len = rows.lens[s];
    const uint32_t held = min((uint64_t)q.len, (uint64_t)rows.max_pages << pool.page_shift);
    q.blocks = max(1u, (held + block - 1) / block);
    q.counted = whole ? 1 : q.blocks + unit_cost;
    return q;
}
__device__ __forceinline__ uint64_t blocks_of(const KvPool& pool, const Seq& q) { return (uint64_t)q.n * pool.n_kv_heads * q.counted; }

__device__ __forceinline__ uint64_t warp_sum_u64(uint64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Rows of sums that a warp leaves at a unit's end.
template <bool PACKED>
constexpr uint32_t sum_rows() { return PACKED ? kRows / 2 : kRows; }
template <int FMT, int HD>
constexpr size_t rings_bytes() { return (size_t)kWarps * Ring<FMT, HD>::kSteps * Ring<FMT, HD>::kBytes; }
template <int HD, bool PACKED>
constexpr size_t sums_bytes() { return (size_t)kWarps * sum_rows<PACKED>() * (HD + 4) * 4; }
// CTAs that an SM holds, by their registers: heads of 256 take more than half (131072 positions of four 8-bit heads 60 us, 86 with two CTAs and spills).
constexpr uint32_t ctas_per_sm(uint32_t head_dim) { return head_dim == 256 ? 1 : 2; }

// Whether the sums have room beside the rings: the next unit's copies are then under way while a unit ends.
template <int FMT, int HD, bool PACKED>
constexpr bool sums_beside() { return (size_t)HD * 32 + rings_bytes<FMT, HD>() + sums_bytes<HD, PACKED>() <= 228 * 1024 / ctas_per_sm(HD) - 4096; }
template <int FMT, int HD, bool PACKED>
constexpr size_t token_smem_bytes() {
    constexpr size_t rings = rings_bytes<FMT, HD>(), sums = sums_bytes<HD, PACKED>();
    return (size_t)HD * 32 + (sums_beside<FMT, HD, PACKED>() ? rings + sums : rings > sums ? rings : sums);
}

// Registers of a warp's step of keys, and of values: 32-bit words per lane.
template <int FMT, int HD>
constexpr int step_words() { return FMT == BC_F16 ? HD / 4 : HD / 8; }

// PACKED: up to four query heads a KV head.
template <int FMT, int HD, bool PACKED>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(HD)) attention_token_paged_kernel(const __grid_constant__ TokenParams p) {
    using R = Ring<FMT, HD>;
    constexpr int kWords = step_words<FMT, HD>(), D = R::kSteps;
    constexpr uint32_t kSumPitch = HD + 4, kStep = R::kStep, kBlock = R::kBlock, kHalves = R::kHalves;
    constexpr int kKSteps = HD / 16, kTiles = HD / 16;
    extern __shared__ __align__(16) uint8_t token_smem[];
    uint4* q_frag = reinterpret_cast<uint4*>(token_smem);                                    // [kKSteps][32]
    uint8_t* rings = token_smem + kKSteps * 32 * 16;                                         // [kWarps][D] steps
    constexpr bool kBeside = sums_beside<FMT, HD, PACKED>();
    constexpr uint32_t kSumRows = sum_rows<PACKED>();
    float* sums = reinterpret_cast<float*>(rings + (kBeside ? rings_bytes<FMT, HD>() : 0));  // [kWarps][kSumRows][kSumPitch], or in the rings' place
    __shared__ float2 stats[kWarps * kRows];
    __shared__ float q_factor[kRows];
    __shared__ uint32_t page_ids[kWarps][64];
    __shared__ int digit_sums[kRows][4];
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const KvPool& pool = p.pool;
    const KvRows& rows = p.rows;
    const float scale = 1.4426950408889634f / sqrtf((float)HD);  // scores in powers of two

    // This CTA's run of blocks, and the sequence that it begins in. Every warp works it out for itself.
    uint64_t total = 0;
    for (uint32_t s = lane; s < rows.n_seqs; s += 32) total += blocks_of(pool, seq_at(pool, rows, s, p.most, kBlock, R::kUnitCost, p.whole));
    total = warp_sum_u64(total);
    const uint64_t runs = min((uint64_t)gridDim.x, total);  // none of them empty
    uint64_t at = blockIdx.x < runs ? total * blockIdx.x / runs : total;
    const uint64_t end = blockIdx.x < runs ? total * (blockIdx.x + 1) / runs : total;
    PartsHead* const heads = reinterpret_cast<PartsHead*>(p.parts + (uint64_t)2 * kMostCtas * kRows * (HD + 2));
    if (at >= end) {
        if (tid == 0) heads[blockIdx.x] = PartsHead{0, 0, 0, 0};
        return;
    }
    uint32_t seq = 0;
    uint64_t base = 0;  // blocks of the sequences before `seq`
    for (uint32_t s0 = 0; s0 < rows.n_seqs; s0 += 32) {
        const uint64_t mine = s0 + lane < rows.n_seqs ? blocks_of(pool, seq_at(pool, rows, s0 + lane, p.most, kBlock, R::kUnitCost, p.whole)) : 0;
        uint64_t upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t other = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= (uint32_t)o) upto += other;
        }
        const uint32_t beyond = __ballot_sync(0xffffffffu, base + upto > at);
        if (beyond) {
            const int who = __ffs(beyond) - 1;
            seq = s0 + who;
            base += __shfl_sync(0xffffffffu, upto - mine, who);
            break;
        }
        base += __shfl_sync(0xffffffffu, upto, 31);
    }
    PartsHead cut{0, 0, 0, 0};

    // The unit at `at`, and the blocks of it that are this CTA's: none where the run ends ahead of them. Rows of a head are neighbours.
    struct Work {
        uint32_t seq, row, head, n_keys, block0, blocks, counted, all_blocks;
        uint64_t last;  // the unit's last place in the call's work
    };
    auto find = [&]() {
        Work w;
        Seq sq = seq_at(pool, rows, seq, p.most, kBlock, R::kUnitCost, p.whole);
        while (base + blocks_of(pool, sq) <= at) {  // sequences without rows have no blocks
            base += blocks_of(pool, sq);
            if (seq + 1 == rows.n_seqs) return Work{};
            sq = seq_at(pool, rows, ++seq, p.most, kBlock, R::kUnitCost, p.whole);
        }
        const uint64_t in_seq = at - base;
        const uint32_t which = (uint32_t)(in_seq / sq.counted);
        w.seq = seq;
        const uint32_t from = (uint32_t)(in_seq % sq.counted), cost = p.whole ? 0 : R::kUnitCost;
        w.counted = (uint32_t)min((uint64_t)(sq.counted - from), end - at);
        w.block0 = max(from, cost) - cost;
        w.blocks = p.whole ? sq.blocks : max(from + w.counted, cost) - cost - w.block0;
        w.last = at - from + sq.counted - 1;
        w.all_blocks = sq.blocks;
        w.head = which / sq.n;
        w.row = sq.row0 + which % sq.n;
        const uint32_t back = sq.end - w.row;  // the row's distance from the end: it sees positions 0 .. len - back
        const uint32_t held = min((uint64_t)sq.len, (uint64_t)rows.max_pages << pool.page_shift);
        w.n_keys = back <= sq.len ? min(sq.len - back + 1, held) : 0;
        if (held < sq.len) leave_fault(pool, kFaultTable);
        return w;
    };

    // What the copies go by: the warp's steps of a unit are one block apart, step n has positions pos0 + n * kBlock on.
    const uint32_t slots = (1u << pool.page_shift) - 1;
    uint8_t* const ring = rings + warp * (D * R::kBytes);
    constexpr uint32_t kPieces = R::kRowBytes / 16;  // of a row; a lane brings every 32nd of the step's
    const uint32_t ring_at = async::smem_u32(ring), key_to = ring_at + lane / kPieces * R::kKeyPitch + lane % kPieces * 16,
                   value_to = ring_at + R::kValues + lane / kPieces * R::kValuePitch + lane % kPieces * 16;
    const uint8_t* const scale_pool = lane < 4 ? pool.k : pool.v;
    const uint32_t* table = nullptr;
    uint32_t pos0 = 0, pos_end = 0, n_steps = 0;
    uint64_t head_at = 0, scales_at = 0;
    auto aim = [&](const Work& w) {
        table = rows.table + (uint64_t)w.seq * rows.max_pages;
        pos0 = w.block0 * kBlock + warp * kStep;
        pos_end = min((w.block0 + w.blocks) * kBlock, w.n_keys);
        n_steps = pos0 < pos_end ? (pos_end - pos0 + kBlock - 1) / kBlock : 0;
        head_at = (uint64_t)(w.head << pool.page_shift) * pool.row_bytes + 16 * lane;
        scales_at = (uint64_t)(pool.n_kv_heads << pool.page_shift) * pool.row_bytes + (uint64_t)(w.head << pool.page_shift) * 4 + 16 * (lane & 3);
    };
    // The pages of a step's halves, 32 halves looked up at a time, by the copies of the first of them, before anything asks. A half behind the
    // last position has none.
    constexpr uint32_t kAtOnce = 32 / kHalves;  // steps
    auto look_up = [&](uint32_t n) {
        if (n % kAtOnce == 0 && n < n_steps) {
            const uint32_t at = pos0 + (n + lane / kHalves) * kBlock + lane % kHalves * kHalf;
            page_ids[warp][(n * kHalves + lane) % 64] = at < pos_end ? table[at >> pool.page_shift] : kNoSlot;
            __syncwarp();
        }
    };
    // Keys (and both scales) of a step, then its values: a group of copies each, empty behind the last step.
    uint64_t rows_at[kHalves] = {};
    bool there[kHalves] = {};
    auto copy_keys = [&](uint32_t n) {
        look_up(n);
        const uint32_t in_ring = n % D * R::kBytes;
#pragma unroll
        for (uint32_t h = 0; h < kHalves; ++h) {
            const uint32_t page = n < n_steps ? page_ids[warp][(n * kHalves + h) % 64] : kNoSlot, slot = (pos0 + n * kBlock + h * kHalf) & slots;
            there[h] = page < pool.n_pages;
            if (there[h]) {
                const uint64_t page_at = page * pool.page_bytes;
                rows_at[h] = page_at + head_at + slot * pool.row_bytes;
                const uint8_t* from = pool.k + rows_at[h];
#pragma unroll
                for (uint32_t i = 0; i < kPieces / 2; ++i) async::cp_async_16(key_to + in_ring + (h * kHalf + i * (32 / kPieces)) * R::kKeyPitch, from + 512 * i);
                if (FMT == BC_I8 && lane < 8)
                    async::cp_async_16(ring_at + in_ring + R::kScales + h * 4 * kHalf + (lane >> 2) * 4 * kStep + 16 * (lane & 3), scale_pool + page_at + scales_at + slot * 4);
            }
        }
        async::cp_async_commit();
    };
    auto copy_values = [&](uint32_t n) {  // behind the same step's copy_keys
#pragma unroll
        for (uint32_t h = 0; h < kHalves; ++h)
            if (there[h]) {
                const uint8_t* from = pool.v + rows_at[h];
#pragma unroll
                for (uint32_t i = 0; i < kPieces / 2; ++i)
                    async::cp_async_16(value_to + n % D * R::kBytes + (h * kHalf + i * (32 / kPieces)) * R::kValuePitch, from + 512 * i);
            }
        async::cp_async_commit();
    };
    auto begin_copies = [&](const Work& w) {
        aim(w);
#pragma unroll
        for (uint32_t n = 0; n < D; ++n) {
            copy_keys(n);
            copy_values(n);
        }
    };
    // A warp's query head of a unit (PACKED: two warps a head), two elements of every 64 to a lane.
    const uint32_t q_head = PACKED ? warp & 3 : warp;
    float2 x[HD / 64];
    auto load_query = [&](const Work& w) {
#pragma unroll
        for (int i = 0; i < HD / 64; ++i)
            x[i] = q_head < p.group ? *reinterpret_cast<const float2*>(p.q + w.row * p.q_stride + (w.head * p.group + q_head) * p.q_head_stride + 64 * i + 2 * lane)
                                    : make_float2(0.f, 0.f);
    };
    Work w = find();
    if (w.blocks == 0) {
        if (tid == 0) heads[blockIdx.x] = cut;
        return;
    }
    begin_copies(w);
    load_query(w);
    while (true) {
        // Query fragments in the order of a lane's key elements, a warp per query head (PACKED: two). A pair of elements is a word of hi and one of
        // lo parts.
        __syncthreads();  // the previous unit's fragments and sums have been read
        {
            uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < HD / 64; ++i) most = max(most, max(__float_as_uint(x[i].x) & 0x7fffffffu, __float_as_uint(x[i].y) & 0x7fffffffu));
            most = __reduce_max_sync(0xffffffffu, most);
            const uint32_t exponent = min(max(most >> 23, 1u), 253u);
            const float up = __uint_as_float((254u - exponent) << 23);  // times 2^14 or 2^29 below: together they may pass the largest float
            const float back = FMT == BC_F16 ? 1.f / 16384.f : 1.f / 536870912.f;
            if (lane == 0) q_factor[warp] = most < 0x7f800000u ? __uint_as_float(exponent << 23) * (scale * back) : __uint_as_float(0x7fc00000u);
            int sum[4] = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < HD / 64; ++i) {
                const uint32_t e = 2 * lane;  // element 64 i + e
                if constexpr (FMT == BC_F16) {
                    uint32_t hi, lo;
                    split_half2(x[i].x * up * 16384.f, x[i].y * up * 16384.f, hi, lo);
                    uint32_t* to = reinterpret_cast<uint32_t*>(q_frag + (4 * i + 2 * (e >> 5) + ((e & 7) >> 2)) * 32 + 4 * warp + ((e & 31) >> 3)) + (e & 3);  // e & 3 is 0 or 2
                    to[0] = hi;
                    to[1] = lo;
                } else {
                    // Signed digits of base 256, of whole numbers up to 2^30; most significant first.
                    int v[2] = {__float2int_rn(x[i].x * up * 536870912.f), __float2int_rn(x[i].y * up * 536870912.f)};
                    uint32_t digits[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int d = 3; d >= 0; --d)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const int digit = (int)((uint32_t)v[k] << 24) >> 24;
                            v[k] = (v[k] - digit) >> 8;
                            digits[d] |= (uint32_t)(digit & 0xff) << (8 * k);
                            sum[d] += digit;
                        }
                    // Words 0 and 2 of a lane's four are rows 0 to 7 of A, 1 and 3 rows 8 to 15: digits 0 and 1 (of the upper four warps when PACKED: 2 and 3).
                    uint8_t* to = reinterpret_cast<uint8_t*>(q_frag + (2 * i + ((e & 15) >> 3)) * 32 + 4 * warp + (e >> 4)) + ((e & 7) >> 2) * 8 + (e & 3);
                    const bool lower = PACKED && warp >= 4;
                    *reinterpret_cast<uint16_t*>(to) = (uint16_t)(lower ? digits[2] : digits[0]);
                    *reinterpret_cast<uint16_t*>(to + 4) = (uint16_t)(lower ? digits[3] : digits[1]);
                    if (!PACKED) {
                        *reinterpret_cast<uint16_t*>(to + kKSteps / 2 * 32 * 16) = (uint16_t)digits[2];
                        *reinterpret_cast<uint16_t*>(to + kKSteps / 2 * 32 * 16 + 4) = (uint16_t)digits[3];
                    }
                }
            }
            if constexpr (FMT == BC_I8) {
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    sum[d] = __reduce_add_sync(0xffffffffu, sum[d]);
                    if (lane == 0) digit_sums[warp][d] = sum[d];
                }
            }
        }
        __syncthreads();
        const float factor_q = q_factor[g];
        // What sums of digits begin with: a float of 1.5 * 2^23, less 128 times the digits (an element is stored as its number plus 128). They end
        // as floats of 1.5 * 2^23 plus the sum.
        constexpr uint32_t kMagic = 0x4b400000u;
        uint32_t begin_sums[4] = {0, 0, 0, 0};
        if constexpr (FMT == BC_I8) {
#pragma unroll
            for (int d = 0; d < (PACKED ? 2 : 4); ++d) begin_sums[d] = kMagic - 128u * (uint32_t)digit_sums[g][PACKED && g >= 4 ? d + 2 : d];
        }

        float2 o[kTiles][2];
#pragma unroll
        for (int n = 0; n < kTiles; ++n) o[n][0] = o[n][1] = make_float2(0.f, 0.f);
        float top = -INFINITY, total_p = 0.f;  // of query head g, the sum over this lane's positions
        float unit = FMT == BC_I8 ? 0.f : 1.f, inverse_unit = unit;  // the sums of query head g are counted in these

        // What comes next is looked up meanwhile.
        const Work done = w;
        at += done.counted;
        bool more = at < end;  // uniform in the CTA
        if (more) {
            w = find();
            more = w.blocks > 0;
        }
        for (uint32_t n = 0; n < n_steps; ++n) {
            const uint8_t* const here = ring + n % D * R::kBytes;
            // Positions of the step that exist, from its first on; halves whose page the pool does not have hold nothing.
            const uint32_t left = pos_end - (pos0 + n * kBlock);
            uint32_t missing = 0;
#pragma unroll
            for (uint32_t h = 0; h < kHalves; ++h) missing |= page_ids[warp][(n * kHalves + h) % 64] >= pool.n_pages ? 1u << h : 0u;
            async::cp_async_wait<2 * D - 1>();
            __syncwarp();  // everyone's copies of the keys
            // Scores of positions 16h + 2t + (i & 1) + 8 (i >> 1), x[4h + i], for query head g.
            constexpr int kTilesOfKeys = 2 * kHalves, kScores = 4 * kHalves;
            float x[kScores];
            float2 dk[kTilesOfKeys], dv[kTilesOfKeys];
            if constexpr (FMT == BC_F16) {
                float s[kTilesOfKeys][4];
#pragma unroll
                for (int c = 0; c < kWords / 8; ++c) {  // 64 bytes of a key: 32 elements
                    const uint4 f0 = q_frag[2 * c * 32 + lane], f1 = q_frag[(2 * c + 1) * 32 + lane];
                    uint4 kw[kTilesOfKeys];
#pragma unroll
                    for (int j = 0; j < kTilesOfKeys; ++j) kw[j] = *reinterpret_cast<const uint4*>(here + (8 * j + g) * R::kKeyPitch + 64 * c + 16 * t);
#pragma unroll
                    for (int j = 0; j < kTilesOfKeys; ++j) {
                        if (c == 0)
                            mma_f16_new(s[j], f0.x, f0.y, f0.z, f0.w, kw[j].x, kw[j].y);
                        else
                            mma_f16(s[j], f0.x, f0.y, f0.z, f0.w, kw[j].x, kw[j].y);
                    }
#pragma unroll
                    for (int j = 0; j < kTilesOfKeys; ++j) mma_f16(s[j], f1.x, f1.y, f1.z, f1.w, kw[j].z, kw[j].w);
                }
#pragma unroll
                for (int j = 0; j < kTilesOfKeys; ++j) {
                    x[2 * j] = s[j][0] + s[j][2];
                    x[2 * j + 1] = s[j][1] + s[j][3];
                }
            } else {
                constexpr int kSets = PACKED ? 1 : 2;
                uint32_t s[kTilesOfKeys][kSets][4];
#pragma unroll
                for (int c = 0; c < kWords / 8; ++c) {  // 64 bytes of a key: 64 elements
                    uint4 kw[kTilesOfKeys];
#pragma unroll
                    for (int j = 0; j < kTilesOfKeys; ++j) kw[j] = *reinterpret_cast<const uint4*>(here + (8 * j + g) * R::kKeyPitch + 64 * c + 16 * t);
#pragma unroll
                    for (int m = 0; m < kSets; ++m) {
                        const uint4 f0 = q_frag[(m * (kKSteps / 2) + 2 * c) * 32 + lane], f1 = q_frag[(m * (kKSteps / 2) + 2 * c + 1) * 32 + lane];
#pragma unroll
                        for (int j = 0; j < kTilesOfKeys; ++j) {
                            if (c == 0)
                                mma_i8_new(s[j][m], f0, kw[j].x, kw[j].y, begin_sums[2 * m], begin_sums[2 * m + 1]);
                            else
                                mma_i8(s[j][m], f0, kw[j].x, kw[j].y);
                        }
#pragma unroll
                        for (int j = 0; j < kTilesOfKeys; ++j) mma_i8(s[j][m], f1, kw[j].z, kw[j].w);
                    }
                }
                // The digits' sums together: two here, the other two in the lane of the row four on, or here too.
#pragma unroll
                for (int i = 0; i < kScores; ++i) {
                    const int j = i >> 1, k = i & 1;
                    x[i] = fmaf(__uint_as_float(s[j][0][k]) - 12582912.f, 256.f, __uint_as_float(s[j][0][k + 2]) - 12582912.f);
                    if constexpr (PACKED) {
                        x[i] *= g < 4 ? 65536.f : 1.f;
                        x[i] += __shfl_xor_sync(0xffffffffu, x[i], 16);
                    } else {
                        x[i] = fmaf(x[i], 65536.f, fmaf(__uint_as_float(s[j][1][k]) - 12582912.f, 256.f, __uint_as_float(s[j][1][k + 2]) - 12582912.f));
                    }
                }
                const float* scales = reinterpret_cast<const float*>(here + R::kScales);
#pragma unroll
                for (int j = 0; j < kTilesOfKeys; ++j) {
                    dk[j] = *reinterpret_cast<const float2*>(scales + 8 * j + 2 * t);
                    dv[j] = *reinterpret_cast<const float2*>(scales + kStep + 8 * j + 2 * t);
                }
            }
            __syncwarp();  // the keys have been read
            copy_keys(n + D);
#pragma unroll
            for (int i = 0; i < kScores; ++i) {
                x[i] *= factor_q;
                if (FMT == BC_I8) x[i] *= i & 1 ? dk[i >> 1].y : dk[i >> 1].x;
            }
            const bool some_unseen = left < kStep || missing;  // uniform
            auto seen = [&](int i) { return 16 * (i >> 2) + 2 * t + (i & 1) + 8 * (i >> 1 & 1) < left && !(missing >> (i >> 2) & 1); };
            if (some_unseen) {
#pragma unroll
                for (int i = 0; i < kScores; ++i)
                    if (!seen(i)) x[i] = -INFINITY;
                if (missing & ((left + kHalf - 1) / kHalf >= 2 ? 3u : 1u) && lane == 0) leave_fault(pool, kFaultPage);
            }
            float most = x[0];
#pragma unroll
            for (int i = 1; i < kScores; ++i) most = fmaxf(most, x[i]);
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const float now = fmaxf(top, most);
            const float shift = now == -INFINITY ? 0.f : now, down = shift - kLift;
            float factor = exp2_fast(top - shift);
            const bool moved = now > top;
            top = now;
            float total_step = 0.f;
#pragma unroll
            for (int i = 0; i < kScores; ++i) {
                x[i] = exp2_fast(x[i] - down);  // the sums are lifted alike
                total_step += x[i];
            }
            if constexpr (FMT == BC_F16) {
                // No number, for the first time: of an infinite key, perhaps one whose score is minus infinity, which weighs nothing.
                const uint32_t q_head = PACKED ? g & 3 : g;
                if (__builtin_expect(__any_sync(0xffffffffu, total_step != total_step && total_p == total_p && q_head < p.group), 0)) {
                    total_step = 0.f;
#pragma unroll
                    for (int i = 0; i < kScores; ++i) {
                        const uint32_t in_step = 16 * (i >> 2) + 2 * t + (i & 1) + 8 * (i >> 1 & 1), page = page_ids[warp][(n * kHalves + (i >> 2)) % 64];
                        if (x[i] != x[i] && q_head < p.group && page < pool.n_pages &&
                            score_is_minus_infinity(p.q + done.row * p.q_stride + (done.head * p.group + q_head) * p.q_head_stride,
                                                    pool.k + kv_row_at(pool, page, done.head, (pos0 + n * kBlock + in_step) & slots), HD))
                            x[i] = 0.f;
                        total_step += x[i];
                    }
                    __syncwarp();
                }
            }
            total_p = total_p * factor + total_step;
            if constexpr (FMT == BC_I8) {
#pragma unroll
                for (int i = 0; i < kScores; ++i) x[i] *= i & 1 ? dv[i >> 1].y : dv[i >> 1].x;
                if (some_unseen) {  // scales behind the last position may be anything
#pragma unroll
                    for (int i = 0; i < kScores; ++i)
                        if (!seen(i)) x[i] = 0.f;
                }
                float largest = fabsf(x[0]);
#pragma unroll
                for (int i = 1; i < kScores; ++i) largest = fmaxf(largest, fabsf(x[i]));
                largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
                largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
                if (moved || largest > 32768.f * unit) {  // weights of 2^15 units at most: halves end at 2^16
                    // A row's largest weight so far, what went before scaled to the new maximum, is 2^11 to 2^12 units.
                    const uint32_t exponent = __float_as_uint(fmaxf(2048.f * unit * factor, largest)) >> 23;
                    const bool any = exponent > 11;  // smaller ones weigh nothing
                    const float before = unit;
                    unit = any ? __uint_as_float((min(exponent, 253u) - 11u) << 23) : 0.f;
                    inverse_unit = any ? __uint_as_float((265u - min(exponent, 253u)) << 23) : 0.f;
                    factor *= before * inverse_unit;
                }
#pragma unroll
                for (int i = 0; i < kScores; ++i) x[i] *= inverse_unit;
            }
            const float2 f = make_float2(__shfl_sync(0xffffffffu, factor, 8 * t), __shfl_sync(0xffffffffu, factor, 8 * t + 4));  // of columns 2t and 2t + 1
            uint32_t hi[2 * kHalves], lo[2 * kHalves];
#pragma unroll
            for (int j = 0; j < kTilesOfKeys; ++j) {
                split_half2(x[2 * j], x[2 * j + 1], hi[j], lo[j]);
                if (PACKED && g >= 4) hi[j] = lo[j];
            }
            async::cp_async_wait<2 * D - 1>();
            __syncwarp();  // everyone's copies of the values
            // A step's sums, from zero, join the others rounded: of 16 elements, by the fragments of both halves.
            auto product = [&](int tile, const uint32_t (&a)[kHalves][4]) {
                float d[4];
                if (PACKED) {
                    mma_f16_new(d, a[0][0], a[0][1], a[0][2], a[0][3], hi[0], hi[1]);
                    if (kHalves == 2) mma_f16(d, a[kHalves - 1][0], a[kHalves - 1][1], a[kHalves - 1][2], a[kHalves - 1][3], hi[2 * kHalves - 2], hi[2 * kHalves - 1]);
                } else {
                    mma_f16_new(d, a[0][0], a[0][1], a[0][2], a[0][3], lo[0], lo[1]);
                    if (kHalves == 2) mma_f16(d, a[kHalves - 1][0], a[kHalves - 1][1], a[kHalves - 1][2], a[kHalves - 1][3], lo[2 * kHalves - 2], lo[2 * kHalves - 1]);
                    mma_f16(d, a[0][0], a[0][1], a[0][2], a[0][3], hi[0], hi[1]);
                    if (kHalves == 2) mma_f16(d, a[kHalves - 1][0], a[kHalves - 1][1], a[kHalves - 1][2], a[kHalves - 1][3], hi[2 * kHalves - 2], hi[2 * kHalves - 1]);
                }
                o[tile][0] = fma2(o[tile][0], f, make_float2(d[0], d[1]));
                o[tile][1] = fma2(o[tile][1], f, make_float2(d[2], d[3]));
            };
            // Position 16h + 2t + (i & 1) + 8 (i >> 1) of the step, i = 0 .. 3; a lane's 8 elements 8g .. of every 64.
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) {
                constexpr int kOfRow = FMT == BC_F16 ? 4 : 2;  // words
                uint32_t vw[kHalves][4][kOfRow];
#pragma unroll
                for (int h = 0; h < (int)kHalves; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint8_t* from = here + R::kValues + (16 * h + 2 * t + (i & 1) + 8 * (i >> 1)) * R::kValuePitch;
                        if constexpr (FMT == BC_F16) {
                            const uint4 w = *reinterpret_cast<const uint4*>(from + 128 * c + 16 * g);
                            vw[h][i][0] = w.x, vw[h][i][1] = w.y, vw[h][i][kOfRow - 2] = w.z, vw[h][i][kOfRow - 1] = w.w;
                            if (some_unseen) {  // elements behind the last position may be anything
#pragma unroll
                                for (int k = 0; k < kOfRow; ++k)
                                    if (!seen(4 * h + i)) vw[h][i][k] = 0;
                            }
                        } else {
                            const uint2 w = *reinterpret_cast<const uint2*>(from + 64 * c + 8 * g);
                            vw[h][i][0] = w.x, vw[h][i][1] = w.y;
                        }
                    }
                if (c == HD / 64 - 1) {
                    __syncwarp();  // the values have been read
                    copy_values(n + D);
                }
                if constexpr (FMT == BC_F16) {
#pragma unroll
                    for (int w = 0; w < 4; ++w) {  // elements 2w, 2w + 1 of the lane's: rows g and g + 8 of a tile
                        uint32_t a[kHalves][4];
#pragma unroll
                        for (int h = 0; h < (int)kHalves; ++h) {
                            a[h][0] = __byte_perm(vw[h][0][w], vw[h][1][w], 0x5410);
                            a[h][1] = __byte_perm(vw[h][0][w], vw[h][1][w], 0x7632);
                            a[h][2] = __byte_perm(vw[h][2][w], vw[h][3][w], 0x5410);
                            a[h][3] = __byte_perm(vw[h][2][w], vw[h][3][w], 0x7632);
                        }
                        product(4 * c + w, a);
                    }
                } else {
#pragma unroll
                    for (int w = 0; w < 2; ++w)  // elements 4w .. 4w + 3 of the lane's: two tiles
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            uint32_t a[kHalves][4];  // elements 2e and 2e + 1 of two positions
#pragma unroll
                            for (int h = 0; h < (int)kHalves; ++h) {
                                unpack_i8(__byte_perm(vw[h][0][w], vw[h][1][w], e ? 0x7362 : 0x5140), a[h][0], a[h][1]);
                                unpack_i8(__byte_perm(vw[h][2][w], vw[h][3][w], e ? 0x7362 : 0x5140), a[h][2], a[h][3]);
                            }
                            product(4 * c + 2 * w + e, a);
                        }
                }
            }
        }
        async::cp_async_wait<0>();
        if (kBeside && more) begin_copies(w);
        if (more) load_query(w);

        // The warps' sums, joined through shared memory. Tile n's rows g and g + 8 are elements 2n' and 2n' + 1 of the lane's eight.
        total_p += __shfl_xor_sync(0xffffffffu, total_p, 1);
        total_p += __shfl_xor_sync(0xffffffffu, total_p, 2);
        if (t == 0) stats[warp * kRows + g] = make_float2(top, total_p);
        const float u0 = __shfl_sync(0xffffffffu, unit, 8 * t), u1 = __shfl_sync(0xffffffffu, unit, 8 * t + 4);
        if (!kBeside) __syncthreads();  // every ring has been read
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
            const uint32_t d = (n / 4) * 64 + 8 * g + 2 * (n % 4);  // elements d and d + 1
            float2 even = make_float2(o[n][0].x * u0, o[n][1].x * u0), odd = make_float2(o[n][0].y * u1, o[n][1].y * u1);
            if (PACKED) {  // the lower halves' sums, two lanes on
                even.x += __shfl_xor_sync(0xffffffffu, even.x, 2);
                even.y += __shfl_xor_sync(0xffffffffu, even.y, 2);
                odd.x += __shfl_xor_sync(0xffffffffu, odd.x, 2);
                odd.y += __shfl_xor_sync(0xffffffffu, odd.y, 2);
            }
            if (!PACKED || t < 2) {
                float* to = sums + (warp * kSumRows + 2 * t) * kSumPitch + d;
                *reinterpret_cast<float2*>(to) = even;
                *reinterpret_cast<float2*>(to + kSumPitch) = odd;
            }
        }
        __syncthreads();
        const bool begins = done.block0 == 0, ends = done.block0 + done.blocks == done.all_blocks;
        const uint32_t slot = 2 * blockIdx.x + (begins ? 1 : 0);
        for (uint32_t quad = tid; quad < p.group * (HD / 4); quad += kThreads) {
            const uint32_t r = quad / (HD / 4), d = quad % (HD / 4) * 4;
            float most = -INFINITY;
#pragma unroll
            for (int i = 0; i < kWarps; ++i) most = fmaxf(most, stats[i * kRows + r].x);
            const float shift = most == -INFINITY ? 0.f : most;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
            float sum_p = 0.f;
#pragma unroll
            for (int i = 0; i < kWarps; ++i) {
                const float2 st = stats[i * kRows + r];
                const float weight = st.x == -INFINITY ? 0.f : exp2f(st.x - shift);
                const float4 v = *reinterpret_cast<const float4*>(sums + (i * kSumRows + r) * kSumPitch + d);
                if (st.x != -INFINITY) {
                    sum.x += weight * v.x;
                    sum.y += weight * v.y;
                    sum.z += weight * v.z;
                    sum.w += weight * v.w;
                }
                sum_p += weight * st.y;
            }
            if (begins && ends) {
                // A row that sees nothing is zeros.
                const float inverse = most == -INFINITY && sum_p == 0.f ? 0.f : 1.f / sum_p;
                *reinterpret_cast<float4*>(p.out + (uint64_t)done.row * p.n_heads * HD + (done.head * p.group + r) * HD + d) =
                    make_float4(sum.x * inverse, sum.y * inverse, sum.z * inverse, sum.w * inverse);
            } else {
                *reinterpret_cast<float4*>(p.parts + ((uint64_t)slot * kRows + r) * HD + d) = sum;
                if (d == 0) *reinterpret_cast<float2*>(p.parts + (uint64_t)2 * kMostCtas * kRows * HD + (slot * kRows + r) * 2) = make_float2(most, sum_p);
            }
        }
        if (begins && !ends) {
            // The CTA whose run holds the unit's last block: run c is [total c / runs, total (c + 1) / runs).
            uint32_t last = (uint32_t)(done.last * runs / total);
            while (total * (last + 1) / runs <= done.last) ++last;
            while (total * last / runs > done.last) --last;
            cut = PartsHead{done.row, done.head, last, 0};
        }
        if (!more) break;
        if (!kBeside) {
            __syncthreads();  // the sums have been read
            begin_copies(w);
        }
    }
    if (tid == 0) heads[blockIdx.x] = cut;
}

// Joins the parts of a unit that begins in CTA c's run and ends in a later one's: a CTA per query head, whose warps take parts in turn, so that a
// unit over many CTAs is joined in a few trips to memory.
template <int HD>
__global__ void __launch_bounds__(256) attention_token_paged_join_kernel(const float* __restrict__ parts, float* __restrict__ out, uint32_t n_heads, uint32_t group) {
    constexpr int kPairs = HD / 64, kAtOnce = 4;
    __shared__ float2 warp_stats[8];
    __shared__ float warp_sums[8][HD];
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = blockIdx.y, c = blockIdx.x;
    const PartsHead cut = reinterpret_cast<const PartsHead*>(parts + (uint64_t)2 * kMostCtas * kRows * (HD + 2))[c];
    if (cut.last == 0) return;
    const float2* stats = reinterpret_cast<const float2*>(parts + (uint64_t)2 * kMostCtas * kRows * HD);
    const uint32_t n = cut.last - c + 1;
    float top = -INFINITY, total = 0.f;
    float2 sum[kPairs];
#pragma unroll
    for (int i = 0; i < kPairs; ++i) sum[i] = make_float2(0.f, 0.f);
    for (uint32_t first = warp; first < n; first += 8 * kAtOnce) {
        float2 st[kAtOnce], v[kAtOnce][kPairs];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            const uint32_t i = first + 8 * k, at = (2 * (c + i) + (i == 0 ? 1 : 0)) * kRows + r;
            st[k] = i < n ? stats[at] : make_float2(-INFINITY, 0.f);
            const float2* from = reinterpret_cast<const float2*>(parts + (uint64_t)at * HD) + lane;
#pragma unroll
            for (int j = 0; j < kPairs; ++j) v[k][j] = i < n ? from[32 * j] : make_float2(0.f, 0.f);
        }
        float now = top;
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) now = fmaxf(now, st[k].x);
        const float shift = now == -INFINITY ? 0.f : now, fall = exp2f(top - shift);
        top = now;
        total *= fall;
#pragma unroll
        for (int j = 0; j < kPairs; ++j) sum[j] = make_float2(sum[j].x * fall, sum[j].y * fall);
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            const float weight = st[k].x == -INFINITY ? 0.f : exp2f(st[k].x - shift);
            total += weight * st[k].y;
            if (st[k].x != -INFINITY) {
#pragma unroll
                for (int j = 0; j < kPairs; ++j) {
                    sum[j].x += weight * v[k][j].x;
                    sum[j].y += weight * v[k][j].y;
                }
            }
        }
    }
    if (lane == 0) warp_stats[warp] = make_float2(top, total);
#pragma unroll
    for (int j = 0; j < kPairs; ++j) *reinterpret_cast<float2*>(&warp_sums[warp][64 * j + 2 * lane]) = sum[j];
    __syncthreads();
    for (uint32_t d = tid; d < HD; d += 256) {
        float most = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) most = fmaxf(most, warp_stats[i].x);
        const float shift = most == -INFINITY ? 0.f : most;
        float all = 0.f, x = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 st = warp_stats[i];
            const float weight = st.x == -INFINITY ? 0.f : exp2f(st.x - shift);
            all += weight * st.y;
            if (st.x != -INFINITY) x += weight * warp_sums[i][d];
        }
        out[(uint64_t)cut.row * n_heads * HD + (cut.head * group + r) * HD + d] = most == -INFINITY && all == 0.f ? 0.f : x / all;
    }
}

uint32_t block_of(const KvPool& pool) {
    const bool half = pool.format == BC_F16;
    switch (pool.head_dim) {
        case 64: return half ? Ring<BC_F16, 64>::kBlock : Ring<BC_I8, 64>::kBlock;
        case 128: return half ? Ring<BC_F16, 128>::kBlock : Ring<BC_I8, 128>::kBlock;
        default: return half ? Ring<BC_F16, 256>::kBlock : Ring<BC_I8, 256>::kBlock;
    }
}

// CTAs of a launch: no more than the blocks that the tables could hold.
uint32_t token_ctas(const KvPool& pool, const KvRows& rows) {
    const uint32_t block = block_of(pool);
    const uint64_t most = (uint64_t)rows.n_rows * pool.n_kv_heads * ((((uint64_t)rows.max_pages << pool.page_shift) + block - 1) / block);
    uint64_t ctas = (uint64_t)sm_count() * ctas_per_sm(pool.head_dim);
    if (ctas > kMostCtas) ctas = kMostCtas;
    return (uint32_t)(ctas > most ? most : ctas);
}

template <int FMT, int HD, bool PACKED>
cudaError_t launch_token_as(cudaStream_t stream, const TokenParams& p, uint32_t ctas) {
    static_assert((token_smem_bytes<FMT, HD, PACKED>() + 4096) * ctas_per_sm(HD) <= 228 * 1024, "shared memory of an SM");
    cudaError_t e = ensure_dynamic_smem((const void*)attention_token_paged_kernel<FMT, HD, PACKED>, token_smem_bytes<FMT, HD, PACKED>());
    if (e != cudaSuccess) return e;
    return launch_dependent(attention_token_paged_kernel<FMT, HD, PACKED>, dim3(ctas), dim3(kThreads), token_smem_bytes<FMT, HD, PACKED>(), stream, p);
}
template <int FMT, int HD>
cudaError_t launch_token(cudaStream_t stream, const TokenParams& p) {
    const uint32_t ctas = token_ctas(p.pool, p.rows);
    cudaError_t e = p.group <= 4 ? launch_token_as<FMT, HD, true>(stream, p, ctas) : launch_token_as<FMT, HD, false>(stream, p, ctas);
    if (e != cudaSuccess || ctas == 1 || p.whole) return e;
    return launch_dependent(attention_token_paged_join_kernel<HD>, dim3(ctas - 1, p.group), dim3(256), 0, stream, static_cast<const float*>(p.parts), p.out, p.n_heads, p.group);
}

// Where tables cannot hold more than this many elements of a head's keys, units stay whole: what a CTA takes longer for the longest unit is less
// than the joining launch (one sequence of 8 heads of 64: 301 positions 6.3 us, cut and joined 7.7; 1024 positions 8.5 and 9.8; 2001 12.3 and 10.2).
constexpr uint64_t kWholeElements = 65536;
bool whole_units(const KvRows& rows, const KvPool& pool) { return ((uint64_t)rows.max_pages << pool.page_shift) * pool.head_dim <= kWholeElements; }

uint64_t token_floats(uint32_t head_dim) {
    return (uint64_t)2 * kMostCtas * kRows * (head_dim + 2) + (uint64_t)kMostCtas * sizeof(PartsHead) / 4;
}

}  // namespace

// Which kernel takes a sequence. The tensor-core kernel reads the positions once for all of a sequence's rows and takes the time of 128 of them: as long as
// three rows here where contexts are long (8 sequences of 25000 positions, 8 heads of 64: 168 us; here 134 with 2 rows, 178 with 3, 252 with 4), and 10 to 20 us
// beside that (8 of 5500 with 3 rows: 34 here, 55 there). So sequences of up to three rows are always taken here, and all of a call's, with no second
// kernel, where what the tables can hold, 256 positions more for a unit's beginning and end, times the rows beyond three, is what those 20 us read: (us, here and
// there) 8 sequences of up to 2900 positions with 2 to 5 rows 19 and 30, 64 of 500 with 4 rows 46 and 61, one of 1500 with 16 rows 16 and 21; past it 8 of 1100
// with 16 rows 43 and 28, 64 of 100 with 8 rows 47 and 32. All these are 8 heads of 64. On nine layouts (halves and 8 bits; heads of 64, 128 and 256; one to eight query heads a KV head),
// 4, 8 and 16 rows of 1 to 64 sequences of 500 to 5000 positions, 103 of 108 choices are the quicker form or within 10 % of it; the worst are 8 sequences of 5000 half positions of 8 heads of
// 128 with 4 rows (80 here, 65 there) and 64 of 500, 2 heads of 64 of 7 query heads each, with 8 (30 and 23).
constexpr uint32_t kTokenRows = 3, kFewRows = 32;
bool few_rows(const KvPool& pool, const KvRows& rows) {
    if (rows.max_queries <= kTokenRows) return true;
    const uint64_t positions = ((uint64_t)rows.max_pages << pool.page_shift) + 256;
    const double elements = (double)positions * rows.n_seqs * pool.n_kv_heads * pool.head_dim * 2;
    return rows.max_queries <= kFewRows && (rows.max_queries - kTokenRows) * elements <= 1.1e8;
}

uint64_t attention_paged_scratch_floats(uint32_t, uint32_t, uint32_t head_dim) {
    return token_floats(head_dim) + attention_chunk_scratch_floats(head_dim);
}

int attention_paged_launches(const KvPool& pool, const KvRows& rows, uint32_t) {
    const int tokens = token_ctas(pool, rows) == 1 || whole_units(rows, pool) ? 1 : 2;
    if (few_rows(pool, rows)) return tokens;
    return attention_chunk_launches() + (rows.n_seqs > 1 ? tokens : 0);
}

cudaError_t attention_paged(cudaStream_t stream, const KvPool& pool, const KvRows& rows, const float* q, uint64_t q_stride, uint64_t q_head_stride,
                            float* scratch, float* out, uint32_t n_heads) {
    if (rows.n_rows == 0 || rows.n_seqs == 0) return cudaSuccess;
    // What the caller says of the rows decides which kernels run; the rows themselves, on the device, which of them takes a sequence.
    const bool chunks = !few_rows(pool, rows), tokens = !chunks || rows.n_seqs > 1;
    const TokenParams p{pool, rows, q, out, scratch, q_stride, q_head_stride, n_heads, n_heads / pool.n_kv_heads, chunks ? kTokenRows : 0xffffffffu, whole_units(rows, pool)};
    const bool half = pool.format == BC_F16;
    cudaError_t e = cudaSuccess;
    if (tokens) {
        switch (pool.head_dim) {
            case 64: e = half ? launch_token<BC_F16, 64>(stream, p) : launch_token<BC_I8, 64>(stream, p); break;
            case 128: e = half ? launch_token<BC_F16, 128>(stream, p) : launch_token<BC_I8, 128>(stream, p); break;
            default: e = half ? launch_token<BC_F16, 256>(stream, p) : launch_token<BC_I8, 256>(stream, p);
        }
    }
    if (e != cudaSuccess || !chunks) return e;
    return attention_chunk(stream, pool, rows, q, q_stride, q_head_stride, scratch + token_floats(pool.head_dim), out, n_heads, tokens ? kTokenRows + 1 : 0);
}

}  // namespace k
}  // namespace bc
