// Causal grouped-query attention of the new rows of several sequences over a pool of key/value pages, a query at a time: the form for
// single tokens, whose time is the cache's bytes.
//
// Work. A unit is one row of one KV head: the group of up to 8 query heads that share the head, over the positions that the row sees.
// Units are cut into blocks of 128 positions, and the blocks of all units, in order, into equal runs, one to a CTA: however
// the lengths differ, every CTA reads the same number of positions, and lengths stay on the device (a captured call serves whatever they
// become). A unit that lies in one CTA's run is written out by it; a unit that is cut leaves unnormalised sums with their maximum and sum of
// exponentials, at most two to a CTA, and a second launch joins them in order.
//
// Arithmetic. Elements are exact in half precision (8-bit ones as whole numbers, their scales multiply scores and probabilities in f32).
// A query element, and a probability times the value's scale, is split into two halves, value = hi + lo (about 22 bits), every product is half x
// half summed in f32. So results are those of f32 arithmetic up to the order of the sums. Halves below 2^-14 lose bits, so what is split is brought
// to the upper end of their range by a power of two first: a query row's largest element to 2^14, the largest probability to 2^15, the largest weight of
// 8-bit values to 2^11 or more (`unit` follows it). What is 2^25 times smaller than these still keeps 22 bits or is lost beside them.
//
// A warp takes 16 positions at a time, from global memory straight into the fragments of mma.m16n8k16, no shared memory between.
// Scores: the 16 rows of A are the group's 8 query heads' hi parts, then their lo parts, so one multiply gives both sums and a thread adds
// its two. A lane's 16 bytes of a key are neighbouring elements; the order of elements within a product is free, and the queries
// are stored in the same order. Values are the A operand (elements x positions), for which pairs of positions are woven together by byte permutes;
// B is the probabilities as the scores left them, hi then lo. The next keys' loads are issued when the scores are done, the next values'
// when the sums are: a warp always has about a step's half under way.

#include "kv_pool.cuh"

#include "../../include/bobcat_cuda.h"

namespace bc {
namespace k {

namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr uint32_t kStep = 16;                 // positions a warp takes at a time
constexpr uint32_t kBlock = kStep * kWarps;    // positions of a block, the unit that work is counted in
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
__device__ __forceinline__ void split_half2(float x, float y, uint32_t& hi, uint32_t& lo) {
    __half2 h = __floats2half2_rn(x, y);
    float2 back = __half22float2(h);
    __half2 l = __floats2half2_rn(x - back.x, y - back.y);
    hi = *reinterpret_cast<uint32_t*>(&h);
    lo = *reinterpret_cast<uint32_t*>(&l);
}

// A sequence of the call: its rows, the positions it holds, the blocks its longest row takes.
struct Seq {
    uint32_t row0, n, end, len;
    uint32_t blocks;
};
__device__ __forceinline__ Seq seq_at(const KvPool& pool, const KvRows& rows, uint32_t s, uint32_t most) {
    Seq q;
    q.row0 = rows.starts[s];
    q.end = rows.starts[s + 1];
    q.n = q.row0 < rows.n_rows && q.end > q.row0 && q.end - q.row0 <= most ? min(q.end, rows.n_rows) - q.row0 : 0;
    q.len = rows.lens[s];
    const uint32_t held = min((uint64_t)q.len, (uint64_t)rows.max_pages << pool.page_shift);
    q.blocks = max(1u, (held + kBlock - 1) / kBlock);
    return q;
}
__device__ __forceinline__ uint64_t blocks_of(const KvPool& pool, const Seq& q) { return (uint64_t)q.n * pool.n_kv_heads * q.blocks; }

__device__ __forceinline__ uint64_t warp_sum_u64(uint64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// CTAs that an SM holds, by their registers.
constexpr uint32_t ctas_per_sm(int32_t format, uint32_t head_dim) { return head_dim == 64 || (head_dim == 128 && format == BC_I8) ? 2 : 1; }

// Registers of a warp's step of keys, and of values: 32-bit words per lane.
template <int FMT, int HD>
constexpr int step_words() { return FMT == BC_F16 ? HD / 4 : HD / 8; }

template <int FMT, int HD>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(FMT, HD)) attention_token_paged_kernel(const __grid_constant__ TokenParams p) {
    constexpr int kWords = step_words<FMT, HD>();
    constexpr int kKSteps = HD / 16, kTiles = HD / 16;
    extern __shared__ __align__(16) float token_smem[];
    uint4* q_frag = reinterpret_cast<uint4*>(token_smem);                                    // [kKSteps][32]
    float* sums = token_smem + kKSteps * 32 * 4;                                             // [kWarps][kRows][HD + 4]
    float2* stats = reinterpret_cast<float2*>(sums + kWarps * kRows * (HD + 4));             // [kWarps][kRows]
    __shared__ float q_factor[kRows];
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const KvPool& pool = p.pool;
    const KvRows& rows = p.rows;
    const float scale = 1.4426950408889634f / sqrtf((float)HD);  // scores in powers of two

    // This CTA's run of blocks, and the sequence that it begins in. Every warp works it out for itself.
    uint64_t total = 0;
    for (uint32_t s = lane; s < rows.n_seqs; s += 32) total += blocks_of(pool, seq_at(pool, rows, s, p.most));
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
        const uint64_t mine = s0 + lane < rows.n_seqs ? blocks_of(pool, seq_at(pool, rows, s0 + lane, p.most)) : 0;
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

    while (at < end) {
        Seq sq = seq_at(pool, rows, seq, p.most);
        while (base + blocks_of(pool, sq) <= at) {  // sequences without rows have no blocks
            base += blocks_of(pool, sq);
            sq = seq_at(pool, rows, ++seq, p.most);
        }
        // The unit, and the blocks of it that are this CTA's. Rows of a head are neighbours.
        const uint64_t in_seq = at - base;
        const uint32_t which = (uint32_t)(in_seq / sq.blocks), block0 = (uint32_t)(in_seq % sq.blocks);
        const uint32_t blocks = (uint32_t)min((uint64_t)(sq.blocks - block0), end - at);
        const uint32_t head = which / sq.n, row = sq.row0 + which % sq.n;
        const uint32_t back = sq.end - row;  // the row's distance from the end: it sees positions 0 .. len - back
        const uint32_t held = min((uint64_t)sq.len, (uint64_t)rows.max_pages << pool.page_shift);
        const uint32_t n_keys = back <= sq.len ? min(sq.len - back + 1, held) : 0;
        if (held < sq.len) leave_fault(pool, kFaultTable);

        // Query fragments in the order of a lane's key elements, a warp per query head. A pair of elements is a word of hi and one of lo parts.
        __syncthreads();  // the previous unit's fragments have been read
        {
            float2 x[HD / 64];
            uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < HD / 64; ++i) {
                x[i] = warp < p.group ? *reinterpret_cast<const float2*>(p.q + row * p.q_stride + (head * p.group + warp) * p.q_head_stride + 64 * i + 2 * lane)
                                      : make_float2(0.f, 0.f);
                most = max(most, max(__float_as_uint(x[i].x) & 0x7fffffffu, __float_as_uint(x[i].y) & 0x7fffffffu));
            }
            const uint32_t exponent = min(max(__reduce_max_sync(0xffffffffu, most) >> 23, 1u), 253u);
            const float up = __uint_as_float((254u - exponent) << 23);  // times 2^14 below: together they may pass the largest float
            if (lane == 0) q_factor[warp] = __uint_as_float(exponent << 23) * (scale / 16384.f);
#pragma unroll
            for (int i = 0; i < HD / 64; ++i) {
                uint32_t hi, lo;
                split_half2(x[i].x * up * 16384.f, x[i].y * up * 16384.f, hi, lo);
                const uint32_t e = 2 * lane;  // element 64 i + e
                const uint32_t ks = FMT == BC_F16 ? 4 * i + 2 * (e >> 5) + ((e & 7) >> 2) : 4 * i + ((e & 15) >> 2);
                const uint32_t of_lane = 4 * warp + (FMT == BC_F16 ? (e & 31) >> 3 : e >> 4);
                uint32_t* to = reinterpret_cast<uint32_t*>(q_frag + ks * 32 + of_lane) + (e & 3);  // e & 3 is 0 or 2
                to[0] = hi;
                to[1] = lo;
            }
        }
        __syncthreads();
        const float factor_q = q_factor[g];

        float o[kTiles][4];
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
        float top = -INFINITY, total_p = 0.f;  // of query head g, the sum over this lane's positions
        float unit = FMT == BC_I8 ? 0.f : 1.f, inverse_unit = unit;  // the sums of query head g are counted in these

        uint32_t kw[kWords], vw[kWords];
        float2 dk[2], dv[2];
        const uint32_t* table = rows.table + (uint64_t)seq * rows.max_pages;
        const uint32_t slots = (1u << pool.page_shift) - 1;
        // The warp's steps are one block apart; `pos` is the first position of one.
        const uint32_t pos_end = min((block0 + blocks) * kBlock, n_keys);
        auto page_of = [&](uint32_t pos) { return pos < pos_end ? table[pos >> pool.page_shift] : 0u; };
        auto load_keys = [&](uint32_t pos, uint32_t page) {
            const uint8_t* from = pool.k + kv_row_at(pool, page, head, pos & slots);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int c = 0; c < kWords / 8; ++c) {
                    const uint4 w = *reinterpret_cast<const uint4*>(from + (8 * j + g) * pool.row_bytes + 64 * c + 16 * t);
                    kw[(j * (kWords / 8) + c) * 4 + 0] = w.x;
                    kw[(j * (kWords / 8) + c) * 4 + 1] = w.y;
                    kw[(j * (kWords / 8) + c) * 4 + 2] = w.z;
                    kw[(j * (kWords / 8) + c) * 4 + 3] = w.w;
                }
            if (FMT == BC_I8) {
                const float* s = reinterpret_cast<const float*>(pool.k + kv_scale_at(pool, page, head, pos & slots));
                dk[0] = *reinterpret_cast<const float2*>(s + 2 * t);
                dk[1] = *reinterpret_cast<const float2*>(s + 8 + 2 * t);
            }
        };
        // Position 2t + (i & 1) + 8 (i >> 1) of the step, i = 0 .. 3; a lane's 8 elements 8g .. of every 64.
        auto load_values = [&](uint32_t pos, uint32_t page) {
            const uint8_t* from = pool.v + kv_row_at(pool, page, head, pos & slots);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint8_t* at_row = from + (2 * t + (i & 1) + 8 * (i >> 1)) * pool.row_bytes;
#pragma unroll
                for (int c = 0; c < HD / 64; ++c) {
                    if constexpr (FMT == BC_F16) {
                        const uint4 w = *reinterpret_cast<const uint4*>(at_row + 128 * c + 16 * g);
                        vw[(i * (HD / 64) + c) * 4 + 0] = w.x;
                        vw[(i * (HD / 64) + c) * 4 + 1] = w.y;
                        vw[(i * (HD / 64) + c) * 4 + 2] = w.z;
                        vw[(i * (HD / 64) + c) * 4 + 3] = w.w;
                    } else {
                        const uint2 w = *reinterpret_cast<const uint2*>(at_row + 64 * c + 8 * g);
                        vw[(i * (HD / 64) + c) * 2 + 0] = w.x;
                        vw[(i * (HD / 64) + c) * 2 + 1] = w.y;
                    }
                }
            }
            if (FMT == BC_I8) {
                const float* s = reinterpret_cast<const float*>(pool.v + kv_scale_at(pool, page, head, pos & slots));
                dv[0] = *reinterpret_cast<const float2*>(s + 2 * t);
                dv[1] = *reinterpret_cast<const float2*>(s + 8 + 2 * t);
            }
        };

        uint32_t pos = block0 * kBlock + warp * kStep;
        uint32_t page = page_of(pos), next_page = page_of(pos + kBlock);
        bool good = page < pool.n_pages;  // a page that the pool does not have holds nothing
        if (pos < pos_end && good) load_keys(pos, page);
        while (pos < pos_end) {  // uniform in the warp
            const uint32_t next = pos + kBlock;
            const bool next_good = next_page < pool.n_pages;
            if (!good) {
                if (lane == 0) leave_fault(pool, kFaultPage);
                if (next < pos_end && next_good) load_keys(next, next_page);
            } else {
                load_values(pos, page);
                float s[2][4];
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[j][i] = 0.f;
#pragma unroll
                for (int ks = 0; ks < kKSteps; ++ks) {
                    const uint4 f = q_frag[ks * 32 + lane];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        uint32_t b0, b1;
                        if constexpr (FMT == BC_F16) {
                            b0 = kw[j * (kWords / 2) + 2 * ks];
                            b1 = kw[j * (kWords / 2) + 2 * ks + 1];
                        } else {
                            unpack_i8(kw[j * (kWords / 2) + ks], b0, b1);
                        }
                        mma_f16(s[j], f.x, f.y, f.z, f.w, b0, b1);
                    }
                }
                float x[4];  // scores of positions 2t, 2t + 1, 8 + 2t, 9 + 2t for query head g
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    x[2 * j] = (s[j][0] + s[j][2]) * factor_q;
                    x[2 * j + 1] = (s[j][1] + s[j][3]) * factor_q;
                    if (FMT == BC_I8) {
                        x[2 * j] *= dk[j].x;
                        x[2 * j + 1] *= dk[j].y;
                    }
                }
                if (next < pos_end && next_good) load_keys(next, next_page);
                const uint32_t left = n_keys - pos;  // positions of the step that exist, if fewer than 16
                if (left < kStep) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (2 * t + (i & 1) + 8 * (i >> 1) >= left) x[i] = -INFINITY;
                }
                float most = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                const float now = fmaxf(top, most);
                const float shift = now == -INFINITY ? 0.f : now;
                float factor = exp2f(top - shift);
                bool moved = now > top;
                top = now;
                float total_step = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] = exp2f(x[i] - shift + kLift);  // the sums are lifted alike
                    total_step += x[i];
                }
                total_p = total_p * factor + total_step;
                if (FMT == BC_I8) {
                    float largest = 0.f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float d = i & 1 ? dv[i >> 1].y : dv[i >> 1].x;
                        x[i] = 2 * t + (i & 1) + 8 * (i >> 1) < left ? x[i] * d : 0.f;  // scales behind the last position may be anything
                        largest = fmaxf(largest, fabsf(x[i]));
                    }
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
                        moved = true;
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] *= inverse_unit;
                }
                if (__any_sync(0xffffffffu, moved)) {
                    const float f0 = __shfl_sync(0xffffffffu, factor, 8 * t), f1 = __shfl_sync(0xffffffffu, factor, 8 * t + 4);
#pragma unroll
                    for (int n = 0; n < kTiles; ++n) {
                        o[n][0] *= f0;
                        o[n][1] *= f1;
                        o[n][2] *= f0;
                        o[n][3] *= f1;
                    }
                }
                uint32_t hi0, lo0, hi1, lo1;
                split_half2(x[0], x[1], hi0, lo0);
                split_half2(x[2], x[3], hi1, lo1);
                if constexpr (FMT == BC_F16) {
                    if (left < kStep) {  // elements behind the last position may be anything
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (2 * t + (i & 1) + 8 * (i >> 1) >= left) {
#pragma unroll
                                for (int w = 0; w < kWords / 4; ++w) vw[i * (kWords / 4) + w] = 0;
                            }
                    }
#pragma unroll
                    for (int w = 0; w < kWords / 4; ++w) {  // elements 2w, 2w + 1 of the lane's: rows g and g + 8 of a tile
                        const uint32_t a = vw[w], b = vw[kWords / 4 + w], c = vw[2 * (kWords / 4) + w], d = vw[3 * (kWords / 4) + w];
                        const uint32_t a0 = __byte_perm(a, b, 0x5410), a1 = __byte_perm(a, b, 0x7632), a2 = __byte_perm(c, d, 0x5410), a3 = __byte_perm(c, d, 0x7632);
                        mma_f16(o[w], a0, a1, a2, a3, hi0, hi1);
                        mma_f16(o[w], a0, a1, a2, a3, lo0, lo1);
                    }
                } else {
#pragma unroll
                    for (int w = 0; w < kWords / 4; ++w) {  // elements 4w .. 4w + 3 of the lane's: two tiles
                        const uint32_t a = vw[w], b = vw[kWords / 4 + w], c = vw[2 * (kWords / 4) + w], d = vw[3 * (kWords / 4) + w];
                        const uint32_t ab_lo = __byte_perm(a, b, 0x5140), ab_hi = __byte_perm(a, b, 0x7362);  // a0 b0 a1 b1, a2 b2 a3 b3
                        const uint32_t cd_lo = __byte_perm(c, d, 0x5140), cd_hi = __byte_perm(c, d, 0x7362);
                        uint32_t a0, a1, a2, a3;
                        unpack_i8(ab_lo, a0, a1);
                        unpack_i8(cd_lo, a2, a3);
                        mma_f16(o[2 * w], a0, a1, a2, a3, hi0, hi1);
                        mma_f16(o[2 * w], a0, a1, a2, a3, lo0, lo1);
                        unpack_i8(ab_hi, a0, a1);
                        unpack_i8(cd_hi, a2, a3);
                        mma_f16(o[2 * w + 1], a0, a1, a2, a3, hi0, hi1);
                        mma_f16(o[2 * w + 1], a0, a1, a2, a3, lo0, lo1);
                    }
                }
            }
            pos = next;
            page = next_page;
            good = next_good;
            next_page = page_of(pos + kBlock);
        }

        // The warps' sums, joined through shared memory. Tile n's rows g and g + 8 are elements 2n' and 2n' + 1 of the lane's eight: see load_values.
        total_p += __shfl_xor_sync(0xffffffffu, total_p, 1);
        total_p += __shfl_xor_sync(0xffffffffu, total_p, 2);
        if (t == 0) stats[warp * kRows + g] = make_float2(top, total_p);
        const float u0 = __shfl_sync(0xffffffffu, unit, 8 * t), u1 = __shfl_sync(0xffffffffu, unit, 8 * t + 4);
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
            const uint32_t d = (n / 4) * 64 + 8 * g + 2 * (n % 4);  // elements d and d + 1
            float* to = sums + (warp * kRows + 2 * t) * (HD + 4) + d;
            *reinterpret_cast<float2*>(to) = make_float2(o[n][0] * u0, o[n][2] * u0);
            *reinterpret_cast<float2*>(to + HD + 4) = make_float2(o[n][1] * u1, o[n][3] * u1);
        }
        __syncthreads();
        const bool begins = block0 == 0, ends = block0 + blocks == sq.blocks;
        const uint32_t slot = 2 * blockIdx.x + (begins ? 1 : 0);
        for (uint32_t i = tid; i < p.group * (HD / 4); i += kThreads) {
            const uint32_t r = i / (HD / 4), d = i % (HD / 4) * 4;
            float most = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) most = fmaxf(most, stats[w * kRows + r].x);
            const float shift = most == -INFINITY ? 0.f : most;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
            float sum_p = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float2 st = stats[w * kRows + r];
                const float weight = st.x == -INFINITY ? 0.f : exp2f(st.x - shift);
                const float4 v = *reinterpret_cast<const float4*>(sums + (w * kRows + r) * (HD + 4) + d);
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
                *reinterpret_cast<float4*>(p.out + (uint64_t)row * p.n_heads * HD + (head * p.group + r) * HD + d) =
                    make_float4(sum.x * inverse, sum.y * inverse, sum.z * inverse, sum.w * inverse);
            } else {
                *reinterpret_cast<float4*>(p.parts + ((uint64_t)slot * kRows + r) * HD + d) = sum;
                if (d == 0) *reinterpret_cast<float2*>(p.parts + (uint64_t)2 * kMostCtas * kRows * HD + (slot * kRows + r) * 2) = make_float2(most, sum_p);
            }
        }
        if (begins && !ends) {
            // The CTA whose run holds the unit's last block: run c is [total c / runs, total (c + 1) / runs).
            const uint64_t last_block = at + sq.blocks - 1;
            uint32_t last = (uint32_t)(last_block * runs / total);
            while (total * (last + 1) / runs <= last_block) ++last;
            while (total * last / runs > last_block) --last;
            cut = PartsHead{row, head, last, 0};
        }
        at += blocks;
    }
    if (tid == 0) heads[blockIdx.x] = cut;
}

// Joins the parts of a unit that begins in CTA c's run and ends in a later one's: a warp per query head.
template <int HD>
__global__ void __launch_bounds__(32 * kRows) attention_token_join_kernel(const float* __restrict__ parts, float* __restrict__ out, uint32_t n_heads, uint32_t group) {
    constexpr int kPairs = HD / 64;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t lane = threadIdx.x & 31, r = threadIdx.x >> 5, c = blockIdx.x;
    const PartsHead cut = reinterpret_cast<const PartsHead*>(parts + (uint64_t)2 * kMostCtas * kRows * (HD + 2))[c];
    if (cut.last == 0 || r >= group) return;
    const float2* stats = reinterpret_cast<const float2*>(parts + (uint64_t)2 * kMostCtas * kRows * HD);
    const uint32_t n = cut.last - c + 1;
    auto slot_of = [&](uint32_t i) { return 2 * (c + i) + (i == 0 ? 1 : 0); };
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
            const float2* from = reinterpret_cast<const float2*>(parts + ((uint64_t)slot_of(i0 + i) * kRows + r) * HD) + lane;
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
    const float inverse = top == -INFINITY && total == 0.f ? 0.f : 1.f / total;
    float2* to = reinterpret_cast<float2*>(out + (uint64_t)cut.row * n_heads * HD + (cut.head * group + r) * HD) + lane;
#pragma unroll
    for (int k = 0; k < kPairs; ++k) to[32 * k] = make_float2(sum[k].x * inverse, sum[k].y * inverse);
}

template <int HD>
constexpr size_t token_smem_bytes() { return (size_t)(HD / 16) * 32 * 16 + (size_t)kWarps * kRows * (HD + 4) * 4 + kWarps * kRows * 8; }

// CTAs of a launch: no more than the blocks that the tables could hold.
uint32_t token_ctas(const KvPool& pool, const KvRows& rows) {
    const uint64_t most = (uint64_t)rows.n_rows * pool.n_kv_heads * ((((uint64_t)rows.max_pages << pool.page_shift) + kBlock - 1) / kBlock);
    uint64_t ctas = (uint64_t)sm_count() * ctas_per_sm(pool.format, pool.head_dim);
    if (ctas > kMostCtas) ctas = kMostCtas;
    return (uint32_t)(ctas > most ? most : ctas);
}

template <int FMT, int HD>
cudaError_t launch_token(cudaStream_t stream, const TokenParams& p) {
    cudaError_t e = ensure_dynamic_smem((const void*)attention_token_paged_kernel<FMT, HD>, token_smem_bytes<HD>());
    if (e != cudaSuccess) return e;
    const uint32_t ctas = token_ctas(p.pool, p.rows);
    e = launch_dependent(attention_token_paged_kernel<FMT, HD>, dim3(ctas), dim3(kThreads), token_smem_bytes<HD>(), stream, p);
    if (e != cudaSuccess || ctas == 1) return e;
    return launch_dependent(attention_token_join_kernel<HD>, dim3(ctas - 1), dim3(32 * kRows), 0, stream, static_cast<const float*>(p.parts), p.out, p.n_heads, p.group);
}

uint64_t token_floats(uint32_t head_dim) {
    return (uint64_t)2 * kMostCtas * kRows * (head_dim + 2) + (uint64_t)kMostCtas * sizeof(PartsHead) / 4;
}

}  // namespace

// Rows of a sequence up to which each is a unit of its own. The tensor-core kernel reads the positions once for all rows, and takes
// the time of 128.
constexpr uint32_t kTokenRows = 1;

uint64_t attention_paged_scratch_floats(uint32_t, uint32_t, uint32_t head_dim) {
    return token_floats(head_dim) + attention_chunk_scratch_floats(head_dim);
}

int attention_paged_launches(const KvPool& pool, const KvRows& rows, uint32_t) {
    const int tokens = token_ctas(pool, rows) == 1 ? 1 : 2;
    if (rows.max_queries <= kTokenRows) return tokens;
    return attention_chunk_launches() + (rows.n_seqs > 1 ? tokens : 0);
}

cudaError_t attention_paged(cudaStream_t stream, const KvPool& pool, const KvRows& rows, const float* q, uint64_t q_stride, uint64_t q_head_stride,
                            float* scratch, float* out, uint32_t n_heads) {
    if (rows.n_rows == 0 || rows.n_seqs == 0) return cudaSuccess;
    // What the caller says of the rows decides which kernels run; the rows themselves, on the device, which of them takes a sequence.
    const bool chunks = rows.max_queries > kTokenRows, tokens = !chunks || rows.n_seqs > 1;
    const TokenParams p{pool, rows, q, out, scratch, q_stride, q_head_stride, n_heads, n_heads / pool.n_kv_heads, chunks ? kTokenRows : 0xffffffffu};
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
