// A pool of key/value pages as the kernels see it, and where a row of a call lies in it.
//
// A page holds `page_size` positions (a power of two, 16 to 256) of every KV head, [KV head][position][head_dim], keys and
// values in a pool each. Halves are stored as they are; an 8-bit page stores an element's integer plus 128, which the
// readers turn into a half with one byte permute and one subtraction, and has f32 scales [KV head][position] behind its elements.
// A head's positions of one page lie next to each other, so the readers' tiles are runs of up to a whole page.
#pragma once

#include "device_utils.cuh"
#include "kernels.h"

namespace bc {
namespace k {

constexpr uint32_t kNoSlot = 0xffffffffu;
// Codes left in KvPool::fault.
constexpr int kFaultPage = 1, kFaultTable = 2;

__device__ __forceinline__ void leave_fault(const KvPool& p, int code) { *reinterpret_cast<volatile int*>(p.fault) = code; }

// Byte offset in a pool of position `slot` of `head` in page `page`, of its elements and of its scale.
__device__ __forceinline__ uint64_t kv_row_at(const KvPool& p, uint32_t page, uint32_t head, uint32_t slot) {
    return (uint64_t)page * p.page_bytes + (uint64_t)((head << p.page_shift) + slot) * p.row_bytes;
}
__device__ __forceinline__ uint64_t kv_scale_at(const KvPool& p, uint32_t page, uint32_t head, uint32_t slot) {
    return (uint64_t)page * p.page_bytes + ((uint64_t)(p.n_kv_heads << p.page_shift) * p.row_bytes) + (uint64_t)((head << p.page_shift) + slot) * 4;
}

// The sequence that row `r` belongs to, by one warp: starts[] ascends, so it is the number of sequences that begin at or before r, less
// one. n_seqs for a row behind the last sequence (the end of the last one counts too) or ahead of the first. 32 candidates a step, one step for up to 31
// sequences, four for 65535 (a row each: 27 us; with every start read by every row 1190).
__device__ __forceinline__ uint32_t seq_of_row(const KvRows& rows, uint32_t r) {
    const uint32_t lane = threadIdx.x & 31;
    uint32_t lo = 0, span = rows.n_seqs + 1;
    while (true) {
        const uint32_t step = (span + 31) / 32;
        const uint32_t below = __popc(__ballot_sync(0xffffffffu, lane * step < span && rows.starts[lo + lane * step] <= r));
        if (below == 0) return rows.n_seqs;  // ahead of the first
        lo += (below - 1) * step;
        span = min(step, span - (below - 1) * step);
        if (span == 1) return lo;
    }
}

// Page and slot of position `pos` of a sequence; kNoSlot, and a fault left behind, where the table has none.
__device__ __forceinline__ uint2 kv_place(const KvPool& pool, const KvRows& rows, uint32_t seq, uint32_t pos) {
    const uint32_t column = pos >> pool.page_shift;
    if (column >= rows.max_pages) {
        leave_fault(pool, kFaultTable);
        return make_uint2(kNoSlot, 0);
    }
    const uint32_t page = rows.table[(uint64_t)seq * rows.max_pages + column];
    if (page >= pool.n_pages) {
        leave_fault(pool, kFaultPage);
        return make_uint2(kNoSlot, 0);
    }
    return make_uint2(page, pos & ((1u << pool.page_shift) - 1));
}

// Four stored bytes as two pairs of halves: the bytes become the low mantissa bits of 1024 + byte.
__device__ __forceinline__ void unpack_i8(uint32_t w, uint32_t& lo, uint32_t& hi) {
    const __half2 bias = __floats2half2_rn(1152.f, 1152.f);
    uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
    __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), bias), y = __hsub2(*reinterpret_cast<__half2*>(&b), bias);
    lo = *reinterpret_cast<uint32_t*>(&x);
    hi = *reinterpret_cast<uint32_t*>(&y);
}

// Arithmetic of both kernels of attention over pages.
__device__ __forceinline__ float exp2_fast(float x) {  // results below the normal numbers are zero
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {  // two in one instruction
    float2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t&>(r))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
    return r;
}
// (x, y) as halves and what they leave over, as halves.
__device__ __forceinline__ void split_half2(float x, float y, uint32_t& hi, uint32_t& lo) {
    __half2 h = __floats2half2_rn(x, y);
    float2 back = __half22float2(h);
    __half2 l = __floats2half2_rn(x - back.x, y - back.y);
    hi = *reinterpret_cast<uint32_t*>(&h);
    lo = *reinterpret_cast<uint32_t*>(&l);
}

// Whether the score of a query with a half key that is not finite is minus infinity: every infinite element's product with the query's is, and there is no NaN.
// (Products of a query's halves with an infinity need not have its sign, and are no number where a half is zero.)
__device__ __forceinline__ bool score_is_minus_infinity(const float* q, const uint8_t* key, uint32_t head_dim) {
    bool minus = false;
#pragma unroll 1
    for (uint32_t e = 0; e < head_dim; e += 2) {
        const uint32_t pair = *reinterpret_cast<const uint32_t*>(key + 2 * e);
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
            const uint32_t bits = pair >> (16 * i) & 0xffffu;
            if ((bits & 0x7fffu) < 0x7c00u) continue;
            const float x = q[e + i];
            if ((bits & 0x7fffu) > 0x7c00u || !(bits >> 15 ? x > 0.f : x < 0.f)) return false;
            minus = true;
        }
    }
    return minus;
}

}  // namespace k
}  // namespace bc
