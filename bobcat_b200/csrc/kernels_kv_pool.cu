// Rows into the pages of a key/value pool, and back.
//
// Writing (8 bit). A row is the head_dim elements of one head at one position: d = f32(max |x| / 127), q = the whole number nearest to
// x / d, ties to even. One fma rounds x * (1 / d) to a whole number (added to 1.5 * 2^23 + 128, whose last byte is then the one stored); the product
// is within 2^-16 of x / d, so only where it lies that near the middle between two numbers (one element in 5000 is taken to) does a second look
// decide: x - q d, which an fma gives without error (a multiple of both operands' last places, no longer than a float), against d / 2.
// Rows whose d is not a normal number (all elements below 127 * 2^-126) are stored as zeros; a row with an infinity or a NaN gets a scale of
// NaN, so it reads as NaN throughout. Half pages store the elements rounded to nearest.
//
// What bounds it: bytes, 4 read and 1 (+ 4 / head_dim) or 2 written per element, and the look-up of a row's place before the
// first store. A lane holds 8 elements (two 16-byte loads, one 8- or 16-byte store), a cell (one head's row of keys or of values) is
// 8, 16 or 32 lanes. A CTA takes neighbouring token rows; its warps look the rows' places up while the first cells' loads are on their way. Large
// calls are bound by bytes as long as an element costs few instructions: the rows of eight prompts (32 008 of 2 x 8 heads of 128) take 60 us (262 MB read, 68 written:
// 5.5 TB/s), with the exact test for every element, 50 instructions, 117.

#include "kv_pool.cuh"

#include "../../include/bobcat_cuda.h"

namespace bc {
namespace k {

namespace {

constexpr int kThreads = 256;
constexpr uint32_t kRowsPerCta = 8;  // at most: one warp looks up each

// Cells of a token row, and how to divide by their number.
struct Cells {
    uint32_t per_row, magic, rows_per_cta;
    __device__ __forceinline__ uint32_t row(uint32_t cell) const { return __umulhi(cell, magic); }  // cell * per_row < 2^32
};

// The larger magnitude; NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Places of the CTA's rows; the sequence look-up is a warp's.
__device__ __forceinline__ void look_up(const KvPool& pool, const KvRows& rows, uint32_t row0, uint32_t n, uint2* place) {
    const uint32_t warp = threadIdx.x >> 5;
    if (warp < n) {
        const uint32_t r = row0 + warp, seq = seq_of_row(rows, r);
        if ((threadIdx.x & 31) == 0) {
            uint2 at = make_uint2(kNoSlot, 1);  // 1: no such row of any sequence, 0: a row without a place
            if (seq < rows.n_seqs) {
                const uint32_t back = rows.starts[seq + 1] - r, len = rows.lens[seq];
                at = back <= len ? kv_place(pool, rows, seq, len - back) : make_uint2(kNoSlot, 0);
            }
            place[warp] = at;
        }
    }
}

struct Sources {
    const float *k, *v;
    uint64_t k_stride, v_stride;
};

template <int FMT, int HD>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const __grid_constant__ KvPool pool, const __grid_constant__ KvRows rows,
                                                            const __grid_constant__ Sources src, const __grid_constant__ Cells cells) {
    constexpr uint32_t kLanes = HD / 8, kCellsAtOnce = kThreads / kLanes;
    __shared__ uint2 place[kRowsPerCta];
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t row0 = blockIdx.x * cells.rows_per_cta, n = min(cells.rows_per_cta, rows.n_rows - row0);
    const uint32_t n_cells = n * cells.per_row;
    const uint32_t lane = threadIdx.x % kLanes, first = threadIdx.x / kLanes;
    auto load = [&](uint32_t cell, float (&x)[8]) {
        const uint32_t row = cells.row(cell), head = cell - row * cells.per_row;
        const bool value = head >= pool.n_kv_heads;
        const float* from = value ? src.v + (row0 + row) * src.v_stride + (head - pool.n_kv_heads) * HD : src.k + (row0 + row) * src.k_stride + head * HD;
        const float4 a = __ldcs(reinterpret_cast<const float4*>(from) + 2 * lane), b = __ldcs(reinterpret_cast<const float4*>(from) + 2 * lane + 1);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    };
    float next[8] = {};
    if (first < n_cells) load(first, next);
    look_up(pool, rows, row0, n, place);
    __syncthreads();
    for (uint32_t cell0 = 0; cell0 < n_cells; cell0 += kCellsAtOnce) {
        const uint32_t cell = cell0 + first;
        const bool mine = cell < n_cells;
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = next[i];
        if (cell + kCellsAtOnce < n_cells) load(cell + kCellsAtOnce, next);
        const uint32_t row = mine ? cells.row(cell) : 0, head = mine ? cell - row * cells.per_row : 0;
        const bool value = head >= pool.n_kv_heads;
        const uint2 at = place[row];
        uint8_t* const to = value ? pool.v : pool.k;
        const uint32_t kv_head = value ? head - pool.n_kv_heads : head;
        const bool store = mine && at.x != kNoSlot;
        if constexpr (FMT == BC_F16) {
            if (store) {
                __half2 h[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
                *reinterpret_cast<uint4*>(to + kv_row_at(pool, at.x, kv_head, at.y) + 16 * lane) = *reinterpret_cast<uint4*>(h);
            }
        } else {
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max_nan(top, fabsf(x[i]));
#pragma unroll
            for (uint32_t o = kLanes / 2; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
            float d = __fdiv_rn(top, 127.f);
            const bool finite = top < INFINITY;
            if (!(d >= 1.17549435e-38f)) d = 0.f;
            const float inverse = d > 0.f && finite ? __frcp_rn(d) : 0.f;
            constexpr float kMagic = 12583040.f;  // 1.5 * 2^23 + 128
            uint32_t bytes[2] = {0x80808080u, 0x80808080u};
            if (inverse > 0.f) {
                float whole[8], furthest = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    whole[i] = fmaf(x[i], inverse, kMagic);
                    furthest = fmaxf(furthest, fabsf(fmaf(x[i], inverse, kMagic - whole[i])));
                }
                if (furthest > 0.4999f) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float q = whole[i] - kMagic, twice = 2.f * fmaf(-q, d, x[i]);
                        const bool odd = __float_as_uint(whole[i]) & 1;
                        if (twice > d || (twice == d && odd)) whole[i] += 1.f;
                        if (twice < -d || (twice == -d && odd)) whole[i] -= 1.f;
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t low = __byte_perm(__float_as_uint(whole[4 * h]), __float_as_uint(whole[4 * h + 1]), 0x0040);
                    const uint32_t high = __byte_perm(__float_as_uint(whole[4 * h + 2]), __float_as_uint(whole[4 * h + 3]), 0x0040);
                    bytes[h] = __byte_perm(low, high, 0x5410);
                }
            }
            if (store) {
                *reinterpret_cast<uint2*>(to + kv_row_at(pool, at.x, kv_head, at.y) + 8 * lane) = make_uint2(bytes[0], bytes[1]);
                if (lane == 0) *reinterpret_cast<float*>(to + kv_scale_at(pool, at.x, kv_head, at.y)) = finite ? d : __uint_as_float(0x7fc00000u);
            }
        }
    }
}

// Reading. Rows of a sequence without a place (before its first position, behind the table, in no page of the pool) read as zeros; rows
// of no sequence stay as they are. A lane takes two eights of a cell where what it writes of each is one store: what a cell costs beside its bytes counts
// once (contexts of 104 000 positions of 2 x 4 heads of 256, 8 bits, as halves: 99 us, 115 with one eight); as floats, 206 us and 182, it takes one.
struct Targets {
    void *k, *v;
    uint64_t k_stride, v_stride;
};

template <int FMT, int HD, typename Out>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const __grid_constant__ KvPool pool, const __grid_constant__ KvRows rows,
                                                           const __grid_constant__ Targets dst, const __grid_constant__ Cells cells) {
    constexpr uint32_t kEights = sizeof(Out) == 2 ? 2 : 1;
    constexpr uint32_t kLanes = HD / (8 * kEights), kCellsAtOnce = kThreads / kLanes;
    constexpr int kAhead = 4 / kEights;  // cells a lane has loads under way for
    __shared__ uint2 place[kRowsPerCta];
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t row0 = blockIdx.x * cells.rows_per_cta, n = min(cells.rows_per_cta, rows.n_rows - row0);
    const uint32_t n_cells = n * cells.per_row;
    const uint32_t lane = threadIdx.x % kLanes, first = threadIdx.x / kLanes;
    look_up(pool, rows, row0, n, place);
    __syncthreads();
    for (uint32_t cell0 = first; cell0 < n_cells; cell0 += kAhead * kCellsAtOnce) {
        uint4 raw[kAhead][kEights];
        float scale[kAhead];
        Out* to[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const uint32_t cell = cell0 + j * kCellsAtOnce;
#pragma unroll
            for (uint32_t g = 0; g < kEights; ++g) raw[j][g] = FMT == BC_F16 ? make_uint4(0, 0, 0, 0) : make_uint4(0x80808080u, 0x80808080u, 0, 0);
            scale[j] = 0.f;
            to[j] = nullptr;
            if (cell >= n_cells) continue;
            const uint32_t row = cells.row(cell), head = cell - row * cells.per_row;
            const bool value = head >= pool.n_kv_heads;
            const uint2 at = place[row];
            void* const base = value ? dst.v : dst.k;
            if (!base || (at.x == kNoSlot && at.y == 1)) continue;
            const uint32_t kv_head = value ? head - pool.n_kv_heads : head;
            to[j] = static_cast<Out*>(base) + (row0 + row) * (value ? dst.v_stride : dst.k_stride) + kv_head * HD + 8 * lane;
            if (at.x == kNoSlot) continue;
            const uint8_t* const from = value ? pool.v : pool.k;
            const uint8_t* const row_from = from + kv_row_at(pool, at.x, kv_head, at.y);
#pragma unroll
            for (uint32_t g = 0; g < kEights; ++g) {
                if constexpr (FMT == BC_F16) {
                    raw[j][g] = __ldcs(reinterpret_cast<const uint4*>(row_from + 16 * (lane + g * kLanes)));
                } else {
                    const uint2 b = __ldcs(reinterpret_cast<const uint2*>(row_from + 8 * (lane + g * kLanes)));
                    raw[j][g].x = b.x;
                    raw[j][g].y = b.y;
                }
            }
            if constexpr (FMT == BC_I8) scale[j] = *reinterpret_cast<const float*>(from + kv_scale_at(pool, at.x, kv_head, at.y));
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (!to[j]) continue;
#pragma unroll
            for (uint32_t g = 0; g < kEights; ++g) {
                Out* const eight = to[j] + 8 * g * kLanes;
                if constexpr (FMT == BC_F16 && sizeof(Out) == 2) {
                    __stcs(reinterpret_cast<uint4*>(eight), raw[j][g]);
                    continue;
                }
                float x[8];
                if constexpr (FMT == BC_F16) {
                    const __half2* h = reinterpret_cast<const __half2*>(&raw[j][g]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 f = __half22float2(h[i]);
                        x[2 * i] = f.x;
                        x[2 * i + 1] = f.y;
                    }
                } else {
                    const uint32_t words[2] = {raw[j][g].x, raw[j][g].y};
#pragma unroll
                    for (int i = 0; i < 8; ++i)  // the byte as the last of 2^23's
                        x[i] = (__uint_as_float(__byte_perm(words[i / 4], 0x4b000000u, 0x7440 + i % 4)) - 8388736.f) * scale[j];
                }
                if constexpr (sizeof(Out) == 4) {
                    __stcs(reinterpret_cast<float4*>(eight), make_float4(x[0], x[1], x[2], x[3]));
                    __stcs(reinterpret_cast<float4*>(eight) + 1, make_float4(x[4], x[5], x[6], x[7]));
                } else {
                    __half2 h[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
                    __stcs(reinterpret_cast<uint4*>(eight), *reinterpret_cast<uint4*>(h));
                }
            }
        }
    }
}

// Token rows per CTA: a CTA works through at most about `rounds` rounds of its threads, fewer where that leaves SMs without one. 104 000 positions of 2 x 4
// heads of 256 are read as halves in 99 us in 4 rounds (115 in 2, 139 in one), as floats in 182 in 8 (196 in 4).
Cells cells_of(const KvPool& pool, const KvRows& rows, uint32_t rounds) {
    const uint32_t per_row = 2 * pool.n_kv_heads, lanes_per_row = per_row * (pool.head_dim / 8);
    uint32_t n = rounds * kThreads / lanes_per_row;
    if (n > kRowsPerCta) n = kRowsPerCta;
    while (n > 1 && (rows.n_rows + n - 1) / n < 4 * (uint32_t)sm_count()) n /= 2;
    return Cells{per_row, (uint32_t)(((1ull << 32) + per_row - 1) / per_row), n < 1 ? 1 : n};
}

template <int FMT, int HD>
cudaError_t write_as(cudaStream_t stream, const KvPool& pool, const KvRows& rows, const Sources& src) {
    const Cells cells = cells_of(pool, rows, 4);
    return launch_dependent(kv_write_kernel<FMT, HD>, dim3((rows.n_rows + cells.rows_per_cta - 1) / cells.rows_per_cta), dim3(kThreads), 0, stream, pool, rows, src, cells);
}
template <int FMT, int HD>
cudaError_t read_as(cudaStream_t stream, const KvPool& pool, const KvRows& rows, const Targets& dst, bool half) {
    const Cells cells = cells_of(pool, rows, half ? 4 : 8);
    const dim3 grid((rows.n_rows + cells.rows_per_cta - 1) / cells.rows_per_cta);
    return half ? launch_dependent(kv_read_kernel<FMT, HD, __half>, grid, dim3(kThreads), 0, stream, pool, rows, dst, cells)
                : launch_dependent(kv_read_kernel<FMT, HD, float>, grid, dim3(kThreads), 0, stream, pool, rows, dst, cells);
}

}  // namespace

cudaError_t kv_write(cudaStream_t stream, const KvPool& pool, const KvRows& rows, const float* k, const float* v, uint64_t k_stride, uint64_t v_stride) {
    if (rows.n_rows == 0) return cudaSuccess;
    const Sources src{k, v, k_stride, v_stride};
    const bool half = pool.format == BC_F16;
    switch (pool.head_dim) {
        case 64: return half ? write_as<BC_F16, 64>(stream, pool, rows, src) : write_as<BC_I8, 64>(stream, pool, rows, src);
        case 128: return half ? write_as<BC_F16, 128>(stream, pool, rows, src) : write_as<BC_I8, 128>(stream, pool, rows, src);
        default: return half ? write_as<BC_F16, 256>(stream, pool, rows, src) : write_as<BC_I8, 256>(stream, pool, rows, src);
    }
}

cudaError_t kv_read(cudaStream_t stream, const KvPool& pool, const KvRows& rows, void* k, void* v, bool out_half, uint64_t k_stride, uint64_t v_stride) {
    if (rows.n_rows == 0) return cudaSuccess;
    const Targets dst{k, v, k_stride, v_stride};
    const bool half = pool.format == BC_F16;
    switch (pool.head_dim) {
        case 64: return half ? read_as<BC_F16, 64>(stream, pool, rows, dst, out_half) : read_as<BC_I8, 64>(stream, pool, rows, dst, out_half);
        case 128: return half ? read_as<BC_F16, 128>(stream, pool, rows, dst, out_half) : read_as<BC_I8, 128>(stream, pool, rows, dst, out_half);
        default: return half ? read_as<BC_F16, 256>(stream, pool, rows, dst, out_half) : read_as<BC_I8, 256>(stream, pool, rows, dst, out_half);
    }
}

}  // namespace k
}  // namespace bc
