// Bounds-checked op wrappers of the key/value pool, and buffers over memory of the caller's. What lies on the device (page tables, row
// starts, lengths) is checked by the kernels: see kv_pool.cuh.

#include <cuda.h>

#include <new>

#include "backend.h"

using namespace bc;

namespace {

bc_status recording(bc_backend* b) {
    if (!b) return fail(BC_ERR_ARGUMENT, "backend must be non-null");
    if (!b->recording) return fail(BC_ERR_NOT_RECORDING, "no recording is open");
    return b->activate();
}

template <typename T>
T* at(bc_buffer* buffer, size_t offset) {
    return buffer ? reinterpret_cast<T*>(static_cast<char*>(buffer->ptr) + offset) : nullptr;
}

constexpr uint32_t kMostKvHeads = 1024, kMostSeqs = 65535;

bool pool_shape(int32_t format, uint32_t page_size, uint32_t n_kv_heads, uint32_t head_dim) {
    return (format == BC_F16 || format == BC_I8) && page_size >= 16 && page_size <= 256 && (page_size & (page_size - 1)) == 0 && n_kv_heads >= 1 &&
           n_kv_heads <= kMostKvHeads && (head_dim == 64 || head_dim == 128 || head_dim == 256);
}
uint64_t row_bytes(int32_t format, uint32_t head_dim) { return format == BC_F16 ? 2 * head_dim : head_dim; }
uint64_t page_bytes(int32_t format, uint32_t page_size, uint32_t n_kv_heads, uint32_t head_dim) {
    return (uint64_t)page_size * n_kv_heads * (row_bytes(format, head_dim) + (format == BC_I8 ? 4 : 0));
}

bc_status aligned(const char* op, const char* what, size_t offset, size_t to) {
    if (offset % to != 0) return fail(BC_ERR_ARGUMENT, "the %s launch needs %s at a multiple of %zu bytes, got %zu", op, what, to, offset);
    return BC_OK;
}

// The pool and the rows of a call, checked, as the kernels take them.
bc_status pool_and_rows(bc_backend* b, const bc_kv_pool* pool, const bc_kv_rows* rows, const char* op, k::KvPool* p, k::KvRows* r) {
    if (!pool || !rows) return fail(BC_ERR_ARGUMENT, "the %s launch got no pool or no rows", op);
    if (pool->format != BC_F16 && pool->format != BC_I8) return fail(BC_ERR_UNSUPPORTED, "key/value pages in format %d", pool->format);
    if (!pool_shape(pool->format, pool->page_size, pool->n_kv_heads, pool->head_dim))
        return fail(BC_ERR_ATTENTION_LIMITS,
                    "key/value pages hold a power of two of 16 to 256 positions of 1 to %u heads of 64, 128 or 256 elements, got %u, %u and %u", kMostKvHeads,
                    pool->page_size, pool->n_kv_heads, pool->head_dim);
    if (pool->n_pages == 0 || rows->n_seqs == 0 || rows->n_seqs > kMostSeqs || rows->max_pages == 0 || (uint64_t)rows->max_pages * pool->page_size > 1ull << 31)
        return fail(BC_ERR_ARGUMENT, "the %s launch needs at least one page, 1 to %u sequences and tables of 1 to 2^31 positions, got %u, %u and %u pages", op,
                    kMostSeqs, pool->n_pages, rows->n_seqs, rows->max_pages);
    if (rows->max_queries == 0 || rows->n_rows > 1u << 24) return fail(BC_ERR_ARGUMENT, "the %s launch takes up to 2^24 rows, at least one to a sequence", op);
    const uint64_t page = page_bytes(pool->format, pool->page_size, pool->n_kv_heads, pool->head_dim);
    BC_TRY(check_range(b, pool->k, pool->k_off, pool->n_pages * page, op));
    BC_TRY(check_range(b, pool->v, pool->v_off, pool->n_pages * page, op));
    BC_TRY(aligned(op, "pages", pool->k_off, 16));
    BC_TRY(aligned(op, "pages", pool->v_off, 16));
    BC_TRY(check_range(b, rows->table, rows->table_off, (size_t)rows->n_seqs * rows->max_pages * 4, op));
    BC_TRY(check_range(b, rows->starts, rows->starts_off, ((size_t)rows->n_seqs + 1) * 4, op));
    BC_TRY(check_range(b, rows->lens, rows->lens_off, (size_t)rows->n_seqs * 4, op));
    BC_TRY(aligned(op, "tables", rows->table_off, 4));
    BC_TRY(aligned(op, "starts", rows->starts_off, 4));
    BC_TRY(aligned(op, "lengths", rows->lens_off, 4));
    int* fault = page_fault_word(b);
    if (!fault) return fail(BC_ERR_ALLOCATION, "no host memory for the %s launch's faults", op);
    uint32_t shift = 0;
    while (1u << shift < pool->page_size) ++shift;
    *p = k::KvPool{pool->format, pool->n_pages, shift, pool->n_kv_heads, pool->head_dim, (uint32_t)row_bytes(pool->format, pool->head_dim), page,
                   at<uint8_t>(pool->k, pool->k_off), at<uint8_t>(pool->v, pool->v_off), fault};
    *r = k::KvRows{at<const uint32_t>(rows->table, rows->table_off), at<const uint32_t>(rows->starts, rows->starts_off),
                   at<const uint32_t>(rows->lens, rows->lens_off), rows->n_seqs, rows->n_rows, rows->max_queries, rows->max_pages};
    return BC_OK;
}

// Rows of `width` elements of `element` bytes, `stride` elements apart, that are read or written 16 bytes at a time.
bc_status strided(bc_backend* b, bc_buffer* buffer, size_t offset, uint32_t n_rows, uint32_t width, uint32_t stride, size_t element, const char* op) {
    if (stride < width) return fail(BC_ERR_ARGUMENT, "the %s launch has rows of %u elements %u apart", op, width, stride);
    BC_TRY(aligned(op, "rows", offset, 16));
    BC_TRY(aligned(op, "the distance of rows", stride * element, 16));
    return check_range(b, buffer, offset, n_rows ? ((size_t)(n_rows - 1) * stride + width) * element : 0, op);
}

// Floats from a view on.
struct Floats {
    uintptr_t at;
    uint64_t n;
};
Floats floats_at(bc_buffer* buffer, size_t offset, uint64_t n) { return Floats{reinterpret_cast<uintptr_t>(buffer->ptr) + offset, n}; }
bool overlap(const Floats& a, const Floats& b) { return a.at < b.at + 4 * b.n && b.at < a.at + 4 * a.n; }

// Whether `x` lies over some head of strided rows, whose strides are no less than what they step over: heads ascend, so only the last one that begins before the end of
// `x` can reach into it.
bool over_heads(const Floats& x, uintptr_t first, uint32_t n_rows, uint64_t stride, uint32_t n_heads, uint64_t head_stride, uint32_t head_dim) {
    const uintptr_t end = x.at + 4 * x.n;
    if (end <= first) return false;
    const uint64_t ahead = (end - first - 1) / 4, row = ahead / stride < n_rows ? ahead / stride : n_rows - 1, in_row = (ahead - row * stride) / head_stride;
    const uint64_t head = in_row < n_heads ? in_row : n_heads - 1;
    return first + 4 * (row * stride + head * head_stride + head_dim) > x.at;
}

// Whether [at, at + len) is allocated device memory. The driver, reached through cudaGetDriverEntryPoint, names one allocation or mapping at a time; a range
// may lie over several neighbouring mappings.
bool allocated(uintptr_t at, size_t len) {
    using AddressRange = CUresult (*)(CUdeviceptr*, size_t*, CUdeviceptr);
    static const AddressRange range_of = [] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult found;
        const bool ok = cudaGetDriverEntryPoint("cuMemGetAddressRange", &fn, cudaEnableDefault, &found) == cudaSuccess && found == cudaDriverEntryPointSuccess;
        return ok ? reinterpret_cast<AddressRange>(fn) : nullptr;
    }();
    while (len > 0) {
        CUdeviceptr base = 0;
        size_t size = 0;
        if (!range_of || range_of(&base, &size, (CUdeviceptr)at) != CUDA_SUCCESS || at < base || at - base >= size) return false;
        const size_t here = size - (at - base);
        if (here >= len) return true;
        at += here;
        len -= here;
    }
    return true;
}

}  // namespace

extern "C" {

bc_status bc_buffer_at(bc_backend* b, void* ptr, size_t len, bc_buffer** out) {
    if (!b || !out || (!ptr && len)) return fail(BC_ERR_ARGUMENT, "backend, ptr and out must be non-null");
    if (reinterpret_cast<uintptr_t>(ptr) % 256 != 0) return fail(BC_ERR_ARGUMENT, "a buffer starts at a multiple of 256 bytes");
    BC_TRY(b->activate());
    if (ptr) {
        cudaPointerAttributes attributes;
        cudaError_t e = cudaPointerGetAttributes(&attributes, ptr);
        if (e != cudaSuccess) {
            cudaGetLastError();
            return cuda_fail(e, "cudaPointerGetAttributes", BC_ERR_ARGUMENT);
        }
        if (attributes.type != cudaMemoryTypeDevice || attributes.device != b->device)
            return fail(BC_ERR_ARGUMENT, "the pointer is not memory of device %d", b->device);
        if (!allocated(reinterpret_cast<uintptr_t>(ptr), len)) return fail(BC_ERR_ARGUMENT, "the memory at the pointer ends before %zu bytes", len);
    }
    try {
        std::unique_ptr<bc_buffer> buffer(new bc_buffer());
        buffer->backend = b;
        buffer->ptr = ptr;
        buffer->len = len;
        buffer->owned = false;
        b->buffers.insert(buffer.get());
        *out = buffer.release();
    } catch (const std::bad_alloc&) {
        return fail(BC_ERR_ALLOCATION, "no memory for a buffer handle");
    }
    return BC_OK;
}

size_t bc_kv_pool_bytes(int32_t format, uint32_t n_pages, uint32_t page_size, uint32_t n_kv_heads, uint32_t head_dim) {
    return pool_shape(format, page_size, n_kv_heads, head_dim) ? n_pages * page_bytes(format, page_size, n_kv_heads, head_dim) : 0;
}

bc_status bc_op_kv_write(bc_backend* b, const bc_kv_pool* pool, const bc_kv_rows* rows, bc_buffer* k, size_t k_off, bc_buffer* v, size_t v_off,
                         uint32_t k_stride, uint32_t v_stride) {
    BC_TRY(recording(b));
    k::KvPool p;
    k::KvRows r;
    BC_TRY(pool_and_rows(b, pool, rows, "kv_write", &p, &r));
    const uint32_t width = p.n_kv_heads * p.head_dim;
    BC_TRY(strided(b, k, k_off, r.n_rows, width, k_stride, 4, "kv_write"));
    BC_TRY(strided(b, v, v_off, r.n_rows, width, v_stride, 4, "kv_write"));
    if (r.n_rows == 0) return BC_OK;
    return b->run("kv_write", r.n_rows, width, 0, 1,
                  [&] { return k::kv_write(b->stream, p, r, at<const float>(k, k_off), at<const float>(v, v_off), k_stride, v_stride); });
}

bc_status bc_op_kv_read(bc_backend* b, const bc_kv_pool* pool, const bc_kv_rows* rows, bc_buffer* k, size_t k_off, bc_buffer* v, size_t v_off, int32_t out_half,
                        uint32_t k_stride, uint32_t v_stride) {
    BC_TRY(recording(b));
    k::KvPool p;
    k::KvRows r;
    BC_TRY(pool_and_rows(b, pool, rows, "kv_read", &p, &r));
    const uint32_t width = p.n_kv_heads * p.head_dim;
    if (!k && !v) return fail(BC_ERR_ARGUMENT, "the kv_read launch got neither keys nor values to fill");
    if (k) BC_TRY(strided(b, k, k_off, r.n_rows, width, k_stride, out_half ? 2 : 4, "kv_read"));
    if (v) BC_TRY(strided(b, v, v_off, r.n_rows, width, v_stride, out_half ? 2 : 4, "kv_read"));
    if (r.n_rows == 0) return BC_OK;
    return b->run("kv_read", r.n_rows, width, 0, 1,
                  [&] { return k::kv_read(b->stream, p, r, at<void>(k, k_off), at<void>(v, v_off), out_half != 0, k_stride, v_stride); });
}

size_t bc_attention_paged_scratch_floats(uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim) {
    return (size_t)k::attention_paged_scratch_floats(n_heads, n_kv_heads, head_dim);
}

bc_status bc_op_attention_paged(bc_backend* b, const bc_kv_pool* pool, const bc_kv_rows* rows, bc_buffer* q, size_t q_off, bc_buffer* scratch, size_t s_off,
                                bc_buffer* out, size_t out_off, uint32_t n_heads, uint32_t q_stride, uint32_t q_head_stride) {
    BC_TRY(recording(b));
    k::KvPool p;
    k::KvRows r;
    BC_TRY(pool_and_rows(b, pool, rows, "attention_paged", &p, &r));
    if (n_heads == 0 || n_heads % p.n_kv_heads != 0 || n_heads / p.n_kv_heads > 8)
        return fail(BC_ERR_ATTENTION_LIMITS, "attention_paged needs 1 to 8 query heads per KV head, got %u/%u heads", n_heads, p.n_kv_heads);
    if (q_head_stride < p.head_dim || q_head_stride % 4 != 0)
        return fail(BC_ERR_ARGUMENT, "the attention_paged launch has heads of %u elements %u apart (a multiple of 4)", p.head_dim, q_head_stride);
    const uint64_t width = (uint64_t)(n_heads - 1) * q_head_stride + p.head_dim;
    if (width > 0xffffffffull) return fail(BC_ERR_ARGUMENT, "the attention_paged launch has rows of %llu elements", (unsigned long long)width);
    BC_TRY(strided(b, q, q_off, r.n_rows, (uint32_t)width, q_stride, 4, "attention_paged"));
    BC_TRY(strided(b, out, out_off, r.n_rows, n_heads * p.head_dim, n_heads * p.head_dim, 4, "attention_paged"));
    BC_TRY(aligned("attention_paged", "scratch", s_off, 16));
    BC_TRY(check_range(b, scratch, s_off, bc_attention_paged_scratch_floats(n_heads, p.n_kv_heads, p.head_dim) * 4, "attention_paged"));
    if (r.n_rows == 0) return BC_OK;
    const Floats outs = floats_at(out, out_off, (uint64_t)r.n_rows * n_heads * p.head_dim),
                 parts = floats_at(scratch, s_off, bc_attention_paged_scratch_floats(n_heads, p.n_kv_heads, p.head_dim));
    const uintptr_t queries = reinterpret_cast<uintptr_t>(at<const float>(q, q_off));
    if (overlap(outs, parts) || over_heads(outs, queries, r.n_rows, q_stride, n_heads, q_head_stride, p.head_dim) ||
        over_heads(parts, queries, r.n_rows, q_stride, n_heads, q_head_stride, p.head_dim))
        return fail(BC_ERR_ARGUMENT, "the attention_paged launch has queries, scratch and results that overlap");
    return b->run("attention_paged", r.n_rows, r.n_seqs, 0, k::attention_paged_launches(p, r, n_heads), [&] {
        return k::attention_paged(b->stream, p, r, at<const float>(q, q_off), q_stride, q_head_stride, at<float>(scratch, s_off), at<float>(out, out_off), n_heads);
    });
}

}  // extern "C"
