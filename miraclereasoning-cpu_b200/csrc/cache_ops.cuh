// What the paged cache's operators share (cache_pages.cu, paged_attention.cu,
// window_attention.cu): checks of caller-described arrays, scratch memory, the
// device guard, and row addressing through a page table.
#pragma once

#include <algorithm>
#include <atomic>

#include "common.cuh"

namespace mr {
namespace cache {

constexpr int kMaxDim = 128;

inline int dtype_bytes(int dtype) {
    return dtype == MR_DTYPE_F16 || dtype == MR_DTYPE_BF16 ? 2 : dtype == MR_DTYPE_U8 ? 1 : 4;
}
inline bool is_float(int dtype) { return dtype == MR_DTYPE_F32 || dtype == MR_DTYPE_F16 || dtype == MR_DTYPE_BF16; }

// One array argument: its shape, type and strides are usable by the kernels.
// rows: the last dimension is read in 16-byte pieces.  Sets the error and
// returns its code, or MR_OK.
inline int check_array(const mr_array *a, const char *name, int ndim, bool rows, bool written) {
    MR_REQUIRE(a, "%s is missing", name);
    MR_REQUIRE(a->ndim == ndim, "%s must have %d dimensions, not %d", name, ndim, a->ndim);
    MR_REQUIRE(a->dtype >= MR_DTYPE_F32 && a->dtype <= MR_DTYPE_U8, "%s has an unknown type", name);
    const int64_t size = dtype_bytes(a->dtype), most = int64_t(1) << 46;
    bool empty = false;
    for (int i = 0; i < ndim; ++i) {
        MR_REQUIRE(a->shape[i] >= 0 && a->shape[i] <= INT32_MAX, "%s: dimension %d is out of range", name, i);
        MR_REQUIRE(a->stride[i] >= 0 && a->stride[i] <= most / std::max<int64_t>(a->shape[i], 1),
                   "%s: stride %d is out of range", name, i);
        empty = empty || a->shape[i] == 0;
    }
    if (empty) return MR_OK;
    MR_REQUIRE(a->data, "%s has no memory", name);
    MR_REQUIRE(ndim == 1 || a->shape[ndim - 1] == 1 || a->stride[ndim - 1] == 1, "%s: the last dimension must be contiguous", name);
    const uintptr_t unit = rows ? 16 : static_cast<uintptr_t>(size);
    MR_REQUIRE(reinterpret_cast<uintptr_t>(a->data) % unit == 0, "%s must start on a %d-byte boundary", name,
               static_cast<int>(unit));
    if (rows) {
        MR_REQUIRE(a->shape[ndim - 1] * size % 16 == 0 && a->shape[ndim - 1] <= kMaxDim,
                   "%s: rows must be whole 16-byte pieces of at most %d values, not %lld values", name, kMaxDim,
                   static_cast<long long>(a->shape[ndim - 1]));
        for (int i = 0; i + 1 < ndim; ++i)
            MR_REQUIRE(a->shape[i] == 1 || a->stride[i] * size % 16 == 0, "%s: stride %d is not a multiple of 16 bytes",
                       name, i);
    }
    if (written) {  // no two elements at one address: in rising order each stride spans the dimensions below it
        int order[4] = {0, 1, 2, 3};
        std::sort(order, order + ndim, [&](int x, int y) { return a->stride[x] < a->stride[y]; });
        int64_t span = 1;
        for (int k = 0; k < ndim; ++k) {
            const int i = order[k];
            if (a->shape[i] == 1) continue;
            MR_REQUIRE(a->stride[i] >= span, "%s is written and must not overlap itself", name);
            span = a->stride[i] * (a->shape[i] - 1) + span;
        }
    }
    return MR_OK;
}

#define MR_CHECK(call)              \
    do {                            \
        const int _rc = (call);     \
        if (_rc) return _rc;        \
    } while (0)

inline int check_ints(const mr_array *a, const char *name, int ndim, bool written = false) {
    MR_CHECK(check_array(a, name, ndim, false, written));
    MR_REQUIRE(a->dtype == MR_DTYPE_I32, "%s must be int32", name);
    return MR_OK;
}

inline int check_weights(const mr_array *a, const char *name, int64_t batch, int64_t kv_heads, int64_t rows,
                         bool written) {
    MR_CHECK(check_array(a, name, 3, false, written));
    MR_REQUIRE(a->dtype == MR_DTYPE_F32, "%s must be float32", name);
    MR_REQUIRE(a->shape[0] == batch && a->shape[1] == kv_heads && a->shape[2] == rows,
               "%s must be [%lld, %lld, %lld] (batch, kv heads, the table's rows)", name,
               static_cast<long long>(batch), static_cast<long long>(kv_heads), static_cast<long long>(rows));
    return MR_OK;
}

// A key and a value pool of one shape and type.
inline int check_pools(const mr_array *k, const mr_array *v, const char *kn, const char *vn, bool written) {
    MR_CHECK(check_array(k, kn, 4, true, written));
    MR_CHECK(check_array(v, vn, 4, true, written));
    MR_REQUIRE(is_float(k->dtype) && k->dtype == v->dtype, "%s and %s must be of one floating type", kn, vn);
    for (int i = 0; i < 4; ++i) MR_REQUIRE(k->shape[i] == v->shape[i], "%s and %s differ in shape", kn, vn);
    MR_REQUIRE(k->shape[1] > 0 && k->shape[2] > 0 && k->shape[3] > 0, "%s: an empty page row", kn);
    return MR_OK;
}

// A page table over pools of `page` rows: int32 [batch, table pages], its rows countable in 31 bits.
inline int check_table(const mr_array *table, const char *name, int64_t batch, int64_t page) {
    MR_CHECK(check_ints(table, name, 2));
    MR_REQUIRE(table->shape[0] == batch, "%s must have a row for each of the %lld sequences", name,
               static_cast<long long>(batch));
    MR_REQUIRE(table->shape[1] * page < INT32_MAX / 2, "%s spans too many rows", name);
    return MR_OK;
}

// Two arguments that a call reads and writes in no fixed order.
inline int check_apart(const mr_array *a, const char *an, const mr_array *b, const char *bn) {
    MR_REQUIRE(a->data != b->data || !a->data, "%s and %s must not share memory", an, bn);
    return MR_OK;
}

// Makes the context's device current for a call and puts the caller's back.
struct DeviceGuard {
    int before = -1;
    explicit DeviceGuard(int device) {
        cudaGetDevice(&before);
        if (before != device) cudaSetDevice(device);
        else before = -1;
    }
    ~DeviceGuard() {
        if (before >= 0) cudaSetDevice(before);
    }
};

// Scratch of one call.  Outside a capture it is the context's own block, grown
// on demand: calls on one context are in stream order, so each call's kernels
// are done with it before the next call's start.  Inside a capture the block is
// allocated and freed by nodes of the graph itself, so that two graphs, or a
// graph and eager calls, never share one.
struct Scratch {
    mr_context *ctx;
    void *data = nullptr;
    bool captured = false;
    explicit Scratch(mr_context *c) : ctx(c) {}
    int take(size_t bytes) {
        if (!bytes) return MR_OK;
        cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
        MR_CUDA_TRY(cudaStreamIsCapturing(ctx->stream, &status));
        if (status != cudaStreamCaptureStatusNone) {
            MR_CUDA_TRY(cudaMallocAsync(&data, bytes, ctx->stream));
            captured = true;
            return MR_OK;
        }
        if (ctx->scratch_bytes < bytes) {
            const size_t want = std::max(bytes + bytes / 4, size_t(4) << 20);
            if (ctx->scratch) MR_CUDA_TRY(cudaFreeAsync(ctx->scratch, ctx->stream));
            ctx->scratch = nullptr;
            ctx->scratch_bytes = 0;
            MR_CUDA_TRY(cudaMallocAsync(&ctx->scratch, want, ctx->stream));
            ctx->scratch_bytes = want;
        }
        data = ctx->scratch;
        return MR_OK;
    }
    ~Scratch() {
        if (captured) cudaFreeAsync(data, ctx->stream);
    }
};

// Lets a kernel take more than 48 KB of shared memory; asked of the driver once a device
// (`done`: a bit each, of the kernel's own).
inline int allow_shared(int device, const void *kernel, int bytes, std::atomic<uint64_t> &done) {
    const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
    if (done.load(std::memory_order_relaxed) & bit) return MR_OK;
    MR_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.fetch_or(bit, std::memory_order_relaxed);
    return MR_OK;
}

// Launches a kernel that may start while the one before it runs (programmatic dependent
// launch) and waits for that one's end itself (griddepcontrol.wait).
template <typename Args>
int launch_early(mr_context *ctx, dim3 grid, dim3 threads, void (*kernel)(Args), const Args &args) {
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = threads;
    config.stream = ctx->stream;
    config.attrs = &early;
    config.numAttrs = 1;
    MR_CUDA_TRY(cudaLaunchKernelEx(&config, kernel, args));
    return MR_OK;
}

// ---- device side ------------------------------------------------------------------
// t / d and t % d for 0 <= t < 2^31 by a multiplication: floor(t m / 2^63) with
// m = floor(2^63 / d) + 1 is exact, since t (m d - 2^63) <= t d < 2^63.
struct Divider {
    uint64_t m;
    int d;
    Divider() = default;
    explicit Divider(int divisor) : m((uint64_t(1) << 63) / static_cast<uint64_t>(divisor) + 1), d(divisor) {}
    __device__ __forceinline__ int div(int t) const {
        return static_cast<int>(__umul64hi(static_cast<uint64_t>(t) * 2, m));
    }
};

// Rows of a pool through the page tables; offsets and strides in bytes.
struct Pages {
    const int *table;
    int64_t table_stride;
    int table_pages, pages;
    Divider page;
    // Byte offset of row t of sequence s without its head, given the pool's page
    // and row strides; -1 where the table has no valid page for it.
    __device__ __forceinline__ int64_t row(int s, int t, int64_t page_stride, int64_t row_stride) const {
        const int p = page.div(t);
        if (p >= table_pages) return -1;
        const int id = __ldg(table + s * table_stride + p);
        if (static_cast<unsigned>(id) >= static_cast<unsigned>(pages)) return -1;
        return id * page_stride + (t - p * page.d) * row_stride;
    }
};

inline Pages make_pages(const mr_array *pool, const mr_array *table) {
    Pages p;
    p.table = static_cast<const int *>(table->data);
    p.table_stride = table->stride[0];
    p.table_pages = static_cast<int>(table->shape[1]);
    p.pages = static_cast<int>(pool->shape[0]);
    p.page = Divider(static_cast<int>(pool->shape[1]));
    return p;
}

// The rows of a sequence: its length cut to what its table can hold.
__device__ __forceinline__ int sequence_rows(const int *lengths, int64_t stride, int s, int capacity) {
    return max(0, min(__ldg(lengths + s * stride), capacity));
}

__device__ __forceinline__ float widen(const float *p) { return *p; }
__device__ __forceinline__ float widen(const __half *p) { return __half2float(*p); }
__device__ __forceinline__ float widen(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ void narrow(float v, float *p) { *p = v; }
__device__ __forceinline__ void narrow(float v, __half *p) { *p = __float2half_rn(v); }
__device__ __forceinline__ void narrow(float v, __nv_bfloat16 *p) { *p = __float2bfloat16_rn(v); }

}  // namespace cache
}  // namespace mr
