// One-token attention over rows of the query's type (paged_core.cuh has the rest): about one
// multiplication a byte, so bound by memory.
#include "packed.cuh"
#include "paged_core.cuh"

namespace mr {
namespace cache {
namespace {

// The two ways to work on a step.  Each keeps, per warp, kHeads running maxima
// and sums and weighted values; lanes hold them as the comments say.

// 16-bit types, on the tensor cores: S^T = K Q^T and O^T += V^T P^T with rows (keys,
// then dims) as the 16-high side and up to 8 query heads as the 8-wide side, so that a
// group of 1 to 8 heads costs the same: 2 DP / 16 x 3 small products for 16 rows of
// 2 KB (DP 128), well below what mma.sync can do in the time the rows take to arrive.
// (tcgen05 would want 128 query rows; there are at most 8.)
template <typename T, int DP_>
struct Math16 : Heads8<T, DP_ / 16> {
    using Heads8<T, DP_ / 16>::o;
    using Heads8<T, DP_ / 16>::m;
    using Heads8<T, DP_ / 16>::l;
    static constexpr bool kAgain = true, kRuns = false;
    static int ctas(int64_t, int, bool) { return kCtas; }
    static constexpr int kCtas = 2, DP = DP_, kHeads = 8, STEP = DP == 128 ? 16 : 32, STAGES = DP == 32 ? 6 : 3;
    using R = Ring<T, DP, STEP, STAGES>;
    uint32_t qf[DP / 16][2];   // Q^T fragments: head lane / 4

    __device__ __forceinline__ void begin(const PagedArgs &a, const char *q, int heads) {
        const int lane = threadIdx.x % 32, h = lane / 4;
#pragma unroll
        for (int b = 0; b < DP / 16; ++b) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int j = b * 16 + e * 8 + 2 * (lane % 4);
                qf[b][e] = h < heads && j < a.dim ? __ldg(reinterpret_cast<const uint32_t *>(q + h * a.q_head + j * 2)) : 0u;
            }
        }
        this->clear();
    }

    // One step: `rows` rows in `stage` (keys, then values), bit r of `live`: row r is seen.
    __device__ __forceinline__ void step(const PagedArgs &a, uint32_t stage, uint32_t live, int rows, float *scores) {
        const int lane = threadIdx.x % 32;
        constexpr int S = STEP / 16;
        float s[S][4];
#pragma unroll
        for (int x = 0; x < S; ++x) {
            s[x][0] = s[x][1] = s[x][2] = s[x][3] = 0.f;
#pragma unroll
            for (int b = 0; b < DP / 16; ++b) {
                uint32_t k[4];
                ldmatrix(k, stage + R::offset(x * 16 + lane % 16, b * 2 + lane / 16));
                mma16(s[x], k, qf[b][0], qf[b][1], T());
            }
        }
        float ref[2];
        this->template settle<false>(a, s, a.scale, a.scale, live, rows, scores, ref);
#pragma unroll
        for (int x = 0; x < S; ++x) {
            uint32_t b0, b1, c0, c1;
            this->weigh(s[x], ref, b0, b1, c0, c1);
#pragma unroll
            for (int b = 0; b < DP / 16; ++b) {
                uint32_t v[4];
                ldmatrix_t(v, stage + STEP * R::kRowBytes +
                                  R::offset(x * 16 + lane % 8 + (lane / 16) * 8, b * 2 + ((lane / 8) & 1)));
                mma16(o[b], v, b0, b1, T());
                mma16(o[b], v, c0, c1, T());
            }
        }
    }

    // Every pair of values of consecutive dims of a head, times its head's factor:
    // put(head, dim, x, y).  Lanes whose rows are neighbours swap one of their two heads.
    template <typename Put>
    __device__ __forceinline__ void each(float f0, float f1, const Put &put) const {
        const int lane = threadIdx.x % 32, h = 2 * (lane % 4);
        const bool odd = lane & 4;
#pragma unroll
        for (int b = 0; b < DP / 16; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float x = o[b][2 * e] * f0, y = o[b][2 * e + 1] * f1;
                const float z = __shfl_xor_sync(0xffffffffu, odd ? x : y, 4);
                const int dim = b * 16 + e * 8 + (lane / 4 & ~1);
                put(odd ? h + 1 : h, dim, odd ? z : x, odd ? y : z);
            }
    }
    __device__ __forceinline__ void put_out(const PagedArgs &a, char *out, int heads) const {
        each(l[0] != 0.f ? 1.f / l[0] : 0.f, l[1] != 0.f ? 1.f / l[1] : 0.f, [&](int h, int dim, float x, float y) {
            if (h < heads && dim < a.dim) *reinterpret_cast<uint32_t *>(out + h * a.o_head + dim * 2) = pack2(x, y, T());
        });
    }
    // values [head][DP], and the maxima and sums `stride` apart
    __device__ __forceinline__ void put_partial(float *to, float2 *sums, int64_t stride, int heads) const {
        const int lane = threadIdx.x % 32;
        each(1.f, 1.f, [&](int h, int dim, float x, float y) {
            if (h < heads) *reinterpret_cast<float2 *>(to + h * DP + dim) = make_float2(x, y);
        });
        if (lane < 4)
#pragma unroll
            for (int e = 0; e < 2; ++e) sums[(2 * lane + e) * stride] = make_float2(m[e], l[e]);
    }
};

// float32 on the CUDA cores: DP / 4 lanes share a row, four values each, and keep the
// same four dims of up to 4 query heads and of their weighted values in registers; the
// 8 rows x 4 heads of a step give 32 sums, folded so that each lane ends with one.
template <int DP_>
struct Math32 {
    static constexpr bool kAgain = true, kRuns = false;
    static int ctas(int64_t, int, bool) { return kCtas; }
    static constexpr int kCtas = 2, DP = DP_, kHeads = 4, STEP = 8, STAGES = DP == 128 ? 3 : DP == 64 ? 6 : 8;
    static constexpr int kLanes = DP / 4, kRows = 32 / kLanes, kEach = STEP / kRows;  // lanes a row, rows at a time
    using R = Ring<float, DP, STEP, STAGES>;
    float4 q[4], o[4];
    float m, l;  // head lane % 4; l only of this lane's rows

    __device__ __forceinline__ void begin(const PagedArgs &a, const char *src, int heads) {
        const int j = 4 * (threadIdx.x % kLanes);
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            q[h] = h < heads && j < a.dim ? __ldg(reinterpret_cast<const float4 *>(src + h * a.q_head + j * 4)) : float4{};
            o[h] = float4{};
        }
        m = -INFINITY;
        l = 0.f;
    }
    __device__ __forceinline__ float4 piece(uint32_t stage, int row) const {
        float4 x;
        asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];"
                     : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
                     : "r"(stage + R::offset(row, threadIdx.x % kLanes)));
        return x;
    }
    // Row r of the step belongs to lanes r / kEach * kLanes ..; after the fold lane i of
    // those has row r = (its part) * kEach + i / 4 and head i % 4.
    __device__ __forceinline__ void step(const PagedArgs &a, uint32_t stage, uint32_t live, int rows, float *scores) {
        const int lane = threadIdx.x % 32, part = lane / kLanes, i = lane % kLanes;
        float s[kLanes];  // [row][head]
#pragma unroll
        for (int r = 0; r < kEach; ++r) {
            const float4 k = piece(stage, part * kEach + r);
#pragma unroll
            for (int h = 0; h < 4; ++h)
                s[r * 4 + h] = fmaf(q[h].x, k.x, fmaf(q[h].y, k.y, fmaf(q[h].z, k.z, q[h].w * k.w)));
        }
#pragma unroll
        for (int w = kLanes / 2; w > 0; w >>= 1) {
            const bool upper = i & w;
#pragma unroll
            for (int e = 0; e < w; ++e) {
                const float keep = upper ? s[e + w] : s[e], give = upper ? s[e] : s[e + w];
                s[e] = keep + __shfl_xor_sync(0xffffffffu, give, w);
            }
        }
        const int row = part * kEach + i / 4, head = i % 4;
        const float x = (live >> row) & 1u ? s[0] * a.scale : -INFINITY;
        if (scores && head < a.heads2 && row < rows) scores[row * a.heads2 + head] = x;
        float top = x;
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
        top = fmaxf(top, m);
        const float ref = top == -INFINITY ? 0.f : top;
        if (__any_sync(0xffffffffu, top > m)) {
            const float c = ex2(m - ref);
            l *= c;
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                const float ch = __shfl_sync(0xffffffffu, c, h);
                o[h].x *= ch;
                o[h].y *= ch;
                o[h].z *= ch;
                o[h].w *= ch;
            }
            m = top;
        }
        const float p = ex2(x - ref);
        l += p;
#pragma unroll
        for (int r = 0; r < kEach; ++r) {
            const float4 v = piece(stage + STEP * R::kRowBytes, part * kEach + r);
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                const float w = __shfl_sync(0xffffffffu, p, r * 4 + h, kLanes);
                o[h].x = fmaf(w, v.x, o[h].x);
                o[h].y = fmaf(w, v.y, o[h].y);
                o[h].z = fmaf(w, v.z, o[h].z);
                o[h].w = fmaf(w, v.w, o[h].w);
            }
        }
    }
    __device__ __forceinline__ bool finish() {
#pragma unroll
        for (int h = 0; h < 4; ++h)
#pragma unroll
            for (int w = kLanes; w < 32; w <<= 1) {
                o[h].x += __shfl_xor_sync(0xffffffffu, o[h].x, w);
                o[h].y += __shfl_xor_sync(0xffffffffu, o[h].y, w);
                o[h].z += __shfl_xor_sync(0xffffffffu, o[h].z, w);
                o[h].w += __shfl_xor_sync(0xffffffffu, o[h].w, w);
            }
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
        return true;
    }
    __device__ __forceinline__ void put_out(const PagedArgs &a, char *out, int heads) const {
        const int j = 4 * (threadIdx.x % 32);
        const float f = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            const float fh = __shfl_sync(0xffffffffu, f, h);
            if (h < heads && j < min(DP, a.dim))
                *reinterpret_cast<float4 *>(out + h * a.o_head + j * 4) =
                    make_float4(o[h].x * fh, o[h].y * fh, o[h].z * fh, o[h].w * fh);
        }
    }
    __device__ __forceinline__ void put_partial(float *to, float2 *sums, int64_t stride, int heads) const {
        const int lane = threadIdx.x % 32;
#pragma unroll
        for (int h = 0; h < 4; ++h)
            if (h < heads && lane < kLanes) *reinterpret_cast<float4 *>(to + h * DP + 4 * lane) = o[h];
        if (lane < 4) sums[lane * stride] = make_float2(m, l);
    }
    __device__ __forceinline__ void put_lse(float *lse) const {
        if (threadIdx.x % 32 < 4) lse[threadIdx.x % 32] = log_sum(m, l);
    }
};

template <typename T>
int launch16(mr_context *ctx, PagedArgs &a) {
    return a.dim <= 32   ? launch<T, Math16<T, 32>>(ctx, a)
           : a.dim <= 64 ? launch<T, Math16<T, 64>>(ctx, a)
                         : launch<T, Math16<T, 128>>(ctx, a);
}
int launch32(mr_context *ctx, PagedArgs &a) {
    return a.dim <= 32   ? launch<float, Math32<32>>(ctx, a)
           : a.dim <= 64 ? launch<float, Math32<64>>(ctx, a)
                         : launch<float, Math32<128>>(ctx, a);
}

}  // namespace
}  // namespace cache
}  // namespace mr

using namespace mr::cache;

extern "C" int mr_paged_attention(mr_context *ctx, const mr_array *query, const mr_array *key_pages,
                                  const mr_array *value_pages, const mr_array *page_table, const mr_array *lengths,
                                  const mr_array *weights, const mr_array *out, int window, int sinks, float scale) {
    MR_CHECK(check_array(query, "query", 3, true, false));
    MR_CHECK(check_array(out, "out", 3, true, true));
    const bool packed = key_pages && key_pages->dtype == MR_DTYPE_U8;
    if (packed) {
        MR_CHECK(check_packed(key_pages, value_pages, "key_pages", "value_pages", false));
        MR_REQUIRE(is_float(query->dtype) && out->dtype == query->dtype, "query and out must be of one floating type");
    } else {
        MR_CHECK(check_pools(key_pages, value_pages, "key_pages", "value_pages", false));
        MR_REQUIRE(query->dtype == key_pages->dtype && out->dtype == key_pages->dtype,
                   "query, out and the pages must be of one type");
    }
    const int64_t dim = packed ? packed_dim(key_pages->shape[3]) : key_pages->shape[3];
    for (int i = 0; i < 3; ++i) MR_REQUIRE(query->shape[i] == out->shape[i], "query and out differ in shape");
    MR_CHECK(check_apart(query, "query", out, "out"));
    const int64_t batch = query->shape[0], heads = query->shape[1], kv_heads = key_pages->shape[2];
    MR_REQUIRE(query->shape[2] == dim, "query has %lld values a head, the pages %lld",
               static_cast<long long>(query->shape[2]), static_cast<long long>(dim));
    MR_REQUIRE(heads > 0 && heads % kv_heads == 0, "the %lld query heads must be a multiple of the pages' %lld heads",
               static_cast<long long>(heads), static_cast<long long>(kv_heads));
    MR_CHECK(check_ints(lengths, "lengths", 1));
    MR_REQUIRE(lengths->shape[0] == batch, "lengths must have %lld values", static_cast<long long>(batch));
    MR_CHECK(check_table(page_table, "page_table", batch, key_pages->shape[1]));
    MR_REQUIRE(batch * heads <= INT32_MAX / 2 && heads * query->shape[2] <= INT32_MAX, "too many heads");
    MR_REQUIRE(window >= 0 && sinks >= 0, "window and sinks must not be negative");
    MR_REQUIRE(std::isfinite(scale), "scale must be finite");
    const int64_t capacity = page_table->shape[1] * key_pages->shape[1];
    for (const mr_array *pool : {key_pages, value_pages})
        for (int i = 0; i < 2; ++i)
            MR_REQUIRE(pool->stride[i] < (int64_t(1) << 32) / dtype_bytes(pool->dtype),
                       "the pages' stride %d passes 4 GB", i);
    if (weights) MR_CHECK(check_weights(weights, "weights", batch, kv_heads, capacity, true));
    MR_REQUIRE(ctx, "ctx is NULL");
    MR_CHECK(mr::check_waits(ctx));
    if (!batch) return MR_OK;
    DeviceGuard guard(ctx->device);
    const int64_t size = dtype_bytes(query->dtype), page_size = dtype_bytes(key_pages->dtype);
    PagedArgs a;
    a.q = static_cast<const char *>(query->data);
    a.k = static_cast<const char *>(key_pages->data);
    a.v = static_cast<const char *>(value_pages->data);
    a.out = static_cast<char *>(out->data);
    a.q_batch = query->stride[0] * size;
    a.q_head = query->stride[1] * size;
    a.o_batch = out->stride[0] * size;
    a.o_head = out->stride[1] * size;
    a.k_page = static_cast<uint32_t>(key_pages->stride[0] * page_size);
    a.k_row = static_cast<uint32_t>(key_pages->stride[1] * page_size);
    a.k_head = key_pages->stride[2] * page_size;
    a.v_page = static_cast<uint32_t>(value_pages->stride[0] * page_size);
    a.v_row = static_cast<uint32_t>(value_pages->stride[1] * page_size);
    a.v_head = value_pages->stride[2] * page_size;
    a.pages = make_pages(key_pages, page_table);
    a.lengths = static_cast<const int *>(lengths->data);
    a.length_stride = lengths->stride[0];
    a.weights = weights ? static_cast<float *>(weights->data) : nullptr;
    a.w_batch = weights ? weights->stride[0] : 0;
    a.w_head = weights ? weights->stride[1] : 0;
    a.batch = static_cast<int>(batch);
    a.kv_heads = static_cast<int>(kv_heads);
    a.group = static_cast<int>(heads / kv_heads);
    a.dim = static_cast<int>(query->shape[2]);
    a.capacity = static_cast<int>(capacity);
    a.window = window;
    a.sinks = sinks;
    a.scale = scale * kLog2e;
    if (packed) return launch_packed(ctx, a, query->dtype);
    return query->dtype == MR_DTYPE_F32   ? launch32(ctx, a)
           : query->dtype == MR_DTYPE_F16 ? launch16<__half>(ctx, a)
                                          : launch16<__nv_bfloat16>(ctx, a);
}
