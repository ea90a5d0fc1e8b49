// Attention of packed prompts: causal, optionally in a sliding window with a few
// first rows that stay visible.
//
//   p = m - n + i   (query i of a sequence of n queries and m keys)
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j  over the j that query i sees:
//           j <= p and (no window, or p - j < window, or j < sinks).
#include <cmath>

#include "cache_ops.cuh"

namespace mr {
namespace cache {
namespace {

struct WindowArgs {
    const char *q, *k, *v;
    char *out;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;  // bytes
    const int *q_offsets, *k_offsets;
    int64_t qo_stride, ko_stride;
    int tokens, rows, batch, heads, kv_heads, group, dim, window, sinks;
    float scale;
};

// Where sequence s lies, cut to the arrays: first query, queries, first key, keys.
struct Span {
    int q0, n, k0, m;
};
__device__ __forceinline__ Span span_of(const WindowArgs &a, int s) {
    Span x;
    x.q0 = max(0, min(__ldg(a.q_offsets + s * a.qo_stride), a.tokens));
    x.n = max(0, min(__ldg(a.q_offsets + (s + 1) * a.qo_stride), a.tokens) - x.q0);
    x.k0 = max(0, min(__ldg(a.k_offsets + s * a.ko_stride), a.rows));
    x.m = max(0, min(__ldg(a.k_offsets + (s + 1) * a.ko_stride), a.rows) - x.k0);
    return x;
}

// A warp per (query row, head), four values of a row a lane.
template <typename T>
__global__ void __launch_bounds__(128) k_rows(WindowArgs a) {
    const int64_t id = blockIdx.x * static_cast<int64_t>(4) + threadIdx.x / 32;
    const int lane = threadIdx.x % 32, i = static_cast<int>(id / a.heads), h = static_cast<int>(id % a.heads);
    if (i >= a.tokens) return;
    int s = 0;
    Span x = {};
    for (; s < a.batch; ++s) {
        x = span_of(a, s);
        if (i >= x.q0 && i < x.q0 + x.n) break;
    }
    if (s == a.batch) return;
    auto load = [&](const char *row, float (&y)[4]) {
        for (int j = 0; j < 4; ++j)
            y[j] = 4 * lane + j < a.dim ? widen(reinterpret_cast<const T *>(row) + 4 * lane + j) : 0.f;
    };
    const int p = x.m - x.n + i - x.q0, kh = h / a.group;
    float q[4], o[4] = {}, m = -INFINITY, l = 0.f;
    load(a.q + i * a.q_row + h * a.q_head, q);
    for (int j = 0; j <= p; ++j) {
        if (a.window && p - j >= a.window && j >= a.sinks) {
            j = p - a.window;
            continue;
        }
        float k[4], v[4];
        load(a.k + (x.k0 + j) * a.k_row + kh * a.k_head, k);
        load(a.v + (x.k0 + j) * a.v_row + kh * a.v_head, v);
        const float y = warp_sum(q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3]) * a.scale;
        const float m_new = fmaxf(m, y), c = expf(m - m_new), w = expf(y - m_new);
        l = l * c + w;
        for (int e = 0; e < 4; ++e) o[e] = o[e] * c + w * v[e];
        m = m_new;
    }
    T *out = reinterpret_cast<T *>(a.out + i * a.o_row + h * a.o_head);
    for (int j = 0; j < 4; ++j)
        if (4 * lane + j < a.dim) narrow(l > 0.f ? o[j] / l : 0.f, out + 4 * lane + j);
}

}  // namespace
}  // namespace cache
}  // namespace mr

using namespace mr::cache;

extern "C" int mr_window_attention(mr_context *ctx, const mr_array *query, const mr_array *keys, const mr_array *values,
                                   const mr_array *query_offsets, const mr_array *key_offsets, const mr_array *out,
                                   int window, int sinks, float scale) {
    MR_CHECK(check_array(query, "query", 3, true, false));
    MR_CHECK(check_array(keys, "keys", 3, true, false));
    MR_CHECK(check_array(values, "values", 3, true, false));
    MR_CHECK(check_array(out, "out", 3, true, true));
    MR_REQUIRE(query->dtype != MR_DTYPE_I32 && keys->dtype == query->dtype && values->dtype == query->dtype &&
                   out->dtype == query->dtype,
               "query, keys, values and out must be of one floating type");
    for (int i = 0; i < 3; ++i) {
        MR_REQUIRE(query->shape[i] == out->shape[i], "query and out differ in shape");
        MR_REQUIRE(keys->shape[i] == values->shape[i], "keys and values differ in shape");
    }
    MR_CHECK(check_apart(query, "query", out, "out"));
    const int64_t heads = query->shape[1], kv_heads = keys->shape[1];
    MR_REQUIRE(query->shape[2] == keys->shape[2] && query->shape[2] > 0, "query has %lld values a head, keys %lld",
               static_cast<long long>(query->shape[2]), static_cast<long long>(keys->shape[2]));
    MR_REQUIRE(kv_heads > 0 && heads > 0 && heads % kv_heads == 0,
               "the %lld query heads must be a multiple of the %lld key heads", static_cast<long long>(heads),
               static_cast<long long>(kv_heads));
    MR_CHECK(check_ints(query_offsets, "query_offsets", 1));
    MR_CHECK(check_ints(key_offsets, "key_offsets", 1));
    MR_REQUIRE(query_offsets->shape[0] > 0 && query_offsets->shape[0] == key_offsets->shape[0],
               "query_offsets and key_offsets must have one value more than there are sequences");
    MR_REQUIRE(query->shape[0] < INT32_MAX / 2 && keys->shape[0] < INT32_MAX / 2, "too many rows");
    MR_REQUIRE(window >= 0 && sinks >= 0, "window and sinks must not be negative");
    MR_REQUIRE(std::isfinite(scale), "scale must be finite");
    MR_REQUIRE(ctx, "ctx is NULL");
    if (!query->shape[0] || query_offsets->shape[0] == 1) return MR_OK;
    DeviceGuard guard(ctx->device);
    const int64_t size = dtype_bytes(query->dtype);
    WindowArgs a;
    a.q = static_cast<const char *>(query->data);
    a.k = static_cast<const char *>(keys->data);
    a.v = static_cast<const char *>(values->data);
    a.out = static_cast<char *>(out->data);
    a.q_row = query->stride[0] * size;
    a.q_head = query->stride[1] * size;
    a.k_row = keys->stride[0] * size;
    a.k_head = keys->stride[1] * size;
    a.v_row = values->stride[0] * size;
    a.v_head = values->stride[1] * size;
    a.o_row = out->stride[0] * size;
    a.o_head = out->stride[1] * size;
    a.q_offsets = static_cast<const int *>(query_offsets->data);
    a.k_offsets = static_cast<const int *>(key_offsets->data);
    a.qo_stride = query_offsets->stride[0];
    a.ko_stride = key_offsets->stride[0];
    a.tokens = static_cast<int>(query->shape[0]);
    a.rows = static_cast<int>(keys->shape[0]);
    a.batch = static_cast<int>(query_offsets->shape[0] - 1);
    a.heads = static_cast<int>(heads);
    a.kv_heads = static_cast<int>(kv_heads);
    a.group = static_cast<int>(heads / kv_heads);
    a.dim = static_cast<int>(query->shape[2]);
    a.window = window;
    a.sinks = sinks;
    a.scale = scale;
    auto kernel = query->dtype == MR_DTYPE_F32   ? k_rows<float>
                  : query->dtype == MR_DTYPE_F16 ? k_rows<__half>
                                                 : k_rows<__nv_bfloat16>;
    const int64_t warps = static_cast<int64_t>(a.tokens) * a.heads;
    kernel<<<static_cast<unsigned>((warps + 3) / 4), 128, 0, ctx->stream>>>(a);
    MR_CUDA_TRY(cudaGetLastError());
    return MR_OK;
}
