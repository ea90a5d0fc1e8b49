// Attention of one new token per sequence over a paged key / value cache.
//
//   s_t = scale q . k_t  over the rows t that the token sees,
//   out = sum_t exp(s_t - max s) v_t / sum_t exp(s_t - max s),
//
// per query head; heads / kv heads query heads read the same key / value rows.
#include <cmath>

#include "cache_ops.cuh"

namespace mr {
namespace cache {
namespace {

struct PagedArgs {
    const char *q, *k, *v;
    char *out;
    int64_t q_batch, q_head, o_batch, o_head;  // bytes
    int64_t k_page, k_row, k_head, v_page, v_row, v_head;
    Pages pages;
    const int *lengths;
    int64_t length_stride;
    float *weights;  // or NULL
    int64_t w_batch, w_head;
    int batch, kv_heads, group, dim, capacity, window, sinks;
    float scale;
};

// CTA = (sequence, key / value head); each warp takes every 4th row, four values of a row a lane.
template <typename T>
__global__ void __launch_bounds__(128) k_paged(PagedArgs a) {
    __shared__ float sm[4], sl[4], so[4][kMaxDim];
    const int s = blockIdx.x / a.kv_heads, kh = blockIdx.x % a.kv_heads, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int n = sequence_rows(a.lengths, a.length_stride, s, a.capacity);
    auto seen = [&](int t) { return a.window == 0 || n - 1 - t < a.window || t < a.sinks; };
    auto load = [&](const char *row, float (&x)[4]) {
        for (int j = 0; j < 4; ++j)
            x[j] = 4 * lane + j < a.dim ? widen(reinterpret_cast<const T *>(row) + 4 * lane + j) : 0.f;
    };
    for (int g = 0; g < a.group; ++g) {
        const int h = kh * a.group + g;
        float q[4], o[4] = {}, m = -INFINITY, l = 0.f;
        load(a.q + s * a.q_batch + h * a.q_head, q);
        auto score = [&](int t) {
            const int64_t r = a.pages.row(s, t, a.k_page, a.k_row);
            if (r < 0 || !seen(t)) return -INFINITY;
            float k[4];
            load(a.k + r + kh * a.k_head, k);
            return warp_sum(q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3]) * a.scale;
        };
        for (int t = warp; t < n; t += 4) {
            const float x = score(t);
            if (x == -INFINITY) continue;
            float v[4];
            load(a.v + a.pages.row(s, t, a.v_page, a.v_row) + kh * a.v_head, v);
            const float m_new = fmaxf(m, x), c = expf(m - m_new), p = expf(x - m_new);
            l = l * c + p;
            for (int j = 0; j < 4; ++j) o[j] = o[j] * c + p * v[j];
            m = m_new;
        }
        sm[warp] = m;
        sl[warp] = l;
        for (int j = 0; j < 4; ++j) so[warp][4 * lane + j] = o[j];
        __syncthreads();
        const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
        float sum = 0.f, c[4];
        for (int w = 0; w < 4; ++w) {
            c[w] = sm[w] == -INFINITY ? 0.f : expf(sm[w] - top);
            sum += sl[w] * c[w];
        }
        for (int j = threadIdx.x; j < a.dim; j += blockDim.x) {
            float x = 0.f;
            for (int w = 0; w < 4; ++w) x += so[w][j] * c[w];
            narrow(sum > 0.f ? x / sum : 0.f,
                   reinterpret_cast<T *>(a.out + s * a.o_batch + h * a.o_head) + j);
        }
        if (a.weights)
            for (int t = warp; t < n; t += 4) {
                const float x = score(t);
                if (x != -INFINITY && lane == 0) a.weights[s * a.w_batch + kh * a.w_head + t] += expf(x - top) / sum;
            }
        __syncthreads();
    }
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
    MR_CHECK(check_pools(key_pages, value_pages, "key_pages", "value_pages", false));
    MR_REQUIRE(query->dtype == key_pages->dtype && out->dtype == key_pages->dtype,
               "query, out and the pages must be of one type");
    for (int i = 0; i < 3; ++i) MR_REQUIRE(query->shape[i] == out->shape[i], "query and out differ in shape");
    MR_CHECK(check_apart(query, "query", out, "out"));
    const int64_t batch = query->shape[0], heads = query->shape[1], kv_heads = key_pages->shape[2];
    MR_REQUIRE(query->shape[2] == key_pages->shape[3], "query has %lld values a head, the pages %lld",
               static_cast<long long>(query->shape[2]), static_cast<long long>(key_pages->shape[3]));
    MR_REQUIRE(heads > 0 && heads % kv_heads == 0, "the %lld query heads must be a multiple of the pages' %lld heads",
               static_cast<long long>(heads), static_cast<long long>(kv_heads));
    MR_CHECK(check_ints(lengths, "lengths", 1));
    MR_REQUIRE(lengths->shape[0] == batch, "lengths must have %lld values", static_cast<long long>(batch));
    MR_CHECK(check_table(page_table, "page_table", batch, key_pages->shape[1]));
    MR_REQUIRE(batch * heads <= INT32_MAX / 2, "too many heads");
    MR_REQUIRE(window >= 0 && sinks >= 0, "window and sinks must not be negative");
    MR_REQUIRE(std::isfinite(scale), "scale must be finite");
    const int64_t capacity = page_table->shape[1] * key_pages->shape[1];
    if (weights) MR_CHECK(check_weights(weights, "weights", batch, kv_heads, capacity, true));
    MR_REQUIRE(ctx, "ctx is NULL");
    if (!batch) return MR_OK;
    DeviceGuard guard(ctx->device);
    const int64_t size = dtype_bytes(query->dtype);
    PagedArgs a;
    a.q = static_cast<const char *>(query->data);
    a.k = static_cast<const char *>(key_pages->data);
    a.v = static_cast<const char *>(value_pages->data);
    a.out = static_cast<char *>(out->data);
    a.q_batch = query->stride[0] * size;
    a.q_head = query->stride[1] * size;
    a.o_batch = out->stride[0] * size;
    a.o_head = out->stride[1] * size;
    a.k_page = key_pages->stride[0] * size;
    a.k_row = key_pages->stride[1] * size;
    a.k_head = key_pages->stride[2] * size;
    a.v_page = value_pages->stride[0] * size;
    a.v_row = value_pages->stride[1] * size;
    a.v_head = value_pages->stride[2] * size;
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
    a.scale = scale;
    auto kernel = query->dtype == MR_DTYPE_F32   ? k_paged<float>
                  : query->dtype == MR_DTYPE_F16 ? k_paged<__half>
                                                 : k_paged<__nv_bfloat16>;
    kernel<<<a.batch * a.kv_heads, 128, 0, ctx->stream>>>(a);
    MR_CUDA_TRY(cudaGetLastError());
    return MR_OK;
}
