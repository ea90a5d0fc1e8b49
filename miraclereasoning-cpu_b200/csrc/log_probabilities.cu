// Log probabilities of given tokens, the entropy and the most likely tokens of rows
// of logits x:
//
//   S = sum e^(x - m),  log p_t = x_t - m - log S,  H = log S - sum e^(x - m) (x - m) / S
//
// (m: about the maximum; differences, so that logits far from 0 cost no digits).
//
// One pass: every logit is read once, at about seven operations, and each thread
// keeps a running maximum, S and the entropy's sum of its own elements.  Bound by
// memory where there are many rows; a row is one CTA's, or where rows are few a
// cluster's of up to 8, whose sums and candidates meet in the first CTA's shared
// memory.
//
// The most likely tokens come from the threads' maxima.  The k-th largest maximum T
// is a lower bound of the k-th largest logit, and only a thread whose own maximum
// reaches T can have such logits: about k threads' elements (of 256) are read again,
// from L2, and the few that reach T are ranked by counting.  No work is added to the
// pass, and none of it depends on the order of the logits.  Where very many logits
// equal T (rows masked by -inf, constant rows), only larger ones are taken and the
// rest filled with the first ones that equal it.
#include <cooperative_groups.h>

#include "cache_ops.cuh"

namespace mr {
namespace cache {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256, kWarps = kThreads / 32, kMostTop = 128, kRoom = 1024, kMostCtas = 8;
constexpr float kLog2e = 1.4426950408889634f;
// e^-kFar is 0 in float32: differences are cut there where they are factors, so that 0 x -inf is no NaN
constexpr float kFar = 1e4f;

struct ScoreArgs {
    const char *logits;
    int64_t row_bytes;
    const int *tokens;
    float *logprobs, *entropy;
    int64_t token_row, logprob_row, entropy_row;
    int *top_tokens;
    float *top_logprobs;
    int64_t top_token_row, top_logprob_row;
    int vocab, given, top, ctas;  // ctas: of a row
};

// Logits in rising order as unsigned numbers; both zeros equal, NaN the lowest.
__device__ __forceinline__ uint32_t order_of(float x) {
    if (x != x) return 0;
    const uint32_t bits = __float_as_uint(x + 0.f);
    return bits ^ (static_cast<uint32_t>(static_cast<int32_t>(bits) >> 31) | 0x80000000u);
}
// The same with the token: larger is more likely, the lower token first; 0 is none.
__device__ __forceinline__ uint64_t candidate(uint32_t order, int token) {
    return static_cast<uint64_t>(order) << 32 | ~static_cast<uint32_t>(token);
}
__device__ __forceinline__ int token_of(uint64_t c) { return static_cast<int>(~static_cast<uint32_t>(c)); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Sums over elements x: s of e^(x - top), a of e^(x - top) (x - top).
struct Sums {
    float top, s, a;  // no elements, or -inf alone: top -inf
    __device__ __forceinline__ void add(const Sums &o) {
        const float to = fmaxf(top, o.top);
        auto moved = [&](const Sums &x, float &s2, float &a2) {
            const float by = x.top - to, c = ex2(by * kLog2e);
            const bool none = x.top == -INFINITY;  // nothing to move; s may be the NaN of a NaN
            s2 = none ? x.s : x.s * c;
            a2 = none ? x.a : c * fmaf(x.s, fmaxf(by, -kFar), x.a);
        };
        float s0, a0, s1, a1;
        moved(*this, s0, a0);
        moved(o, s1, a1);
        top = to;
        s = s0 + s1;
        a = a0 + a1;
    }
};

template <typename T>
struct Vector {
    static constexpr int kValues = 16 / sizeof(T);
    union {
        uint4 raw;
        T v[kValues];
    };
    __device__ __forceinline__ Vector() {}
    __device__ __forceinline__ float operator[](int i) const { return widen(&v[i]); }
};

// A CTA's part of a row: some single elements up to the first 16-byte boundary (the first CTA's),
// vectors, and the elements behind the last whole one (the last CTA's).
template <typename T>
struct Slice {
    static constexpr int V = Vector<T>::kValues;
    const T *row;
    const uint4 *vectors;  // vector 0 of the row
    int head, head_count;  // elements before vector 0, and those of this CTA
    int v0, v1;            // this CTA's vectors
    int tail, tail_count;  // first element behind the vectors, and those of this CTA
    __device__ __forceinline__ Slice(const ScoreArgs &a, int64_t r, int rank) {
        row = reinterpret_cast<const T *>(a.logits + r * a.row_bytes);
        const int odd = static_cast<int>((16 - reinterpret_cast<uintptr_t>(row) % 16) % 16 / sizeof(T));
        head = min(odd, a.vocab);
        vectors = reinterpret_cast<const uint4 *>(row + head);
        const int n = (a.vocab - head) / V;
        v0 = static_cast<int>(static_cast<int64_t>(n) * rank / a.ctas);
        v1 = static_cast<int>(static_cast<int64_t>(n) * (rank + 1) / a.ctas);
        tail = head + n * V;
        head_count = rank == 0 ? head : 0;
        tail_count = rank == a.ctas - 1 ? a.vocab - tail : 0;
    }
    __device__ __forceinline__ int count() const { return head_count + (v1 - v0) * V + tail_count; }
    __device__ __forceinline__ Vector<T> load(int v) const {
        Vector<T> x;
        x.raw = __ldg(vectors + v);
        return x;
    }
    // Elements that are no vector's: thread t's, at most two.  f(token, value)
    template <typename F>
    __device__ __forceinline__ void singles(int t, const F &f) const {
        if (t < head_count) f(t, widen(row + t));
        if (t < tail_count) f(tail + t, widen(row + tail + t));
    }
};

struct Shared {
    uint64_t found[kRoom];    // candidates
    uint64_t best[kMostTop];  // of them the largest, falling; 0 behind
    uint64_t all[kMostTop * kMostCtas];
    uint32_t maxima[kThreads];
    Sums sums[kWarps];
    Sums total;
    uint32_t bound;
    int count;
    int tally[kWarps];
};

// Candidates of the slice: elements from `bound` on, or past it.
template <typename T>
__device__ __forceinline__ void collect(const Slice<T> &slice, Shared &sh, uint32_t bound, bool past) {
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    auto push = [&](int token, float x) {
        const uint32_t o = order_of(x);
        if (past ? o > bound : o >= bound) {
            const int at = atomicAdd(&sh.count, 1);
            if (at < kRoom) sh.found[at] = candidate(o, token);
        }
    };
    slice.singles(tid, push);
    uint32_t mask = __ballot_sync(0xffffffffu, sh.maxima[tid] >= bound);
    while (mask) {
        const int t = warp * 32 + __ffs(mask) - 1;
        mask &= mask - 1;
        for (int v = slice.v0 + t + lane * kThreads; v < slice.v1; v += 32 * kThreads) {
            const Vector<T> x = slice.load(v);
#pragma unroll
            for (int j = 0; j < Slice<T>::V; ++j) push(slice.head + v * Slice<T>::V + j, x[j]);
        }
    }
}

// How many elements of the slice are from `bound` on; all threads have it.
template <typename T>
__device__ int count_from(const Slice<T> &slice, Shared &sh, uint32_t bound) {
    const int tid = threadIdx.x;
    int n = 0;
    auto add = [&](int, float x) { n += order_of(x) >= bound; };
    slice.singles(tid, add);
    for (int v = slice.v0 + tid; v < slice.v1; v += kThreads) {
        const Vector<T> x = slice.load(v);
#pragma unroll
        for (int j = 0; j < Slice<T>::V; ++j) add(0, x[j]);
    }
    n = __reduce_add_sync(0xffffffffu, n);
    __syncthreads();
    if (tid % 32 == 0) sh.tally[tid / 32] = n;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) n += sh.tally[w];
    return n;
}

// The slice's `want` largest elements into sh.best.
template <typename T>
__device__ __forceinline__ void choose(const Slice<T> &slice, Shared &sh, float largest, int want) {
    constexpr int V = Slice<T>::V;
    const int tid = threadIdx.x, lane = tid % 32;
    const int mine = (tid < slice.head_count) + (tid < slice.tail_count) + (slice.v0 + tid < slice.v1);
    sh.maxima[tid] = mine ? max(order_of(largest), 1u) : 0u;  // at least 1, of NaN alone too: has elements
    if (tid == 0) sh.count = 0;
    __syncthreads();
    if (tid < 32) {
        // the want-th largest of the maxima, or a number below it that not many more reach: halving
        uint32_t key[kWarps], low = 0xffffffffu, high = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            key[w] = sh.maxima[w * 32 + lane];
            low = min(low, key[w]);
            high = max(high, key[w]);
        }
        low = __reduce_min_sync(0xffffffffu, low);
        high = __reduce_max_sync(0xffffffffu, high);
        int reach = kThreads;
        ++high;  // order_of(+inf) at most: does not wrap
        while (high - low > 1 && reach > want + 8) {
            const uint32_t mid = low + (high - low) / 2;
            int n = 0;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) n += key[w] >= mid;
            n = __reduce_add_sync(0xffffffffu, n);
            if (n >= want) low = mid, reach = n;
            else high = mid;
        }
        // fewer threads with elements than wanted, or among them NaN alone: everything counts
        if (lane == 0) sh.bound = low <= 1 ? 0u : low;
    }
    __syncthreads();
    uint32_t bound = sh.bound;
    auto collected = [&](bool past) {
        collect(slice, sh, bound, past);
        __syncthreads();
        const int n = sh.count;
        __syncthreads();
        if (tid == 0) sh.count = 0;
        __syncthreads();
        return n;
    };
    int n = collected(false);
    bool enough = n >= want;  // from the bound on (threads of NaN alone have less than their maximum says)
    if (enough && n > kRoom) n = collected(true);
    if (!enough || n > kRoom) {
        // the want-th largest itself, bit by bit
        bound = 0;
        for (int bit = 31; bit >= 0; --bit)
            if (count_from(slice, sh, bound | 1u << bit) >= want) bound |= 1u << bit;
        n = collected(true);
    }
    if (n < want) {
        // more than the first `want` equal the bound: the first of them
        if (tid < 32) {
            int at = n;
            auto fill = [&](bool is, int token) {
                const bool equal = is && order_of(widen(slice.row + token)) == bound;
                const uint32_t hit = __ballot_sync(0xffffffffu, equal);
                const int to = at + __popc(hit & ((1u << lane) - 1));
                if (equal && to < want) sh.found[to] = candidate(bound, token);
                at += __popc(hit);
            };
            fill(lane < slice.head_count, lane);
            for (int v = slice.v0; v < slice.v1 && at < want; v += 32 / V)  // V neighbouring lanes have a vector's elements
                fill(v + lane / V < slice.v1, slice.head + v * V + lane);
            fill(lane < slice.tail_count, slice.tail + lane);
        }
        n = want;
        __syncthreads();
    }
    for (int i = tid; i < kMostTop; i += kThreads) sh.best[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) {
        const uint64_t c = sh.found[i];
        int above = 0;
        for (int j = 0; j < n; ++j) above += sh.found[j] > c;
        if (above < want) sh.best[above] = c;
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_log_probabilities(const __grid_constant__ ScoreArgs a) {
    __shared__ Shared sh;
    constexpr int V = Slice<T>::V, kFlight = sizeof(T) == 4 ? 4 : 2;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const int rank = a.ctas == 1 ? 0 : static_cast<int>(cg::this_cluster().block_rank());
    const int64_t r = blockIdx.x / a.ctas;
    const Slice<T> slice(a, r, rank);
    Sums mine = {-INFINITY, 0.f, 0.f};
    float from = 0.f;  // mine.top, 0 while that is -inf: -inf less 0 is no NaN
    auto grow = [&](float top) {
        if (top > mine.top) {
            if (mine.top != -INFINITY) {
                const float by = fmaxf(mine.top - top, -kFar), c = ex2(by * kLog2e);
                mine.a = c * fmaf(mine.s, by, mine.a);
                mine.s *= c;
            }
            mine.top = from = top;
        }
    };
    auto add = [&](float x) {
        const float d = x - from, e = ex2(d * kLog2e);
        mine.s += e;
        mine.a = fmaf(e, fmaxf(d, -kFar), mine.a);
    };
    slice.singles(tid, [&](int, float x) {
        grow(x);
        add(x);
    });
    for (int v = slice.v0 + tid; v < slice.v1; v += kFlight * kThreads) {
        Vector<T> x[kFlight];
#pragma unroll
        for (int f = 0; f < kFlight; ++f)
            if (v + f * kThreads < slice.v1) x[f] = slice.load(v + f * kThreads);
            else x[f].raw = make_uint4(0, 0, 0, 0);
        float top = -INFINITY;
#pragma unroll
        for (int f = 0; f < kFlight; ++f)
            if (v + f * kThreads < slice.v1)
#pragma unroll
                for (int j = 0; j < V; ++j) top = fmaxf(top, x[f][j]);
        grow(top);
#pragma unroll
        for (int f = 0; f < kFlight; ++f)
            if (v + f * kThreads < slice.v1)
#pragma unroll
                for (int j = 0; j < V; ++j) add(x[f][j]);
    }
    // the row's sums
    Sums sum = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Sums other = {__shfl_xor_sync(0xffffffffu, sum.top, o), __shfl_xor_sync(0xffffffffu, sum.s, o),
                            __shfl_xor_sync(0xffffffffu, sum.a, o)};
        sum.add(other);
    }
    if (lane == 0) sh.sums[warp] = sum;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int w = 1; w < kWarps; ++w) sum.add(sh.sums[w]);
        sh.total = sum;
    }
    if (a.top) choose(slice, sh, mine.top, min(a.top, slice.count()));
    if (a.ctas > 1) {
        cg::this_cluster().sync();
        if (rank == 0) {
            if (tid == 0) {
                for (int c = 1; c < a.ctas; ++c) sum.add(cg::this_cluster().map_shared_rank(&sh, c)->total);
                sh.total = sum;
            }
            const int n = a.ctas * a.top;
            for (int i = tid; i < n; i += kThreads)
                sh.all[i] = cg::this_cluster().map_shared_rank(&sh, i / a.top)->best[i % a.top];
        }
        cg::this_cluster().sync();  // the others' memory has been read
        if (rank) return;
        const int n = a.ctas * a.top;
        for (int i = tid; i < n; i += kThreads) {
            const uint64_t c = sh.all[i];
            int above = 0;
            for (int j = 0; j < n; ++j) above += sh.all[j] > c;
            if (c && above < a.top) sh.best[above] = c;
        }
    }
    __syncthreads();
    const Sums all = sh.total;
    const float log_s = logf(all.s);
    // a row of -inf alone: -inf, and no entropy
    auto log_p = [&](int token) { return all.s == 0.f ? -INFINITY : widen(slice.row + token) - all.top - log_s; };
    if (a.entropy && tid == 0) a.entropy[r * a.entropy_row] = all.s == 0.f ? 0.f : log_s - all.a / all.s;
    for (int i = tid; i < a.given; i += kThreads) {
        const int t = a.tokens[r * a.token_row + i];
        a.logprobs[r * a.logprob_row + i] = static_cast<unsigned>(t) < static_cast<unsigned>(a.vocab) ? log_p(t) : 0.f;
    }
    for (int i = tid; i < a.top; i += kThreads) {
        const int t = token_of(sh.best[i]);
        a.top_tokens[r * a.top_token_row + i] = t;
        a.top_logprobs[r * a.top_logprob_row + i] = log_p(t);
    }
}

template <typename T>
int launch(mr_context *ctx, ScoreArgs &a, int64_t rows) {
    // CTAs of a row: as many as give the GPU four an SM, each with two vectors a thread at least
    a.ctas = 1;
    while (a.ctas < kMostCtas && rows * a.ctas * 2 <= 4 * ctx->sm_count &&
           a.vocab / Slice<T>::V >= 2 * kThreads * a.ctas * 2)
        a.ctas *= 2;
    cudaLaunchAttribute cluster;
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = a.ctas;
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(rows * a.ctas));
    config.blockDim = dim3(kThreads);
    config.stream = ctx->stream;
    config.attrs = &cluster;
    config.numAttrs = a.ctas > 1;
    MR_CUDA_TRY(cudaLaunchKernelEx(&config, k_log_probabilities<T>, a));
    return MR_OK;
}

// An output [rows, n] of a type; its row stride.
int check_output(const mr_array *a, const char *name, int dtype, int64_t rows, int64_t n) {
    MR_CHECK(check_array(a, name, 2, false, true));
    MR_REQUIRE(a->dtype == dtype, "%s must be %s", name, dtype == MR_DTYPE_F32 ? "float32" : "int32");
    MR_REQUIRE(a->shape[0] == rows && a->shape[1] == n, "%s must be [%lld, %lld]", name, static_cast<long long>(rows),
               static_cast<long long>(n));
    return MR_OK;
}

}  // namespace
}  // namespace cache
}  // namespace mr

using namespace mr::cache;

extern "C" int mr_log_probabilities(mr_context *ctx, const mr_array *logits, const mr_array *tokens, const mr_array *logprobs,
                                    const mr_array *entropy, const mr_array *top_tokens, const mr_array *top_logprobs) {
    MR_CHECK(check_array(logits, "logits", 2, false, false));
    MR_REQUIRE(is_float(logits->dtype), "logits must be of a floating type");
    const int64_t rows = logits->shape[0], vocab = logits->shape[1];
    MR_REQUIRE(vocab > 0, "logits must have a vocabulary");
    MR_REQUIRE(vocab < INT32_MAX / 2, "the vocabulary is too large");
    MR_REQUIRE(rows <= INT32_MAX / kMostCtas, "too many rows");
    MR_REQUIRE(!tokens == !logprobs, "tokens and logprobs go together");
    MR_REQUIRE(!top_tokens == !top_logprobs, "top_tokens and top_logprobs go together");
    ScoreArgs a = {};
    if (tokens) {
        MR_REQUIRE(tokens->ndim == 1 || tokens->ndim == 2, "tokens must have 1 or 2 dimensions, not %d", tokens->ndim);
        MR_CHECK(check_ints(tokens, "tokens", tokens->ndim));
        MR_CHECK(check_array(logprobs, "logprobs", tokens->ndim, false, true));
        MR_REQUIRE(logprobs->dtype == MR_DTYPE_F32, "logprobs must be float32");
        MR_REQUIRE(tokens->shape[0] == rows, "tokens must have a row for each of the %lld rows of logits",
                   static_cast<long long>(rows));
        for (int i = 0; i < tokens->ndim; ++i)
            MR_REQUIRE(tokens->shape[i] == logprobs->shape[i], "tokens and logprobs differ in shape");
        MR_CHECK(check_apart(tokens, "tokens", logprobs, "logprobs"));
        a.tokens = static_cast<const int *>(tokens->data);
        a.logprobs = static_cast<float *>(logprobs->data);
        a.token_row = tokens->stride[0];
        a.logprob_row = logprobs->stride[0];
        a.given = tokens->ndim == 1 ? 1 : static_cast<int>(tokens->shape[1]);
    }
    if (entropy) {
        MR_CHECK(check_array(entropy, "entropy", 1, false, true));
        MR_REQUIRE(entropy->dtype == MR_DTYPE_F32, "entropy must be float32");
        MR_REQUIRE(entropy->shape[0] == rows, "entropy must have %lld values", static_cast<long long>(rows));
        a.entropy = static_cast<float *>(entropy->data);
        a.entropy_row = entropy->stride[0];
    }
    if (top_tokens) {
        MR_REQUIRE(top_tokens->ndim == 2, "top_tokens must have 2 dimensions, not %d", top_tokens->ndim);
        const int64_t top = top_tokens->shape[1];
        MR_REQUIRE(top <= kMostTop && top <= vocab, "at most %lld tokens can be asked for, not %lld",
                   static_cast<long long>(std::min<int64_t>(kMostTop, vocab)), static_cast<long long>(top));
        MR_CHECK(check_output(top_tokens, "top_tokens", MR_DTYPE_I32, rows, top));
        MR_CHECK(check_output(top_logprobs, "top_logprobs", MR_DTYPE_F32, rows, top));
        MR_CHECK(check_apart(top_tokens, "top_tokens", top_logprobs, "top_logprobs"));
        a.top_tokens = static_cast<int *>(top_tokens->data);
        a.top_logprobs = static_cast<float *>(top_logprobs->data);
        a.top_token_row = top_tokens->stride[0];
        a.top_logprob_row = top_logprobs->stride[0];
        a.top = static_cast<int>(top);
    }
    MR_REQUIRE(ctx, "ctx is NULL");
    MR_CHECK(mr::check_waits(ctx));
    if (!rows) return MR_OK;
    DeviceGuard guard(ctx->device);
    a.logits = static_cast<const char *>(logits->data);
    a.row_bytes = logits->stride[0] * dtype_bytes(logits->dtype);
    a.vocab = static_cast<int>(vocab);
    return logits->dtype == MR_DTYPE_F32   ? launch<float>(ctx, a, rows)
           : logits->dtype == MR_DTYPE_F16 ? launch<__half>(ctx, a, rows)
                                           : launch<__nv_bfloat16>(ctx, a, rows);
}
