// New rows of a paged key / value cache with the position rotation applied on the
// way, into pages of the rows' own type or of 4 bits a value; and rows read back.
//
//   angle = position * frequency[p],  (a, b) -> (a cos - b sin, b cos + a sin)
//
// for each pair p of a query's or key's first 2 n dims.  Everything is read and
// written once, with a few operations a value: bound by memory, once the angles
// are cheap.  They are worked out once a token and part of its rows, in the
// registers of the warp that turns them.
#include <cmath>

#include "packed.cuh"

namespace mr {
namespace cache {
namespace {

struct Pool {
    char *base;
    int64_t page, row, head;  // bytes
};
Pool make_pool(const mr_array *a) {
    const int64_t size = dtype_bytes(a->dtype);
    return Pool{static_cast<char *>(a->data), a->stride[0] * size, a->stride[1] * size, a->stride[2] * size};
}

// Rows [tokens, heads, dim]; strides in bytes.
struct Rows {
    char *base;
    int64_t token, head;
};
Rows make_rows(const mr_array *a) {
    const int64_t size = dtype_bytes(a->dtype);
    return Rows{static_cast<char *>(a->data), a->stride[0] * size, a->stride[1] * size};
}

struct PlaceArgs {
    const int *lengths, *offsets;  // offsets NULL: token i is sequence i's newest row
    int64_t length_stride, offset_stride;
    int batch;
};

// The sequence of packed token i (-1: of none) and its row there, which may lie before the first.
__device__ __forceinline__ int place_of(const PlaceArgs &a, int i, int &row) {
    int s = i, behind = 1;  // rows from this one to the sequence's end
    if (a.offsets) {
        int lo = -1, hi = a.batch;  // offsets[lo] <= i < offsets[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (__ldg(a.offsets + mid * a.offset_stride) <= i) lo = mid;
            else hi = mid;
        }
        if (lo < 0) return -1;
        const int end = __ldg(a.offsets + (lo + 1) * a.offset_stride);
        if (end <= i) return -1;
        s = lo;
        behind = end - i;
    }
    row = max(0, __ldg(a.lengths + s * a.length_stride)) - behind;
    return s;
}

// Four values as float32.
__device__ __forceinline__ void load4(const float *p, float (&x)[4]) {
    const float4 v = *reinterpret_cast<const float4 *>(p);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}
template <typename T>
__device__ __forceinline__ void load4(const T *p, float (&x)[4]) {
    union {
        uint2 raw;
        T v[4];
    } u;
    u.raw = *reinterpret_cast<const uint2 *>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = widen(&u.v[j]);
}
__device__ __forceinline__ void store4(float *p, const float (&x)[4]) {
    *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
template <typename T>
__device__ __forceinline__ void store4(T *p, const float (&x)[4]) {
    union {
        uint2 raw;
        T v[4];
    } u;
#pragma unroll
    for (int j = 0; j < 4; ++j) narrow(x[j], &u.v[j]);
    *reinterpret_cast<uint2 *>(p) = u.raw;
}

__device__ __forceinline__ float min_nan(float a, float b) {
    float x;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(x) : "f"(a), "f"(b));
    return x;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float x;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(x) : "f"(a), "f"(b));
    return x;
}

// sin and cos of position * frequency, each rounded to float32 once.  The product is kept in
// two parts and reduced by multiples of pi / 2 in 64 bits, so that far positions lose nothing
// (2^31 radians leave 2^-70); what is left, at most pi / 4, goes through the Taylor series to
// x^15 and x^16, whose next terms are below 5e-17.  One angle is about 25 64-bit operations.
__device__ __forceinline__ float2 turn_of(int position, float frequency) {
    const double p = position, f = frequency;
    const double a = p * f, rest = fma(p, f, -a);
    const double q = rint(a * 0.63661977236758134308);
    double r = fma(q, -1.57079632679489655800, a);
    r = fma(q, -6.12323399573676603587e-17, r) + rest;
    const double x = r * r;
    double s = -1.0 / 1307674368000.0;
    s = fma(s, x, 1.0 / 6227020800.0);
    s = fma(s, x, -1.0 / 39916800.0);
    s = fma(s, x, 1.0 / 362880.0);
    s = fma(s, x, -1.0 / 5040.0);
    s = fma(s, x, 1.0 / 120.0);
    s = fma(s, x, -1.0 / 6.0);
    s = fma(s * x, r, r);
    double c = 1.0 / 20922789888000.0;
    c = fma(c, x, -1.0 / 87178291200.0);
    c = fma(c, x, 1.0 / 479001600.0);
    c = fma(c, x, -1.0 / 3628800.0);
    c = fma(c, x, 1.0 / 40320.0);
    c = fma(c, x, -1.0 / 720.0);
    c = fma(c, x, 1.0 / 24.0);
    c = fma(c, x, -0.5);
    c = fma(c, x, 1.0);
    const int quarter = static_cast<int>(static_cast<long long>(q) & 3);
    const float sin0 = static_cast<float>(s), cos0 = static_cast<float>(c);
    const float sin1 = quarter & 1 ? cos0 : sin0, cos1 = quarter & 1 ? sin0 : cos0;
    return make_float2(quarter == 1 || quarter == 2 ? -cos1 : cos1, quarter & 2 ? -sin1 : sin1);  // cos, sin
}

struct RotateArgs {
    Rows q, k, v, out;
    Pool key_pool, value_pool;
    Pages pages;
    PlaceArgs place;
    const float *frequencies;
    const int *positions;  // NULL: a token's row
    int64_t frequency_stride, position_stride;
    int tokens, heads, kv_heads, dim, half;  // half: pairs that turn
    int team, share;                         // warps that share a token's rows, tokens of such a team
};

// How pairs lie: neighbours; p and p + half with four dims of a lane alike (half a multiple of
// 4); the same, any half.
enum { kNeighbours, kHalves, kAnyHalves };

// A warp takes `share` tokens, or a part of one token's rows: of the queries, then keys, then
// values.  A lane has the same four dims of every row (L lanes a row), so that a token's
// angles stay in registers; kFlight rows a lane are under way.  Products and sums of a turn are
// rounded one by one, so that a 4-bit code is the same wherever it is worked out.
template <typename T, int PAIRS, bool PACKED>
__global__ void __launch_bounds__(256) k_append_rotated(const __grid_constant__ RotateArgs a) {
    constexpr int kFlight = 4;
    const int lane = threadIdx.x % 32, warp = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    const int64_t first = static_cast<int64_t>(warp / a.team) * a.share;
    const int part = warp % a.team;
    if (first >= a.tokens) return;
    int64_t mine_k = -1, mine_v = -1;
    int mine_position = 0;
    bool mine_owned = false;
    if (lane < a.share && first + lane < a.tokens) {
        const int i = static_cast<int>(first) + lane;
        int t = 0;
        const int s = place_of(a.place, i, t);
        mine_owned = s >= 0;
        if (mine_owned) {
            mine_position = a.positions ? __ldg(a.positions + i * a.position_stride) : t;
            if (t >= 0) {
                mine_k = a.pages.row(s, t, a.key_pool.page, a.key_pool.row);
                mine_v = a.pages.row(s, t, a.value_pool.page, a.value_pool.row);
            }
        }
    }
    int wide = 1;  // lanes a row
    while (wide * 4 < a.dim) wide <<= 1;
    const int sub = lane / wide, d = lane % wide * 4, rows = a.heads + 2 * a.kv_heads, each = 32 / wide * a.team;
    const bool inside = d < a.dim;
    const int dim0 = inside ? d : 0;
    for (int n = 0; n < a.share && first + n < a.tokens; ++n) {
        if (!__shfl_sync(0xffffffffu, mine_owned, n)) continue;
        const int64_t to_k = __shfl_sync(0xffffffffu, mine_k, n), to_v = __shfl_sync(0xffffffffu, mine_v, n);
        const int position = __shfl_sync(0xffffffffu, mine_position, n), token = static_cast<int>(first) + n;
        // cos and sin of the pairs of the lane's dims; (1, 0) where they do not turn
        float2 turn[4];
        auto angle = [&](int p) {
            return p < a.half ? turn_of(position, __ldg(a.frequencies + p * a.frequency_stride)) : make_float2(1.f, 0.f);
        };
        if (PAIRS == kNeighbours) {
            turn[0] = turn[1] = angle(dim0 / 2);
            turn[2] = turn[3] = angle(dim0 / 2 + 1);
        } else if (PAIRS == kHalves) {
            // each of the two lanes that meet the same four pairs works out two of them
            const bool low = dim0 < a.half;
            const int p = low ? dim0 : dim0 - a.half, there = lane + (low ? a.half : -a.half) / 4;
            const float2 x = angle(p + (low ? 0 : 2)), y = angle(p + (low ? 1 : 3));
            const int from = dim0 < 2 * a.half ? there : lane;
            const float2 u = make_float2(__shfl_sync(0xffffffffu, x.x, from), __shfl_sync(0xffffffffu, x.y, from));
            const float2 w = make_float2(__shfl_sync(0xffffffffu, y.x, from), __shfl_sync(0xffffffffu, y.y, from));
            turn[0] = low ? x : u;
            turn[1] = low ? y : w;
            turn[2] = low ? u : x;
            turn[3] = low ? w : y;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) turn[j] = angle(dim0 + j < a.half ? dim0 + j : dim0 + j - a.half);
        }
        for (int base = part * (32 / wide); base < rows; base += each * kFlight) {
            float x[kFlight][4], y[kFlight][4];  // the values, and with pairs of halves their partners
#pragma unroll
            for (int f = 0; f < kFlight; ++f) {
                const int i = base + sub + f * each;
                const bool there = inside && i < rows;
                const Rows &from = i < a.heads ? a.q : i < a.heads + a.kv_heads ? a.k : a.v;
                const int h = i < a.heads ? i : i < a.heads + a.kv_heads ? i - a.heads : i - a.heads - a.kv_heads;
                const T *row = reinterpret_cast<const T *>(from.base + token * from.token + h * from.head);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[f][j] = y[f][j] = 0.f;
                if (there) load4(row + d, x[f]);
                if (PAIRS == kHalves && there && i < a.heads + a.kv_heads && d < 2 * a.half)
                    load4(row + (d < a.half ? d + a.half : d - a.half), y[f]);
                if (PAIRS == kAnyHalves && there && i < a.heads + a.kv_heads) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int e = d + j;
                        if (e < 2 * a.half) y[f][j] = widen(row + (e < a.half ? e + a.half : e - a.half));
                    }
                }
            }
#pragma unroll
            for (int f = 0; f < kFlight; ++f) {
                const int i = base + sub + f * each;
                const bool query = i < a.heads, value = i >= a.heads + a.kv_heads, there = inside && i < rows;
                const int h = query ? i : value ? i - a.heads - a.kv_heads : i - a.heads;
                if (!value) {
                    float z[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int e = d + j;
                        const bool turns = e < 2 * a.half;
                        const bool second = PAIRS == kNeighbours ? j & 1 : e >= a.half;
                        const float other = PAIRS == kNeighbours ? x[f][j ^ 1] : y[f][j];
                        const float p = __fmul_rn(x[f][j], turn[j].x), q = __fmul_rn(other, turn[j].y);
                        z[j] = !turns ? x[f][j] : second ? __fadd_rn(p, q) : __fsub_rn(p, q);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[f][j] = z[j];
                }
                const int64_t place = value ? to_v : to_k;
                const Pool &pool = value ? a.value_pool : a.key_pool;
                char *to = pool.base + place + h * pool.head;
                if (query) {
                    if (there) store4(reinterpret_cast<T *>(a.out.base + token * a.out.token + h * a.out.head) + d, x[f]);
                } else if (!PACKED) {
                    if (there && place >= 0) store4(reinterpret_cast<T *>(to) + d, x[f]);
                }
                if (PACKED && __any_sync(0xffffffffu, there && !query)) {
                    // 8 lanes share a step and a base
                    float lo = min_nan(min_nan(x[f][0], x[f][1]), min_nan(x[f][2], x[f][3]));
                    float hi = max_nan(max_nan(x[f][0], x[f][1]), max_nan(x[f][2], x[f][3]));
#pragma unroll
                    for (int o = 1; o < 8; o <<= 1) {
                        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
                        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
                    }
                    const __half step = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f));
                    const float s = __half2float(step);
                    const __half zero = __float2half_rn(__fsub_rn(lo, __fmul_rn(64.f, s)));
                    const float z = __half2float(zero);
                    const bool held = fabsf(s) < INFINITY && fabsf(z) < INFINITY;
                    uint32_t codes = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float c = rintf(__fdiv_rn(__fsub_rn(x[f][j], z), s)) - 64.f;
                        const uint32_t code = held && s != 0.f ? static_cast<uint32_t>(fminf(fmaxf(c, 0.f), 15.f)) : 0u;
                        codes |= code << (4 * j);
                    }
                    if (!query && there && place >= 0) {
                        *reinterpret_cast<uint16_t *>(to + d / 2) = static_cast<uint16_t>(codes);
                        if (d % kShared == 0) {
                            const uint32_t nan = 0x7e007e00u;
                            *reinterpret_cast<uint32_t *>(to + a.dim / 2 + d / kShared * 4) =
                                held ? __half_as_ushort(step) | static_cast<uint32_t>(__half_as_ushort(zero)) << 16 : nan;
                        }
                    }
                }
            }
        }
    }
}

template <typename T, bool PACKED>
int launch_pairs(mr_context *ctx, const RotateArgs &a, bool split_half) {
    // As many warps to a token as fill the GPU (16 to an SM) when tokens are few, one with several tokens when many.
    const int rows = a.heads + 2 * a.kv_heads;
    RotateArgs b = a;
    const int64_t warps = 16 * static_cast<int64_t>(ctx->sm_count);
    b.team = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(rows, warps / std::max(a.tokens, 1))));
    b.share = b.team > 1 ? 1 : static_cast<int>(std::min<int64_t>(4, (a.tokens + 2 * warps - 1) / (2 * warps)));
    const int64_t all = (static_cast<int64_t>(a.tokens) + b.share - 1) / b.share * b.team;
    constexpr int kWarps = 4;
    const unsigned grid = static_cast<unsigned>((all + kWarps - 1) / kWarps);
    if (!split_half) k_append_rotated<T, kNeighbours, PACKED><<<grid, kWarps * 32, 0, ctx->stream>>>(b);
    else if (a.half % 4 == 0) k_append_rotated<T, kHalves, PACKED><<<grid, kWarps * 32, 0, ctx->stream>>>(b);
    else k_append_rotated<T, kAnyHalves, PACKED><<<grid, kWarps * 32, 0, ctx->stream>>>(b);
    MR_CUDA_TRY(cudaGetLastError());
    return MR_OK;
}
template <typename T>
int launch_rotated(mr_context *ctx, const RotateArgs &a, bool split_half, bool packed) {
    return packed ? launch_pairs<T, true>(ctx, a, split_half) : launch_pairs<T, false>(ctx, a, split_half);
}

// ---- rows read back -----------------------------------------------------------------
struct ReadArgs {
    Rows k, v;
    Pool key_pool, value_pool;
    Pages pages;
    PlaceArgs place;
    int tokens, heads, pieces;  // pieces: 16-byte pieces of a row of the results
    int code_bytes;             // of a 4-bit row
    int team, share;            // warps that share a token's rows, tokens of such a team
};

// 16 bytes of a result's row, from piece c of a pool's row.
template <typename T, bool PACKED>
struct Piece {
    uint4 raw;         // PACKED: x: the codes, y: step and base
    __device__ __forceinline__ void load(const char *row, int c, int code_bytes) {
        constexpr int kValues = 16 / sizeof(T);
        if constexpr (!PACKED) {
            raw = *reinterpret_cast<const uint4 *>(row + 16 * c);
        } else {
            raw.x = kValues == 8 ? *reinterpret_cast<const uint32_t *>(row + 4 * c) : *reinterpret_cast<const uint16_t *>(row + 2 * c);
            raw.y = *reinterpret_cast<const uint32_t *>(row + code_bytes + c * kValues / kShared * 4);
        }
    }
    __device__ __forceinline__ uint4 value() const {
        if constexpr (!PACKED) {
            return raw;
        } else {
            constexpr int kValues = 16 / sizeof(T);
            const __half2 pair = *reinterpret_cast<const __half2 *>(&raw.y);
            const __half2 s = __low2half2(pair), z = __high2half2(pair);
            union {
                uint4 all;
                T v[kValues];
            } u;
#pragma unroll
            for (int j = 0; j < kValues; j += 2) {
                // codes j and j + 1 into bits 4 .. 7 of the two halves
                const uint32_t byte = raw.x >> (4 * j), two = (byte & 0xfu) << 4 | (byte & 0xf0u) << 16;
                const uint32_t x = fma2(codes64(two), s, z);
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&x));
                narrow(f.x, &u.v[j]);
                narrow(f.y, &u.v[j + 1]);
            }
            return u.all;
        }
    }
};

template <typename T, bool PACKED>
__global__ void __launch_bounds__(256) k_read_pages(const __grid_constant__ ReadArgs a) {
    constexpr int kFlight = 4;
    const int lane = threadIdx.x % 32, warp = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    const int64_t first = static_cast<int64_t>(warp / a.team) * a.share;
    if (first >= a.tokens) return;
    int64_t mine_k = -1, mine_v = -1;
    bool mine_owned = false;
    if (lane < a.share && first + lane < a.tokens) {
        int t = 0;
        const int s = place_of(a.place, static_cast<int>(first) + lane, t);
        mine_owned = s >= 0;
        if (s >= 0 && t >= 0) {
            mine_k = a.pages.row(s, t, a.key_pool.page, a.key_pool.row);
            mine_v = a.pages.row(s, t, a.value_pool.page, a.value_pool.row);
        }
    }
    const int n = a.heads * a.pieces;
    const int all = static_cast<int>(min(static_cast<int64_t>(a.share), a.tokens - first)) * n;
    for (int e0 = lane + warp % a.team * 32 * kFlight; e0 - lane < all; e0 += 32 * kFlight * a.team) {
        Piece<T, PACKED> x[kFlight], y[kFlight];
        char *to_k[kFlight], *to_v[kFlight];
#pragma unroll
        for (int f = 0; f < kFlight; ++f) {
            const int e = min(e0 + 32 * f, all - 1), token = e / n, i = e - token * n, h = i / a.pieces, c = i - h * a.pieces;
            const int64_t k = __shfl_sync(0xffffffffu, mine_k, token), v = __shfl_sync(0xffffffffu, mine_v, token);
            const bool owned = __shfl_sync(0xffffffffu, mine_owned, token) && e0 + 32 * f < all;
            to_k[f] = owned ? a.k.base + (first + token) * a.k.token + h * a.k.head + 16 * c : nullptr;
            to_v[f] = a.v.base + (first + token) * a.v.token + h * a.v.head + 16 * c;
            x[f].raw = y[f].raw = make_uint4(0, 0, 0, 0);  // a row that is not there: step and base 0, or zeros
            if (owned && k >= 0) {
                x[f].load(a.key_pool.base + k + h * a.key_pool.head, c, a.code_bytes);
                y[f].load(a.value_pool.base + v + h * a.value_pool.head, c, a.code_bytes);
            }
        }
#pragma unroll
        for (int f = 0; f < kFlight; ++f)
            if (to_k[f]) {
                *reinterpret_cast<uint4 *>(to_k[f]) = x[f].value();
                *reinterpret_cast<uint4 *>(to_v[f]) = y[f].value();
            }
    }
}

// Checks that the three operators share: rows of keys and values that stand for pages' rows.
int check_rows(const mr_array *keys, const mr_array *values, const mr_array *key_pages, const mr_array *value_pages,
               const mr_array *page_table, const mr_array *lengths, const mr_array *offsets, bool read) {
    MR_CHECK(check_array(keys, "keys", 3, true, read));
    MR_CHECK(check_array(values, "values", 3, true, read));
    MR_REQUIRE(is_float(keys->dtype) && values->dtype == keys->dtype, "keys and values must be of one floating type");
    for (int i = 0; i < 3; ++i) MR_REQUIRE(keys->shape[i] == values->shape[i], "keys and values differ in shape");
    MR_REQUIRE(key_pages, "key_pages is missing");
    int64_t dim;
    if (key_pages->dtype == MR_DTYPE_U8) {
        MR_CHECK(check_packed(key_pages, value_pages, "key_pages", "value_pages", !read));
        dim = packed_dim(key_pages->shape[3]);
    } else {
        MR_CHECK(check_pools(key_pages, value_pages, "key_pages", "value_pages", !read));
        MR_REQUIRE(keys->dtype == key_pages->dtype, "keys, values and the pages must be of one type");
        dim = key_pages->shape[3];
    }
    MR_REQUIRE(keys->shape[1] == key_pages->shape[2] && keys->shape[2] == dim,
               "keys must be [tokens, %lld, %lld], as the pages' heads and dim",
               static_cast<long long>(key_pages->shape[2]), static_cast<long long>(dim));
    MR_REQUIRE(keys->shape[1] * dim <= INT32_MAX / 4, "too many heads");
    MR_CHECK(check_ints(lengths, "lengths", 1));
    const int64_t batch = lengths->shape[0];
    MR_CHECK(check_table(page_table, "page_table", batch, key_pages->shape[1]));
    if (offsets) {
        MR_CHECK(check_ints(offsets, "offsets", 1));
        MR_REQUIRE(offsets->shape[0] == batch + 1, "offsets must have %lld values (batch + 1)",
                   static_cast<long long>(batch + 1));
    } else {
        MR_REQUIRE(keys->shape[0] == batch, "without offsets, keys must have one row for each of the %lld sequences",
                   static_cast<long long>(batch));
    }
    return MR_OK;
}

PlaceArgs make_place(const mr_array *lengths, const mr_array *offsets) {
    PlaceArgs p;
    p.lengths = static_cast<const int *>(lengths->data);
    p.length_stride = lengths->stride[0];
    p.offsets = offsets ? static_cast<const int *>(offsets->data) : nullptr;
    p.offset_stride = offsets ? offsets->stride[0] : 0;
    p.batch = static_cast<int>(lengths->shape[0]);
    return p;
}

}  // namespace
}  // namespace cache
}  // namespace mr

using namespace mr::cache;

extern "C" int mr_append_rotated(mr_context *ctx, const mr_array *query, const mr_array *keys, const mr_array *values,
                                 const mr_array *key_pages, const mr_array *value_pages, const mr_array *page_table,
                                 const mr_array *lengths, const mr_array *offsets, const mr_array *frequencies,
                                 const mr_array *positions, const mr_array *out, int split_half) {
    MR_CHECK(check_rows(keys, values, key_pages, value_pages, page_table, lengths, offsets, false));
    const int64_t tokens = keys->shape[0], dim = keys->shape[2];
    MR_REQUIRE(!query == !out, "query and out go together");
    if (query) {
        MR_CHECK(check_array(query, "query", 3, true, false));
        MR_CHECK(check_array(out, "out", 3, true, true));
        MR_REQUIRE(query->dtype == keys->dtype && out->dtype == keys->dtype, "query, out and keys must be of one type");
        for (int i = 0; i < 3; ++i) MR_REQUIRE(query->shape[i] == out->shape[i], "query and out differ in shape");
        MR_REQUIRE(query->shape[0] == tokens && query->shape[2] == dim, "query must be [%lld, heads, %lld], as keys",
                   static_cast<long long>(tokens), static_cast<long long>(dim));
        MR_REQUIRE(query->shape[1] * dim <= INT32_MAX / 4, "too many heads");
        MR_CHECK(check_apart(query, "query", out, "out"));
    }
    if (frequencies) {
        MR_CHECK(check_array(frequencies, "frequencies", 1, false, false));
        MR_REQUIRE(frequencies->dtype == MR_DTYPE_F32, "frequencies must be float32");
        MR_REQUIRE(frequencies->shape[0] <= dim / 2, "frequencies must be at most half of the %lld dims",
                   static_cast<long long>(dim));
    }
    if (positions) {
        MR_CHECK(check_ints(positions, "positions", 1));
        MR_REQUIRE(positions->shape[0] == tokens, "positions must have %lld values", static_cast<long long>(tokens));
    }
    MR_REQUIRE(ctx, "ctx is NULL");
    MR_CHECK(mr::check_waits(ctx));
    if (!tokens || !lengths->shape[0]) return MR_OK;
    DeviceGuard guard(ctx->device);
    RotateArgs a = {};
    a.k = make_rows(keys);
    a.v = make_rows(values);
    if (query) {
        a.q = make_rows(query);
        a.out = make_rows(out);
        a.heads = static_cast<int>(query->shape[1]);
    }
    a.key_pool = make_pool(key_pages);
    a.value_pool = make_pool(value_pages);
    a.pages = make_pages(key_pages, page_table);
    a.place = make_place(lengths, offsets);
    if (frequencies) {
        a.frequencies = static_cast<const float *>(frequencies->data);
        a.frequency_stride = frequencies->stride[0];
        a.half = static_cast<int>(frequencies->shape[0]);
    }
    a.positions = positions ? static_cast<const int *>(positions->data) : nullptr;
    a.position_stride = positions ? positions->stride[0] : 0;
    a.tokens = static_cast<int>(tokens);
    a.kv_heads = static_cast<int>(keys->shape[1]);
    a.dim = static_cast<int>(dim);
    const bool packed = key_pages->dtype == MR_DTYPE_U8;
    return keys->dtype == MR_DTYPE_F32   ? launch_rotated<float>(ctx, a, split_half != 0, packed)
           : keys->dtype == MR_DTYPE_F16 ? launch_rotated<__half>(ctx, a, split_half != 0, packed)
                                         : launch_rotated<__nv_bfloat16>(ctx, a, split_half != 0, packed);
}

extern "C" int mr_read_pages(mr_context *ctx, const mr_array *key_pages, const mr_array *value_pages,
                             const mr_array *page_table, const mr_array *lengths, const mr_array *offsets,
                             const mr_array *keys, const mr_array *values) {
    MR_CHECK(check_rows(keys, values, key_pages, value_pages, page_table, lengths, offsets, true));
    MR_CHECK(check_apart(keys, "keys", values, "values"));
    MR_REQUIRE(ctx, "ctx is NULL");
    MR_CHECK(mr::check_waits(ctx));
    const int64_t tokens = keys->shape[0];
    if (!tokens || !lengths->shape[0]) return MR_OK;
    DeviceGuard guard(ctx->device);
    ReadArgs a;
    a.k = make_rows(keys);
    a.v = make_rows(values);
    a.key_pool = make_pool(key_pages);
    a.value_pool = make_pool(value_pages);
    a.pages = make_pages(key_pages, page_table);
    a.place = make_place(lengths, offsets);
    a.tokens = static_cast<int>(tokens);
    a.heads = static_cast<int>(keys->shape[1]);
    a.pieces = static_cast<int>(keys->shape[2] * dtype_bytes(keys->dtype) / 16);
    a.code_bytes = static_cast<int>(keys->shape[2] / 2);
    // Few tokens: warps share a row.  Else as many tokens to a warp as make about 128 pieces of each pool.
    const int pieces = a.heads * a.pieces;
    const bool few = a.tokens < 4 * ctx->sm_count;
    a.team = few ? std::max(1, std::min(8, pieces / 128)) : 1;
    a.share = few ? 1 : std::max(1, std::min(32, 128 / pieces));
    const int64_t all = (tokens + a.share - 1) / a.share * a.team;
    constexpr int kWarps = 8;
    const unsigned grid = static_cast<unsigned>((all + kWarps - 1) / kWarps);
    auto run = [&](auto kernel) { kernel<<<grid, kWarps * 32, 0, ctx->stream>>>(a); };
    if (key_pages->dtype != MR_DTYPE_U8) run(k_read_pages<float, false>);  // 16-byte pieces of any type
    else if (keys->dtype == MR_DTYPE_F32) run(k_read_pages<float, true>);
    else if (keys->dtype == MR_DTYPE_F16) run(k_read_pages<__half, true>);
    else run(k_read_pages<__nv_bfloat16, true>);
    MR_CUDA_TRY(cudaGetLastError());
    return MR_OK;
}
