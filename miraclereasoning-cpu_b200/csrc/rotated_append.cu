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
#include <type_traits>

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

// Where packed token i stands; the same in all lanes of a warp, which look for it together.
struct Place {
    int sequence;  // -1: of none
    int end;       // behind its last token
    int row;       // of token i there; may lie before the first
    int rows;
    // The last s with offsets[s] <= i, 32 at a time, if its end is behind i.
    __device__ __forceinline__ void find(const PlaceArgs &a, int i) {
        if (!a.offsets) {
            sequence = i;
            end = i + 1;
        } else {
            const int lane = threadIdx.x % 32;
            int lo = 0, n = a.batch + 1;  // it is among lo .. lo + n - 1
            sequence = -1;
            end = i;
            do {
                const int step = (n - 1) / 32 + 1, at = lane * step;
                const bool under = at < n && __ldg(a.offsets + (lo + at) * a.offset_stride) <= i;
                const uint32_t found = __ballot_sync(0xffffffffu, under);
                if (!found) return;
                const int k = 31 - __clz(found);
                lo += k * step;
                n = min(step, n - k * step);
            } while (n > 1);
            if (lo == a.batch) return;
            const int last = __ldg(a.offsets + (lo + 1) * a.offset_stride);
            if (last <= i) return;
            sequence = lo;
            end = last;
        }
        rows = max(0, __ldg(a.lengths + sequence * a.length_stride));
        row = rows - (end - i);
    }
    // The same of a later token.
    __device__ __forceinline__ void next(const PlaceArgs &a, int i) {
        if (sequence >= 0 && i < end) row = rows - (end - i);
        else find(a, i);
    }
};

// 16 bytes of a row: its values as float32, and back.
template <typename T>
struct Vector {
    static constexpr int kValues = 16 / sizeof(T);
    static __device__ __forceinline__ void widen(const uint4 &raw, float (&x)[kValues]) {
        union {
            uint4 raw;
            T v[kValues];
        } u;
        u.raw = raw;
#pragma unroll
        for (int j = 0; j < kValues; ++j) x[j] = cache::widen(&u.v[j]);
    }
    static __device__ __forceinline__ uint4 narrow(const float (&x)[kValues]) {
        union {
            uint4 raw;
            T v[kValues];
        } u;
#pragma unroll
        for (int j = 0; j < kValues; ++j) cache::narrow(x[j], &u.v[j]);
        return u.raw;
    }
};

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

// A lane's V values of a row as codes, and with the other lanes that have the same 32 their step and base (in
// the low and the high half).  The code is rint((x - base) / step) - 64 of float32 operations: a product with
// the step's inverse is off by 2^-16 of a step at most, and where that could round the other way the lane divides.
template <int V>
__device__ __forceinline__ uint32_t quantise(const float (&x)[V], uint32_t &pair) {
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int j = 1; j < V; ++j) {
        lo = min_nan(lo, x[j]);
        hi = max_nan(hi, x[j]);
    }
#pragma unroll
    for (int o = 1; o < kShared / V; o <<= 1) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const __half step = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f));
    const float s = __half2float(step);
    const __half zero = __float2half_rn(__fsub_rn(lo, __fmul_rn(64.f, s)));
    const float z = __half2float(zero);
    const bool held = fabsf(s) < INFINITY && fabsf(z) < INFINITY;
    pair = held ? __half_as_ushort(step) | static_cast<uint32_t>(__half_as_ushort(zero)) << 16 : 0x7e007e00u;
    if (!held || s == 0.f) return 0;
    constexpr float kRound = 12582912.f;  // 1.5 x 2^23: added, it leaves a whole number in the low bits
    const float inverse = __frcp_rn(s);
    uint32_t codes = 0;
    float worst = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float q = fminf(fmaxf(__fmul_rn(__fsub_rn(x[j], z), inverse), 64.f), 79.f);
        const float n = __fadd_rn(q, kRound);
        worst = fmaxf(worst, fabsf(q - (n - kRound)));
        codes |= (__float_as_uint(n) & 15u) << (4 * j);
    }
    if (worst > 0.5f - 0x1p-12f) {
        codes = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float n = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[j], z), s)), 64.f), 79.f);
            codes |= (static_cast<uint32_t>(n) & 15u) << (4 * j);
        }
    }
    return codes;
}

// sin and cos of position * frequency, each rounded to float32 once.  The product is kept in
// two parts and reduced by multiples of pi / 2 in 64 bits, so that far positions lose nothing
// (2^31 radians leave 2^-70); what is left, at most pi / 4, goes through the Taylor series to
// x^15 and x^16, whose next terms are below 5e-17.  One angle is about 25 64-bit operations.
// Past 2^47 radians the product's second part shows in what is left: 1.1 at 2^50, where the series ends at
// 8e-15, still far below a rounding; from 2^54 on results are wrong.
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
    int wide;                                // lanes of a row, as a power of 2
    int query_slots, kv_slots;               // slots of a token's queries, and of its keys or values
    bool split;                              // pairs are p and p + half
    int team, share;                         // warps that share a token's rows, tokens of such a team
};

__device__ __forceinline__ uint4 shared16(uint32_t address) {
    uint4 x;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(address) : "memory");
    return x;
}

// How pairs lie: neighbours, or p and p + half, a lane's dims all turning alike (2 half, or half, a multiple of
// their number); else either, looked at dim by dim, partners of halves read one value at a time (9214 tokens of
// 16 / 4 float16 heads of 64: halves 18.5 us, of 62 dims 28.1; neighbours 15.4 and 19.7).
enum { kNeighbours, kHalves, kAny };

// A warp takes `share` tokens, or a part of one token's rows, in slots of as many rows of one kind (queries,
// then keys, then values) as its lanes hold at 16 bytes each, copied to its ring in shared memory kDepth - 1
// slots ahead, of later tokens too, whether or not they have a place.  A lane has the same dims of every row,
// so that a token's sines, worked out by the warp once, stay in registers.  Products and sums of a turn are
// rounded one by one, so that a 4-bit code is the same wherever it is worked out.
//
// A CTA is a warp: what is the same in all its lanes is worked out once, and 32 of them an SM have the
// registers that they need.  Bound by memory and instructions alike: 9 ragged prompts of 16 / 4 heads of 128 (8290
// tokens, 102 MB) 21.0 us, 4.9 TB/s; loads straight to registers, three slots ahead, took 30 whatever the
// order, and divisions in place of the shifts 1.1 us; the sines are 1.8 us, two or more warps a token 7 us each more,
// and turns and codes by two operations an instruction took 0.4 us more.  Issue slots are 70% busy.  24 sequences of 16 / 4 split-half heads of 64 (9200 tokens,
// 57 MB) 18 us, where what a token costs once (its place, its sines) is a third of the instructions.
template <typename T, int PAIRS, bool PACKED>
__global__ void __launch_bounds__(32, 32) k_append_rotated(const __grid_constant__ RotateArgs a) {
    constexpr int V = Vector<T>::kValues, kDepth = 6, kTurns = PAIRS == kNeighbours ? V / 2 : V;
    __shared__ float2 turns[kMaxDim / 2];
    __shared__ uint4 ring_of[kDepth][32];
    const int lane = threadIdx.x, warp = blockIdx.x;
    const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(ring_of));
    const int unit = a.team == 1 ? warp : warp / a.team, part = warp - unit * a.team;
    const int64_t first = static_cast<int64_t>(unit) * a.share;
    if (first >= a.tokens) return;
    const int sub = lane >> a.wide, piece = lane - (sub << a.wide), d = piece * V, per = 32 >> a.wide, stride = per * a.team;
    const bool inside = d < a.dim, low = d < a.half;
    const bool turning = PAIRS == kAny ? a.half > 0 : d < 2 * a.half;  // this lane's dims
    const int half_bytes = a.half / V * 16;                            // in the ring
    const int lane_bytes = piece * 16;
    const int tokens = static_cast<int>(min(static_cast<int64_t>(a.share), a.tokens - first));
    // The slots of all kinds are dealt out to the team's warps in one row; the first row of each kind that is this warp's.
    auto first_of = [&](int before) { return a.team == 1 ? 0 : (part + a.team - before % a.team) % a.team * per; };
    const int query0 = part * per, key0 = first_of(a.query_slots), value0 = first_of(a.query_slots + a.kv_slots);
    // Copies run through the same slots ahead: a kind's next row of this lane, how many rows are behind it, and where.
    const char *copy_from = nullptr;
    int64_t copy_step = 0;
    int copy_rows = 0, copy_kind = -1, copy_token = static_cast<int>(first);
    const int end_token = copy_token + tokens;
    const uint32_t ring_lane = ring + lane * 16;
    auto copy = [&](int at) {
        while (copy_rows <= 0 && copy_token < end_token) {
            if (++copy_kind == 3) {
                copy_kind = 0;
                if (++copy_token == end_token) break;
            }
            const Rows &rows = copy_kind == 0 ? a.q : copy_kind == 1 ? a.k : a.v;
            const int row = copy_kind == 0 ? query0 : copy_kind == 1 ? key0 : value0;
            copy_rows = (copy_kind == 0 ? a.heads : a.kv_heads) - row;
            copy_from = rows.base + lane_bytes + copy_token * rows.token + (row + sub) * rows.head;
            copy_step = stride * rows.head;
        }
        if (copy_rows > 0) {
            const bool there = inside && sub < copy_rows;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ring_lane + at * 512),
                         "l"(there ? copy_from : a.k.base), "r"(there ? 16 : 0)
                         : "memory");
            copy_from += copy_step;
            copy_rows -= stride;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll 1
    for (int f = 0; f < kDepth - 1; ++f) copy(f);
    int at = 0;
    Place place;
#pragma unroll 1
    for (int n = 0; n < tokens; ++n) {
        const int token = static_cast<int>(first) + n;
        // copies are under way while the place is looked up
        if (n) place.next(a.place, token);
        else place.find(a.place, token);
        const bool owned = place.sequence >= 0;
        const int position = !owned ? 0 : a.positions ? __ldg(a.positions + token * a.position_stride) : place.row;
        char *to_k = nullptr, *to_v = nullptr;
        if (owned && place.row >= 0) {
            const int64_t rk = a.pages.row(place.sequence, place.row, a.key_pool.page, a.key_pool.row);
            const int64_t rv = a.pages.row(place.sequence, place.row, a.value_pool.page, a.value_pool.row);
            if (rk >= 0) {  // both or neither
                to_k = a.key_pool.base + rk;
                to_v = a.value_pool.base + rv;
            }
        }
        // the token's sines
        __syncwarp();  // those of the token before have been read
#pragma unroll 1
        for (int p = lane; p < a.half; p += 32) turns[p] = turn_of(position, __ldg(a.frequencies + p * a.frequency_stride));
        __syncwarp();
        float2 turn[kTurns];
#pragma unroll
        for (int j = 0; j < kTurns; ++j) {
            const int e = d + j, p = PAIRS == kNeighbours ? d / 2 + j : PAIRS == kAny && !a.split ? e / 2 : e < a.half ? e : e - a.half;
            turn[j] = p < a.half ? turns[p] : make_float2(1.f, 0.f);
            if (PAIRS == kHalves && low) turn[j].y = -turn[j].y;  // a cos - b sin as a sum, the same
        }
        // one kind's slots: rows row0, + stride, .. of `count`, to `to` (not written where that is NULL)
        auto work = [&](auto kind, int row0, int count, const Rows &from, char *to, int64_t head) {
            constexpr int kKind = decltype(kind)::value;
            char *dst = to + (row0 + sub) * head;
            const int64_t step = stride * head;
#pragma unroll 1
            for (int rows = count - row0; rows > 0; rows -= stride, dst += step) {
                asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 2) : "memory");
                __syncwarp();  // every lane's copy of the slot has landed, and all are done with the one before it
                copy(at == 0 ? kDepth - 1 : at - 1);
                const uint32_t here = ring_lane + at * 512;
                at = at == kDepth - 1 ? 0 : at + 1;
                const bool there = to && inside && sub < rows;
                float x[V];
                Vector<T>::widen(shared16(here), x);
                if (kKind < 2 && turning) {
                    float y[V], z[V];
                    if (PAIRS == kHalves) {
                        Vector<T>::widen(shared16(low ? here + half_bytes : here - half_bytes), y);
                    } else if (PAIRS == kAny) {
                        const T *row = reinterpret_cast<const T *>(from.base + token * from.token + (count - rows + sub) * from.head);
#pragma unroll
                        for (int j = 0; j < V; ++j) {
                            const int e = d + j, other = e < a.half ? e + a.half : e - a.half;
                            y[j] = !a.split ? x[j ^ 1] : there && e < 2 * a.half ? widen(row + other) : 0.f;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float2 t = turn[PAIRS == kNeighbours ? j / 2 : j];
                        const float p = __fmul_rn(x[j], t.x), q = __fmul_rn(PAIRS == kNeighbours ? x[j ^ 1] : y[j], t.y);
                        const bool second = PAIRS == kAny && a.split ? d + j >= a.half : j & 1;
                        z[j] = PAIRS == kHalves || second ? __fadd_rn(p, q) : __fsub_rn(p, q);
                    }
#pragma unroll
                    for (int j = 0; j < V; ++j)
                        if (PAIRS != kAny || d + j < 2 * a.half) x[j] = z[j];
                }
                if (kKind == 0 || !PACKED) {
                    if (there) *reinterpret_cast<uint4 *>(dst + lane_bytes) = Vector<T>::narrow(x);
                } else {
                    uint32_t pair;
                    const uint32_t codes = quantise<V>(x, pair);
                    if (there) {
                        if (V == 8) *reinterpret_cast<uint32_t *>(dst + d / 2) = codes;
                        else *reinterpret_cast<uint16_t *>(dst + d / 2) = static_cast<uint16_t>(codes);
                        if (d % kShared == 0) *reinterpret_cast<uint32_t *>(dst + a.dim / 2 + d / kShared * 4) = pair;
                    }
                }
            }
        };
        work(std::integral_constant<int, 0>(), query0, a.heads, a.q, owned ? a.out.base + token * a.out.token : nullptr, a.out.head);
        work(std::integral_constant<int, 1>(), key0, a.kv_heads, a.k, to_k, a.key_pool.head);
        work(std::integral_constant<int, 2>(), value0, a.kv_heads, a.v, to_v, a.value_pool.head);
    }
}

// Lanes of a row of n 16-byte pieces, as a power of 2.
int lanes_of(int64_t n) {
    int wide = 0;
    while (1 << wide < n) ++wide;
    return wide;
}

template <typename T, bool PACKED>
int launch_pairs(mr_context *ctx, RotateArgs &a, bool split_half) {
    constexpr int V = Vector<T>::kValues;
    // As many warps to a token as fill the GPU (16 to an SM) when tokens are few; one, with several tokens
    // one after the other, when they are many.
    a.wide = lanes_of(a.dim / V);
    const int per = 32 >> a.wide;
    a.query_slots = (a.heads + per - 1) / per;
    a.kv_slots = (a.kv_heads + per - 1) / per;
    const int slots = a.query_slots + 2 * a.kv_slots;
    const int64_t warps = 16 * static_cast<int64_t>(ctx->sm_count);
    a.team = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(slots, warps / a.tokens)));
    a.share = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(4, a.tokens / (4 * warps))));
    const int64_t all = (static_cast<int64_t>(a.tokens) + a.share - 1) / a.share * a.team;
    auto run = [&](auto kernel) { kernel<<<static_cast<unsigned>(all), 32, 0, ctx->stream>>>(a); };
    a.split = split_half;
    if (!split_half && 2 * a.half % V == 0) run(k_append_rotated<T, kNeighbours, PACKED>);
    else if (split_half && a.half % V == 0) run(k_append_rotated<T, kHalves, PACKED>);
    else run(k_append_rotated<T, kAny, PACKED>);
    MR_CUDA_TRY(cudaGetLastError());
    return MR_OK;
}
template <typename T>
int launch_rotated(mr_context *ctx, RotateArgs &a, bool split_half, bool packed) {
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
    int wide, team, share;      // as in RotateArgs
};

// 16 bytes of a result's row, from piece c of a pool's row.
template <typename T, bool PACKED>
struct Piece {
    enum { V = 16 / sizeof(T) };
    using Raw = std::conditional_t<PACKED, uint2, uint4>;  // PACKED: x: the codes, y: step and base
    Raw raw;
    __device__ __forceinline__ void load(const char *row, int c, int code_bytes) {
        if constexpr (!PACKED) {
            raw = *reinterpret_cast<const uint4 *>(row + 16 * c);
        } else {
            raw.x = V == 8 ? *reinterpret_cast<const uint32_t *>(row + 4 * c) : *reinterpret_cast<const uint16_t *>(row + 2 * c);
            raw.y = *reinterpret_cast<const uint32_t *>(row + code_bytes + c * V / kShared * 4);
        }
    }
    __device__ __forceinline__ uint4 value() const {
        if constexpr (!PACKED) {
            return raw;
        } else {
            const __half2 pair = *reinterpret_cast<const __half2 *>(&raw.y);
            const __half2 s = __low2half2(pair), z = __high2half2(pair);
            if constexpr (V == 8) {
                uint32_t x[4];  // values j and j + 4
                word_codes(raw.x, x);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = fma2(x[j], s, z);
                const uint4 y = make_uint4(__byte_perm(x[0], x[1], 0x5410), __byte_perm(x[2], x[3], 0x5410),
                                           __byte_perm(x[0], x[1], 0x7632), __byte_perm(x[2], x[3], 0x7632));
                if constexpr (std::is_same<T, __half>::value) return y;
                float f[8];
                Vector<__half>::widen(y, f);
                return Vector<T>::narrow(f);
            } else {
                // codes 0 and 1, 2 and 3 into bits 4 .. 7 of the two halves
                const uint32_t low = (raw.x & 0xfu) << 4 | (raw.x & 0xf0u) << 16;
                const uint32_t high = (raw.x & 0xf00u) >> 4 | (raw.x & 0xf000u) << 8;
                const uint32_t x = fma2(codes64(low), s, z), y = fma2(codes64(high), s, z);
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&x));
                const float2 g = __half22float2(*reinterpret_cast<const __half2 *>(&y));
                return make_uint4(__float_as_uint(f.x), __float_as_uint(f.y), __float_as_uint(g.x), __float_as_uint(g.y));
            }
        }
    }
};

constexpr int kReadWarps = 4;

// A warp takes tokens, or a part of one token's heads, as in the append, with four rows of keys and of values a lane
// under way.  Bound by memory: 6 ragged sequences of 33 400 rows of 8 heads of 128 from 4 bits to bfloat16 (176 MB)
// 33.5 us, 5.3 TB/s; 43 700 such rows of bfloat16 pages (358 MB) 59 us, 6.1 TB/s, of float32 ones 115 us.
template <typename T, bool PACKED>
__global__ void __launch_bounds__(kReadWarps * 32) k_read_pages(const __grid_constant__ ReadArgs a) {
    constexpr int kFlight = 4;
    const int lane = threadIdx.x % 32, warp = blockIdx.x * kReadWarps + threadIdx.x / 32;
    const int unit = a.team == 1 ? warp : warp / a.team, part = warp - unit * a.team;
    const int64_t first = static_cast<int64_t>(unit) * a.share;
    if (first >= a.tokens) return;
    const int sub = lane >> a.wide, c = lane - (sub << a.wide), per = 32 >> a.wide, stride = per * a.team;
    Place place;
    place.find(a.place, static_cast<int>(first));
    for (int n = 0; n < a.share && first + n < a.tokens; ++n) {
        const int token = static_cast<int>(first) + n;
        if (n) place.next(a.place, token);
        if (place.sequence < 0) continue;
        int64_t k = -1, v = -1;
        if (place.row >= 0) {
            k = a.pages.row(place.sequence, place.row, a.key_pool.page, a.key_pool.row);
            v = a.pages.row(place.sequence, place.row, a.value_pool.page, a.value_pool.row);
        }
        // this lane's next rows
        int h = part * per + sub;
        const char *from_k = a.key_pool.base + k + h * a.key_pool.head, *from_v = a.value_pool.base + v + h * a.value_pool.head;
        char *to_k = a.k.base + token * a.k.token + 16 * c + h * a.k.head, *to_v = a.v.base + token * a.v.token + 16 * c + h * a.v.head;
        if (c >= a.pieces) h = a.heads;
#pragma unroll 1
        while (__any_sync(0xffffffffu, h < a.heads)) {
            Piece<T, PACKED> x[kFlight], y[kFlight];
#pragma unroll
            for (int f = 0; f < kFlight; ++f) {
                x[f].raw = y[f].raw = typename Piece<T, PACKED>::Raw{};  // a row that is not there: zeros, or step and base 0
                if (k >= 0 && h + f * stride < a.heads) {
                    x[f].load(from_k, c, a.code_bytes);
                    y[f].load(from_v, c, a.code_bytes);
                }
                from_k += stride * a.key_pool.head;
                from_v += stride * a.value_pool.head;
            }
#pragma unroll
            for (int f = 0; f < kFlight; ++f) {
                if (h + f * stride < a.heads) {
                    *reinterpret_cast<uint4 *>(to_k) = x[f].value();
                    *reinterpret_cast<uint4 *>(to_v) = y[f].value();
                }
                to_k += stride * a.k.head;
                to_v += stride * a.v.head;
            }
            h += kFlight * stride;
        }
    }
}

// Checks that both operators share: rows of keys and values that stand for pages' rows.
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
        // rows of other tokens and kinds are read before and while turned queries are written
        MR_CHECK(check_apart(query, "query", out, "out"));
        MR_CHECK(check_apart(keys, "keys", out, "out"));
        MR_CHECK(check_apart(values, "values", out, "out"));
        for (const mr_array *pool : {key_pages, value_pages}) MR_CHECK(check_apart(pool, "the pages", out, "out"));
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
    for (const mr_array *pool : {key_pages, value_pages}) {
        MR_CHECK(check_apart(keys, "keys", pool, "the pages"));
        MR_CHECK(check_apart(values, "values", pool, "the pages"));
    }
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
    // as the appends
    a.wide = lanes_of(a.pieces);
    const int per = 32 >> a.wide, slots = (a.heads + per - 1) / per;
    const int64_t warps = 16 * static_cast<int64_t>(ctx->sm_count);
    a.team = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(slots, warps / tokens)));
    a.share = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(4, tokens / (2 * warps))));
    const int64_t all = (tokens + a.share - 1) / a.share * a.team;
    const unsigned grid = static_cast<unsigned>((all + kReadWarps - 1) / kReadWarps);
    auto run = [&](auto kernel) { kernel<<<grid, kReadWarps * 32, 0, ctx->stream>>>(a); };
    if (key_pages->dtype != MR_DTYPE_U8) run(k_read_pages<float, false>);  // 16-byte pieces of any type
    else if (keys->dtype == MR_DTYPE_F32) run(k_read_pages<float, true>);
    else if (keys->dtype == MR_DTYPE_F16) run(k_read_pages<__half, true>);
    else run(k_read_pages<__nv_bfloat16, true>);
    MR_CUDA_TRY(cudaGetLastError());
    return MR_OK;
}
