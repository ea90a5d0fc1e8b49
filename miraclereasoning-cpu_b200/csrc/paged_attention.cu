// Attention of one new token per sequence over a paged key / value cache.
//
//   s_t = scale q . k_t  over the rows t that the token sees,
//   out = sum_t exp(s_t - max s) v_t / sum_t exp(s_t - max s),
//
// per query head; heads / kv heads query heads read the same key / value rows.
// Every visible row is read once, with about one multiplication per byte, so
// the kernel is bound by memory, and its work is to keep enough rows in flight
// on every SM whatever the lengths are.
//
// Work.  A unit is (sequence, key / value head, block of at most kHeads query
// heads).  Its visible rows, numbered 0 .. without the gap between sinks and
// window, form tiles; the tiles of all units, one after the other, are cut into
// as many even stretches as the grid has CTAs (two an SM, all resident).  So a
// batch of any lengths is balanced to a tile, one long sequence runs on the whole
// GPU, and the host need not know the lengths.  A CTA's stretch holds the end of
// one unit, whole units, and the start of another: whole units are written out,
// the two ends go to scratch as softmax partials (weighted values, maximum, sum),
// and k_join, already resident when the last CTA ends (programmatic dependent
// launch), joins the units that were cut.
//
// Rows.  The warps of a CTA take steps of a tile in turn, each with its own ring
// of row copies (cp.async, 16 bytes a lane, page ids looked up a step ahead) and
// its own running softmax, so nothing in the loop waits for another warp.  The
// partials of the warps meet in shared memory once per unit.
#include <cmath>

#include "cache_ops.cuh"

namespace mr {
namespace cache {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps, kCtasPerSm = 2;
constexpr float kLog2e = 1.4426950408889634f;

struct PagedArgs {
    const char *q, *k, *v;
    char *out;
    int64_t q_batch, q_head, o_batch, o_head;  // bytes
    uint32_t k_page, k_row, v_page, v_row;
    int64_t k_head, v_head;
    Pages pages;
    const int *lengths;
    int64_t length_stride;
    float *weights;  // or NULL
    int64_t w_batch, w_head;
    int batch, kv_heads, group, blocks, dim, capacity, window, sinks;  // blocks: blocks of query heads a group has
    float scale;     // times log2(e): scores are kept as powers of two
    // scratch
    float *partial;  // [CTA][2][kHeads * DP values, kHeads maxima, kHeads sums]
    float *lse;      // [unit][kHeads] of whole units, with weights: log2 of the softmax sum, the maximum in it
    float *scores;   // [unit][seen rows][heads2], with weights
    int64_t seen_max;
    int heads2;      // query heads of a block, rounded up to even
};

// The rows of a sequence that its newest token sees: row i of `seen` is row
// i of the sequence below `sinks`, row i + skip from there on.
struct Seen {
    int rows, sinks, skip;
    __device__ __forceinline__ int at(int i) const { return i < sinks ? i : i + skip; }
};
__device__ __forceinline__ Seen seen_of(const PagedArgs &a, int s) {
    const int n = sequence_rows(a.lengths, a.length_stride, s, a.capacity);
    const int lo = a.window ? max(0, n - a.window) : 0;
    Seen x;
    x.sinks = min(a.sinks, lo);
    x.skip = lo - x.sinks;
    x.rows = n - x.skip;
    return x;
}

// Tiles of all sequences in one row: a sequence's units follow each other, each
// with the sequence's number of tiles.
template <int TILE>
struct Plan {
    int64_t total;
    int units;  // of a sequence
    int ctas;   // that get tiles: at most one each
    // Sum of the sequences' tiles, by every warp on its own.
    __device__ void init(const PagedArgs &a) {
        const int lane = threadIdx.x % 32;
        units = a.kv_heads * a.blocks;
        int64_t sum = 0;
        for (int s = lane; s < a.batch; s += 32) sum += (seen_of(a, s).rows + TILE - 1) / TILE;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        total = sum * units;
        ctas = static_cast<int>(min(total, static_cast<int64_t>(gridDim.x)));
    }
    // First tile of CTA b <= ctas, and the CTA that has tile x: the last b with b total / ctas < x + 1.
    __device__ int64_t start(int b) const { return b * total / ctas; }
    __device__ int cta_of(int64_t x) const { return static_cast<int>(((x + 1) * ctas - 1) / total); }
    // The sequence of tile x (x < total) and its first tile; whole warp.
    __device__ void find(const PagedArgs &a, int64_t x, int &s, int64_t &base) const {
        const int lane = threadIdx.x % 32;
        base = 0;
        for (int s0 = 0;; s0 += 32) {
            int64_t mine = s0 + lane < a.batch ? static_cast<int64_t>((seen_of(a, s0 + lane).rows + TILE - 1) / TILE) * units : 0;
            int64_t sum = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t below = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += below;
            }
            const uint32_t past = __ballot_sync(0xffffffffu, base + sum > x);
            if (past) {
                const int l = __ffs(past) - 1;
                s = s0 + l;
                base += __shfl_sync(0xffffffffu, sum - mine, l);
                return;
            }
            base += __shfl_sync(0xffffffffu, sum, 31);
        }
    }
};

// Walks a CTA's stretch of tiles unit by unit.
template <int TILE>
struct Walk {
    Plan<TILE> plan;
    int64_t x, end, base;  // next tile, end of the stretch, first tile of the sequence
    int s, tiles;          // sequence, tiles of each of its units
    Seen seen;
    __device__ bool init(const PagedArgs &a) {
        plan.init(a);
        if (static_cast<int>(blockIdx.x) >= plan.ctas) return false;
        x = plan.start(blockIdx.x);
        end = plan.start(blockIdx.x + 1);
        plan.find(a, x, s, base);
        load(a);
        return true;
    }
    __device__ void load(const PagedArgs &a) {
        seen = seen_of(a, s);
        tiles = (seen.rows + TILE - 1) / TILE;
    }
    // The next piece: unit u of sequence s, tiles t0 .. t1 - 1.  False behind the last.
    __device__ bool next(const PagedArgs &a, int &u, int &t0, int &t1) {
        if (x >= end) return false;
        while (x >= base + static_cast<int64_t>(tiles) * plan.units) {
            base += static_cast<int64_t>(tiles) * plan.units;
            ++s;
            load(a);
        }
        u = static_cast<int>((x - base) / tiles);
        t0 = static_cast<int>((x - base) - static_cast<int64_t>(u) * tiles);
        t1 = static_cast<int>(min(static_cast<int64_t>(tiles), t0 + (end - x)));
        x += t1 - t0;
        return true;
    }
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t shared_address(const void *p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
// 16 bytes from global to shared memory; zeros without reading where `live` is false.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldmatrix(uint32_t (&r)[4], uint32_t address) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(address));
}
__device__ __forceinline__ void ldmatrix_t(uint32_t (&r)[4], uint32_t address) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(address));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack2(float x, float y, __nv_bfloat16) {
    __nv_bfloat162 p = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<uint32_t *>(&p);
}
__device__ __forceinline__ uint32_t pack2(float x, float y, __half) {
    __half2 p = __floats2half2_rn(x, y);
    return *reinterpret_cast<uint32_t *>(&p);
}
__device__ __forceinline__ float2 unpack2(uint32_t p, __nv_bfloat16) {
    return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162 *>(&p));
}
__device__ __forceinline__ float2 unpack2(uint32_t p, __half) { return __half22float2(*reinterpret_cast<__half2 *>(&p)); }

// log2 of a softmax's denominator; rows of no weight at all get none from it.
__device__ __forceinline__ float log_sum(float top, float sum) { return sum == 0.f ? INFINITY : top + log2f(sum); }

// A running softmax's maximum and sum, and one column's value.
struct Partial {
    float top, sum, x;
    __device__ __forceinline__ void add(float t, float s, float v) {
        const float m = fmaxf(top, t), ref = m == -INFINITY ? 0.f : m;
        const float c = ex2(top - ref), d = ex2(t - ref);
        sum = fmaf(s, d, sum * c);
        x = fmaf(v, d, x * c);
        top = m;
    }
};

// A warp's ring of steps: STEP rows of keys, then of values, DP values a row
// (rows of fewer end in zeros), the 16-byte pieces of a row permuted by its number
// so that eight rows' pieces lie in different banks.
template <typename T, int DP, int STEP, int STAGES>
struct Ring {
    static constexpr int kPieces = DP * sizeof(T) / 16, kRowBytes = DP * sizeof(T);
    static constexpr int kBytes = 2 * STEP * kRowBytes;  // a stage
    static constexpr int kWarpBytes = kBytes * STAGES;
    static __device__ __forceinline__ uint32_t offset(int row, int piece) {
        const int swap = kPieces >= 8 ? row & 7 : (row >> 1) & 3;  // at least 4 pieces a row
        return row * kRowBytes + ((piece ^ swap) << 4);
    }
};

// What a lane looks up for a step: the page of row `lane` of the step and its place there.
struct Place {
    int id, row;  // id -1: hidden
};

// The two ways to work on a step.  Each keeps, per warp, kHeads running maxima
// and sums and weighted values; lanes hold them as the comments say.

// 16-bit types, on the tensor cores: S^T = K Q^T and O^T += V^T P^T with rows (keys,
// then dims) as the 16-high side and up to 8 query heads as the 8-wide side, so that a
// group of 1 to 8 heads costs the same: 2 DP / 16 x 3 small products for 16 rows of
// 2 KB (DP 128), well below what mma.sync can do in the time the rows take to arrive.
// (tcgen05 would want 128 query rows; there are at most 8.)
template <typename T, int DP_>
struct Math16 {
    static constexpr int DP = DP_, kHeads = 8, STEP = DP == 128 ? 16 : 32, STAGES = DP == 32 ? 6 : 3;
    using R = Ring<T, DP, STEP, STAGES>;
    uint32_t qf[DP / 16][2];   // Q^T fragments: head lane / 4
    float o[DP / 16][4];       // O^T: dims 16 b + lane / 4 (+ 8), heads 2 (lane % 4) and + 1
    float m[2], l[2];          // heads 2 (lane % 4), + 1; l only of this lane's rows
    bool fine;                 // weights in two parts

    __device__ __forceinline__ void begin(const PagedArgs &a, const char *q, int heads, bool two_parts) {
        const int lane = threadIdx.x % 32, h = lane / 4;
        fine = two_parts;
#pragma unroll
        for (int b = 0; b < DP / 16; ++b) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int j = b * 16 + e * 8 + 2 * (lane % 4);
                qf[b][e] = h < heads && j < a.dim ? __ldg(reinterpret_cast<const uint32_t *>(q + h * a.q_head + j * 2)) : 0u;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) o[b][e] = 0.f;
        }
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
    }

    // One step: rows in `stage` (keys, then values), bit r of `live`: row r is seen.
    __device__ __forceinline__ void step(const PagedArgs &a, uint32_t stage, uint32_t live, float *scores) {
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
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int x = 0; x < S; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool seen = (live >> (x * 16 + lane / 4 + (e >> 1) * 8)) & 1u;
                s[x][e] = seen ? s[x][e] * a.scale : -INFINITY;
                top[e & 1] = fmaxf(top[e & 1], s[x][e]);
            }
        if (scores) {
            const int h = 2 * (lane % 4);
#pragma unroll
            for (int x = 0; x < 2 * S; ++x) {
                const int r = x * 8 + lane / 4;
                if (h < a.heads2 && (live >> r) & 1u)
                    *reinterpret_cast<float2 *>(scores + r * a.heads2 + h) = make_float2(s[x / 2][(x & 1) * 2], s[x / 2][(x & 1) * 2 + 1]);
            }
        }
        float ref[2];
        bool grown = false;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 4; i < 32; i <<= 1) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], i));
            top[h] = fmaxf(top[h], m[h]);
            grown |= top[h] > m[h];
            ref[h] = top[h] == -INFINITY ? 0.f : top[h];
        }
        if (__any_sync(0xffffffffu, grown)) {
            const float c0 = ex2(m[0] - ref[0]), c1 = ex2(m[1] - ref[1]);
            l[0] *= c0;
            l[1] *= c1;
#pragma unroll
            for (int b = 0; b < DP / 16; ++b) {
                o[b][0] *= c0;
                o[b][1] *= c1;
                o[b][2] *= c0;
                o[b][3] *= c1;
            }
            m[0] = top[0];
            m[1] = top[1];
        }
#pragma unroll
        for (int x = 0; x < S; ++x) {
            float p[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                p[e] = ex2(s[x][e] - ref[e & 1]);
                l[e & 1] += p[e];
            }
            // the weights as the 16-bit operand, and what that rounding left (a second
            // product): one part alone would add as much error again as the output's rounding
            const uint32_t h0 = pack2(p[0], p[1], T()), h1 = pack2(p[2], p[3], T());
            const float2 r0 = unpack2(h0, T()), r1 = unpack2(h1, T());
            const uint32_t b0 = transposed(h0), b1 = transposed(h1);
            const uint32_t c0 = transposed(pack2(p[0] - r0.x, p[1] - r0.y, T()));
            const uint32_t c1 = transposed(pack2(p[2] - r1.x, p[3] - r1.y, T()));
#pragma unroll
            for (int b = 0; b < DP / 16; ++b) {
                uint32_t v[4];
                ldmatrix_t(v, stage + STEP * R::kRowBytes +
                                  R::offset(x * 16 + lane % 8 + (lane / 16) * 8, b * 2 + ((lane / 8) & 1)));
                mma16(o[b], v, b0, b1, T());
                if (fine) mma16(o[b], v, c0, c1, T());
            }
        }
    }

    // The warp's results: values [head][DP + 4], then maxima and sums.  False if a value is not finite.
    __device__ __forceinline__ bool finish(float *values, float *maxima, float *sums) {
        const int lane = threadIdx.x % 32, h = 2 * (lane % 4);
        bool finite = true;
#pragma unroll
        for (int b = 0; b < DP / 16; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                finite &= fabsf(o[b][e]) < INFINITY;
                values[(h + (e & 1)) * (DP + 4) + b * 16 + lane / 4 + (e >> 1) * 8] = o[b][e];
            }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float sum = l[e];
#pragma unroll
            for (int i = 4; i < 32; i <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
            if (lane < 4) {
                maxima[h + e] = m[e];
                sums[h + e] = sum;
            }
        }
        return finite;
    }
};

// float32 on the CUDA cores: DP / 4 lanes share a row, four values each, and keep the
// same four dims of up to 4 query heads and of their weighted values in registers; the
// 8 rows x 4 heads of a step give 32 sums, folded so that each lane ends with one.
template <int DP_>
struct Math32 {
    static constexpr int DP = DP_, kHeads = 4, STEP = 8, STAGES = DP == 128 ? 3 : DP == 64 ? 6 : 8;
    static constexpr int kLanes = DP / 4, kRows = 32 / kLanes, kEach = STEP / kRows;  // lanes a row, rows at a time
    using R = Ring<float, DP, STEP, STAGES>;
    float4 q[4], o[4];
    float m, l;  // head lane % 4; l only of this lane's rows

    __device__ __forceinline__ void begin(const PagedArgs &a, const char *src, int heads, bool) {
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
    __device__ __forceinline__ void step(const PagedArgs &a, uint32_t stage, uint32_t live, float *scores) {
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
        if (scores && head < a.heads2 && (live >> row) & 1u) scores[row * a.heads2 + head] = x;
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
    __device__ __forceinline__ bool finish(float *values, float *maxima, float *sums) {
        const int lane = threadIdx.x % 32;
#pragma unroll
        for (int h = 0; h < 4; ++h)
#pragma unroll
            for (int w = kLanes; w < 32; w <<= 1) {
                o[h].x += __shfl_xor_sync(0xffffffffu, o[h].x, w);
                o[h].y += __shfl_xor_sync(0xffffffffu, o[h].y, w);
                o[h].z += __shfl_xor_sync(0xffffffffu, o[h].z, w);
                o[h].w += __shfl_xor_sync(0xffffffffu, o[h].w, w);
            }
        if (lane < kLanes)
#pragma unroll
            for (int h = 0; h < 4; ++h) *reinterpret_cast<float4 *>(values + h * (DP + 4) + 4 * lane) = o[h];
        float sum = l;
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        if (lane < 4) {
            maxima[lane] = m;
            sums[lane] = sum;
        }
        return true;
    }
};

// One warp's share of a piece of a unit: rows [from, to) of `seen`, in steps
// warp, warp + kWarps, ...
template <typename M>
__device__ __forceinline__ void walk_rows(const PagedArgs &a, M &math, const Seen &seen, int s, const char *k,
                                          const char *v, int from, int to, uint32_t ring, float *scores) {
    using R = typename M::R;
    constexpr int STEP = M::STEP, STAGES = M::STAGES, kCopies = STEP * R::kPieces / 32;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int steps = (to - from + STEP - 1) / STEP;
    const int *table = a.pages.table + s * a.pages.table_stride;
    const int live_pieces = a.dim * static_cast<int>(R::kRowBytes / M::DP) / 16;
    auto place = [&](int step) {  // of row `lane` of a step
        Place p = {-1, 0};
        const int i = from + step * STEP + lane;
        if (lane < STEP && i < to) {
            const int t = seen.at(i), page = a.pages.page.div(t);
            const int id = __ldg(table + page);
            p.row = t - page * a.pages.page.d;
            p.id = static_cast<unsigned>(id) < static_cast<unsigned>(a.pages.pages) ? id : -1;
        }
        return p;
    };
    auto issue = [&](const Place &p, int slot) {
        const uint32_t stage = ring + slot * R::kBytes;
#pragma unroll
        for (int c = 0; c < kCopies; ++c) {
            const int e = c * 32 + lane, row = e / R::kPieces, piece = e % R::kPieces;
            const int id = __shfl_sync(0xffffffffu, p.id, row), r = __shfl_sync(0xffffffffu, p.row, row);
            const bool live = id >= 0 && piece < live_pieces;
            const uint64_t page = live ? id : 0;
            const uint32_t to_shared = stage + R::offset(row, piece);
            copy16(to_shared, k + (page * a.k_page + static_cast<uint64_t>(r) * a.k_row + piece * 16), live);
            copy16(to_shared + STEP * R::kRowBytes, v + (page * a.v_page + static_cast<uint64_t>(r) * a.v_row + piece * 16), live);
        }
    };
    int step = warp, ahead = warp;
    uint32_t masks[STAGES];
    Place next = place(ahead);
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {
        masks[i] = __ballot_sync(0xffffffffu, next.id >= 0);
        if (ahead < steps) issue(next, i);
        asm volatile("cp.async.commit_group;" ::: "memory");
        ahead += kWarps;
        next = place(ahead);
    }
    while (step < steps) {
#pragma unroll
        for (int i = 0; i < STAGES; ++i) {
            if (step < steps) {
                constexpr int kWait = STAGES - 2;
                asm volatile("cp.async.wait_group %0;" ::"n"(kWait) : "memory");
                __syncwarp();  // every lane's copies of this step have landed, and all are done with the slot refilled next
                const int slot = (i + STAGES - 1) % STAGES;
                masks[slot] = __ballot_sync(0xffffffffu, next.id >= 0);
                if (ahead < steps) issue(next, slot);
                asm volatile("cp.async.commit_group;" ::: "memory");
                ahead += kWarps;
                next = place(ahead);
                math.step(a, ring + i * R::kBytes, masks[i],
                          scores ? scores + static_cast<int64_t>(from + step * STEP) * a.heads2 : nullptr);
                step += kWarps;
            }
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
}

// Results of a unit's piece: dims of the block's heads.
template <typename T, typename M>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) k_paged(PagedArgs a) {
    extern __shared__ __align__(128) char smem[];
    constexpr int H = M::kHeads, DP = M::DP, kValues = H * (DP + 4);
    static_assert((kValues + 2 * H) * 4 <= M::R::kWarpBytes, "a warp's results fit its ring");
    const int tid = threadIdx.x, warp = tid / 32;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // sequences that see nothing give zeros
    for (int s = blockIdx.x; s < a.batch; s += gridDim.x) {
        if (seen_of(a, s).rows > 0) continue;
        const int heads = a.kv_heads * a.group;
        for (int e = tid; e < heads * a.dim; e += kThreads)
            narrow(0.f, reinterpret_cast<T *>(a.out + s * a.o_batch + e / a.dim * a.o_head) + e % a.dim);
    }
    Walk<M::STEP * kWarps> walk;
    if (!walk.init(a)) return;
    int u, t0, t1, slot = 0;
    char *mine = smem + warp * M::R::kWarpBytes;
    while (walk.next(a, u, t0, t1)) {
        const int s = walk.s, kh = u / a.blocks, h0 = u % a.blocks * H, heads = min(H, a.group - h0);
        const int from = t0 * M::STEP * kWarps, to = min(t1 * M::STEP * kWarps, walk.seen.rows);
        const bool whole = t0 == 0 && t1 == walk.tiles;
        const int64_t unit = static_cast<int64_t>(s) * walk.plan.units + u;
        const char *q = a.q + s * a.q_batch + (kh * a.group + h0) * a.q_head;
        float *scores = a.scores ? a.scores + unit * a.seen_max * a.heads2 : nullptr;
        float *values = reinterpret_cast<float *>(mine);
        // An infinite value meets a weight's second part as 0 x inf or inf - inf: such a
        // unit is worked out again with the weights in one part.
        for (int parts = 2; parts > 0; --parts) {
            M math;
            math.begin(a, q, heads, parts == 2);
            walk_rows<M>(a, math, walk.seen, s, a.k + kh * a.k_head, a.v + kh * a.v_head, from, to,
                         shared_address(mine), scores);
            const bool finite = math.finish(values, values + kValues, values + kValues + H);
            if (!__syncthreads_or(!finite)) break;
        }
        // the warps' partials: a column of values a thread at a time
        auto part = [&](int w) { return reinterpret_cast<const float *>(smem + w * M::R::kWarpBytes); };
        for (int e = tid; e < heads * DP; e += kThreads) {
            const int h = e / DP, j = e % DP;
            float top = -INFINITY, sum = 0.f, x = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, part(w)[kValues + h]);
            const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float c = ex2(part(w)[kValues + h] - ref);
                sum = fmaf(part(w)[kValues + H + h], c, sum);
                x = fmaf(part(w)[h * (DP + 4) + j], c, x);
            }
            if (whole) {
                if (j < a.dim)
                    narrow(sum != 0.f ? x / sum : 0.f,
                           reinterpret_cast<T *>(a.out + s * a.o_batch + (kh * a.group + h0 + h) * a.o_head) + j);
                if (j == 0 && a.lse) a.lse[unit * H + h] = log_sum(ref, sum);
            } else {
                float *to_join = a.partial + (blockIdx.x * 2 + slot) * static_cast<int64_t>(H * (DP + 2));
                to_join[h * DP + j] = x;
                if (j == 0) {
                    to_join[H * DP + h] = top;
                    to_join[H * DP + H + h] = sum;
                }
            }
        }
        slot = 1;
        __syncthreads();  // the rings are filled again
    }
}

// Joins the units that were cut: the CTAs whose stretch starts inside a unit
// share its columns.  With weights, every CTA then adds up its own stretch's rows.
template <typename T, typename M>
__global__ void __launch_bounds__(kThreads) k_join(PagedArgs a) {
    constexpr int H = M::kHeads, DP = M::DP, TILE = M::STEP * kWarps;
    constexpr int64_t kPart = H * (DP + 2);
    __shared__ float s_lse[8];
    __shared__ Partial s_part[kThreads];
    Walk<TILE> walk;
    const int tid = threadIdx.x;
    const bool work = walk.init(a);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (!work) return;
    const int64_t x0 = walk.x;
    // the partial of CTA b of the unit whose first tile is `first`
    auto part = [&](int b, int64_t first) {
        return a.partial + (b * 2 + (walk.plan.start(b) >= first ? 0 : 1)) * kPart;
    };
    {
        const int u = static_cast<int>((x0 - walk.base) / walk.tiles);
        const int64_t first = walk.base + static_cast<int64_t>(u) * walk.tiles;
        if (first < x0) {
            const int b0 = walk.plan.cta_of(first), b1 = walk.plan.cta_of(first + walk.tiles - 1);
            const int kh = u / a.blocks, h0 = u % a.blocks * H, heads = min(H, a.group - h0);
            // columns of four values: this CTA's share, each on kThreads / share threads
            const int columns = heads * (DP / 4), share = b1 - b0, me = static_cast<int>(blockIdx.x) - b0 - 1;
            for (int c = me; c < columns; c += share) {
                const int h = c / (DP / 4), j = c % (DP / 4) * 4;
                Partial mine = {-INFINITY, 0.f, 0.f};
                for (int b = b0 + tid / 4; b <= b1; b += kThreads / 4) {
                    const float *p = part(b, first);
                    mine.add(__ldcg(p + H * DP + h), __ldcg(p + H * DP + H + h), __ldcg(p + h * DP + j + tid % 4));
                }
                s_part[tid] = mine;
                __syncthreads();
                for (int w = kThreads / 2; w >= 4; w >>= 1) {
                    if (tid < w) s_part[tid].add(s_part[tid + w].top, s_part[tid + w].sum, s_part[tid + w].x);
                    __syncthreads();
                }
                if (tid < 4 && j + tid < a.dim)
                    narrow(s_part[tid].sum != 0.f ? s_part[tid].x / s_part[tid].sum : 0.f,
                           reinterpret_cast<T *>(a.out + walk.s * a.o_batch + (kh * a.group + h0 + h) * a.o_head) + j + tid);
                __syncthreads();
            }
        }
    }
    if (!a.weights) return;
    int u, t0, t1;
    while (walk.next(a, u, t0, t1)) {
        if (u % a.blocks) continue;  // the group's first block of heads adds up for all of them
        const int s = walk.s, kh = u / a.blocks;
        const int from = t0 * TILE, to = min(t1 * TILE, walk.seen.rows);
        for (int b = 0; b < a.blocks; ++b) {
            const int64_t unit = static_cast<int64_t>(s) * walk.plan.units + u + b;
            const int64_t first = walk.base + static_cast<int64_t>(u + b) * walk.tiles;
            const int heads = min(H, a.group - b * H);
            const int b0 = walk.plan.cta_of(first), b1 = walk.plan.cta_of(first + walk.tiles - 1);
            __syncthreads();
            for (int h = tid / 32; h < heads; h += kWarps) {
                float lse;
                if (b0 == b1) {
                    lse = __ldcg(a.lse + unit * H + h);
                } else {
                    Partial mine = {-INFINITY, 0.f, 0.f};
                    for (int c = b0 + tid % 32; c <= b1; c += 32) {
                        const float *p = part(c, first);
                        mine.add(__ldcg(p + H * DP + h), __ldcg(p + H * DP + H + h), 0.f);
                    }
#pragma unroll
                    for (int w = 16; w > 0; w >>= 1) {
                        const float t = __shfl_xor_sync(0xffffffffu, mine.top, w), l = __shfl_xor_sync(0xffffffffu, mine.sum, w);
                        mine.add(t, l, 0.f);
                    }
                    lse = log_sum(mine.top == -INFINITY ? 0.f : mine.top, mine.sum);
                }
                if (tid % 32 == 0) s_lse[h] = lse;
            }
            __syncthreads();
            const float *scores = a.scores + unit * a.seen_max * a.heads2;
            float *weights = a.weights + s * a.w_batch + kh * a.w_head;
            for (int i = from + tid; i < to; i += kThreads) {
                const int t = walk.seen.at(i);
                if (a.pages.row(s, t, 0, 0) < 0) continue;
                float sum = 0.f;
                for (int h = 0; h < heads; ++h)
                    sum += ex2(__ldcg(scores + static_cast<int64_t>(i) * a.heads2 + h) - s_lse[h]);
                weights[t] += sum;
            }
        }
    }
}

template <typename T, typename M>
int launch(mr_context *ctx, PagedArgs &a) {
    constexpr int H = M::kHeads, TILE = M::STEP * kWarps;
    constexpr int kSmem = kWarps * M::R::kWarpBytes;
    a.blocks = (a.group - 1) / H + 1;
    a.heads2 = (std::min(a.group, H) + 1) / 2 * 2;
    // the most rows a token can see, and the most tiles there can be
    a.seen_max = a.window ? std::min<int64_t>(a.capacity, static_cast<int64_t>(a.window) + a.sinks) : a.capacity;
    const int64_t units = static_cast<int64_t>(a.batch) * a.kv_heads * a.blocks;
    const int64_t tiles = (a.seen_max + TILE - 1) / TILE;
    const int grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(units * tiles, kCtasPerSm * ctx->sm_count)));
    const size_t partial = sizeof(float) * 2 * grid * H * (M::DP + 2);
    const size_t lse = a.weights ? sizeof(float) * units * H : 0;
    const size_t scores = a.weights ? sizeof(float) * units * a.seen_max * a.heads2 : 0;
    auto up = [](size_t n) { return (n + 255) & ~size_t(255); };
    Scratch scratch(ctx);
    // with a tile a unit at most, nothing can be cut
    const bool cut = tiles > 1;
    if (cut || a.weights) MR_CHECK(scratch.take(up(partial) + up(lse) + scores));
    char *base = static_cast<char *>(scratch.data);
    a.partial = reinterpret_cast<float *>(base);
    a.lse = a.weights ? reinterpret_cast<float *>(base + up(partial)) : nullptr;
    a.scores = a.weights ? reinterpret_cast<float *>(base + up(partial) + up(lse)) : nullptr;
    auto kernel = k_paged<T, M>;
    MR_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    kernel<<<grid, kThreads, kSmem, ctx->stream>>>(a);
    MR_CUDA_TRY(cudaGetLastError());
    if (cut || a.weights) {
        cudaLaunchAttribute early;
        early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        early.val.programmaticStreamSerializationAllowed = 1;
        cudaLaunchConfig_t config = {};
        config.gridDim = dim3(grid);
        config.blockDim = dim3(kThreads);
        config.stream = ctx->stream;
        config.attrs = &early;
        config.numAttrs = 1;
        MR_CUDA_TRY(cudaLaunchKernelEx(&config, k_join<T, M>, a));
    }
    return MR_OK;
}

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
    for (const mr_array *pool : {key_pages, value_pages})
        for (int i = 0; i < 2; ++i)
            MR_REQUIRE(pool->stride[i] < (int64_t(1) << 32) / dtype_bytes(pool->dtype),
                       "the pages' stride %d passes 4 GB", i);
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
    a.k_page = static_cast<uint32_t>(key_pages->stride[0] * size);
    a.k_row = static_cast<uint32_t>(key_pages->stride[1] * size);
    a.k_head = key_pages->stride[2] * size;
    a.v_page = static_cast<uint32_t>(value_pages->stride[0] * size);
    a.v_row = static_cast<uint32_t>(value_pages->stride[1] * size);
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
    a.scale = scale * kLog2e;
    return query->dtype == MR_DTYPE_F32   ? launch32(ctx, a)
           : query->dtype == MR_DTYPE_F16 ? launch16<__half>(ctx, a)
                                          : launch16<__nv_bfloat16>(ctx, a);
}
