// One-token attention over a paged key / value cache, for any way to work on a step
// of rows (paged_attention.cu: rows of the query's type, packed_attention.cu: of 4 bits).
//
//   s_t = scale q . k_t  over the rows t that the token sees,
//   out = sum_t exp(s_t - max s) v_t / sum_t exp(s_t - max s),
//
// per query head; heads / kv heads query heads read the same key / value rows.
// Every visible row is read once.  What bounds that is said with the ways to work
// on a step; what they share is to keep enough rows in flight on every SM whatever
// the lengths are.
//
// Work.  A unit is (sequence, key / value head, block of at most kHeads query
// heads).  Its visible rows, numbered 0 .. without the gap between sinks and
// window, form steps of STEP rows; the steps of all units, one after the other,
// are cut into as many even stretches as the grid has warps (four a CTA, of
// which M::ctas() an SM are resident).  So a batch of any lengths is balanced to a step, one long sequence
// runs on the whole GPU, and the host need not know the lengths.  A warp's
// stretch holds the end of one unit, whole units, and the start of another: whole
// units are written out, the two ends go to scratch as softmax partials (weighted
// values, maximum, sum), and k_join (launched early, waiting for this kernel's
// end) joins the units that were cut.
//
// Where no token can see more than kFewSteps steps (a window, a short table), a
// unit is a CTA's instead, a quarter of it each warp's: there is nothing to join
// but the four warps' partials, in shared memory, and the second launch is saved
// (flashnano-1.7's window of 516 rows in a batch of 48: 9.7 us, cut and joined 20.1).
// The host goes by what the table could hold, so tables much longer than their sequences
// lose that: 32 sequences of 500 rows (8 heads of 128 in 4 bits) 11.2 us, in tables for 32768 rows 16.3; with
// weights 13.9 and 23.8.  From 1500 rows on there is little in it (27.3 and 27.9; 33.6 and 38.4).
//
// Rows.  Warps never wait for each other there: each has its own ring of row copies
// (cp.async, R::kUnit bytes a lane: 16, for rows of 4 bits what they are whole
// multiples of; page ids looked up a step ahead), which runs on from one unit into
// the next, and its own running softmax.
#pragma once

#include <cmath>
#include <type_traits>

#include "cache_ops.cuh"

namespace mr {
namespace cache {

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
    float *partial;  // [warp][2][kHeads * DP values]
    float2 *sums;    // [2][kHeads][warps]: their maxima and sums, side by side as k_join reads them
    float *lse;      // [unit][kHeads] of whole units, with weights: log2 of the softmax sum, the maximum in it
    float *scores;   // [unit][seen rows][heads2], with weights
    int64_t seen_max;
    int warps;       // of k_paged
    int heads2;      // query heads of a block, rounded up to even
    int page_shift;  // log2 of the page's rows, -1 if they are no power of 2
};


// On pages of 4 bits (packed_attention.cu): for queries and results of a type.
int launch_packed(mr_context *ctx, PagedArgs &a, int dtype);

namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int64_t kMaxSteps = INT32_MAX / 2;
constexpr int kFewSteps = 32;
constexpr float kLog2e = 1.4426950408889634f;

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

// Steps of all sequences in one row: a sequence's units follow each other, each
// with the sequence's number of steps.
template <int STEP>
struct Plan {
    int total, units;  // units of a sequence
    int workers;       // warps that get steps
    int each, more;    // steps of a worker: each + 1 for the first `more`, then each
    static __device__ __forceinline__ int steps_of(const Seen &seen) { return (seen.rows + STEP - 1) / STEP; }
    __device__ void init(const PagedArgs &a) {
        const int lane = threadIdx.x % 32;
        units = a.kv_heads * a.blocks;
        int sum = 0;
        for (int s = lane; s < a.batch; s += 32) sum += steps_of(seen_of(a, s));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        total = sum * units;
        workers = min(total, a.warps);
        each = total / max(workers, 1);
        more = total - each * workers;
    }
    // First step of worker b <= workers, and the worker that has step x.
    __device__ __forceinline__ int start(int b) const { return b * each + min(b, more); }
    __device__ __forceinline__ int worker_of(int x) const {
        const int longer = more * (each + 1);
        return x < longer ? x / (each + 1) : more + (x - longer) / each;
    }
    // The sequence of step x (x < total) and its first step.
    __device__ void find(const PagedArgs &a, int x, int &s, int &base) const {
        const int lane = threadIdx.x % 32;
        base = 0;
        for (int s0 = 0;; s0 += 32) {
            const int mine = s0 + lane < a.batch ? steps_of(seen_of(a, s0 + lane)) * units : 0;
            int sum = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int below = __shfl_up_sync(0xffffffffu, sum, o);
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

// A piece of work: steps t0 .. t1 - 1 of unit u of sequence s, whose units have `steps` steps each.
struct Piece {
    int s, u, t0, t1, steps;
    Seen seen;
};

// Walks a stretch of steps unit by unit.
struct Walk : Piece {
    int x, end, base;  // next step, end of the stretch, first step of the sequence
    template <int STEP>
    __device__ bool init(const PagedArgs &a, const Plan<STEP> &plan, int worker) {
        if (worker >= plan.workers) return false;
        x = plan.start(worker);
        end = plan.start(worker + 1);
        plan.find(a, x, s, base);
        seen = seen_of(a, s);
        steps = Plan<STEP>::steps_of(seen);
        return true;
    }
    // The next piece; false behind the last.
    template <int STEP>
    __device__ __forceinline__ bool next(const PagedArgs &a, const Plan<STEP> &plan) {
        if (x >= end) return false;
        while (x >= base + steps * plan.units) {
            base += steps * plan.units;
            ++s;
            seen = seen_of(a, s);
            steps = Plan<STEP>::steps_of(seen);
        }
        u = (x - base) / steps;
        t0 = (x - base) - u * steps;
        t1 = min(steps, t0 + (end - x));
        x += t1 - t0;
        return true;
    }
};

// Walks the units of a CTA, a quarter of each.
template <int STEP>
struct Quarters : Piece {
    int unit;  // the next
    __device__ __forceinline__ bool next(const PagedArgs &a) {
        const int units = a.kv_heads * a.blocks;
        if (unit >= a.batch * units) return false;
        s = unit / units;
        u = unit - s * units;
        seen = seen_of(a, s);
        steps = (seen.rows + STEP - 1) / STEP;
        const int warp = threadIdx.x / 32;
        t0 = steps * warp / kWarps;
        t1 = steps * (warp + 1) / kWarps;
        unit += gridDim.x;
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
// 4, 8 or 16 bytes from global to shared memory; zeros without reading where `live` is false.
template <int BYTES>
__device__ __forceinline__ void copy_piece(uint32_t dst, const void *src, bool live) {
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(live ? BYTES : 0), "n"(BYTES)
                     : "memory");
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
    static constexpr int kUnit = 16, kPieces = DP * sizeof(T) / kUnit, kRowBytes = DP * sizeof(T);  // kUnit: bytes of a copy
    static constexpr int kBytes = 2 * STEP * kRowBytes;  // a stage
    static constexpr int kWarpBytes = kBytes * STAGES;
    // pieces of a row that are there
    static __device__ __forceinline__ int pieces(const PagedArgs &a) { return a.dim * static_cast<int>(sizeof(T)) / kUnit; }
    static __device__ __forceinline__ uint32_t offset(int row, int piece) {
        const int swap = kPieces >= 8 ? row & 7 : (row >> 1) & 3;  // at least 4 pieces a row
        return row * kRowBytes + ((piece ^ swap) << 4);
    }
};

// What a lane looks up for a step: the page of row `lane` of the step and its place there.
struct Place {
    int id, row;  // id -1: hidden
};

// Up to 8 query heads' running softmax beside the tensor cores' products S^T = K Q^T and O^T += V^T P^T of
// operands of type T: what lanes hold, between the two.
template <typename T, int TILES>
struct Heads8 {
    // Weights are taken against the maximum / 2^kLift, so that the largest is 2^kLift: float16 ends at 2^-25
    // below, and what is less than 2^-40 of the largest weight is lost instead of 2^-25 (32768 rows of
    // 2^-25.2 beside one: 8e-4 of the sum).  All statistics of a warp are of that reference.
    static constexpr float kLift = std::is_same<T, __half>::value ? 15.f : 0.f;
    float o[TILES][4];  // O^T: rows lane / 4 (+ 8) of each tile, heads 2 (lane % 4) and + 1
    float m[2], l[2];   // heads 2 (lane % 4), + 1: maximum - kLift, sum; l only of this lane's rows

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int b = 0; b < TILES; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[b][e] = 0.f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
    }

    // The products of S x 16 rows: scaled (f0, f1: of the lane's two heads), hidden ones taken out (kAllSeen: after
    // a look whether there are any), kept for the weights; the maxima raised and what is there rescaled.  ref:
    // what weights are taken against.
    template <bool kAllSeen, int S>
    __device__ __forceinline__ void settle(const PagedArgs &a, float (&s)[S][4], float f0, float f1, uint32_t live, int rows,
                                           float *scores, float (&ref)[2]) {
        const int lane = threadIdx.x % 32;
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int x = 0; x < S; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[x][e] *= e & 1 ? f1 : f0;
                if constexpr (!kAllSeen) {
                    const bool seen = (live >> (x * 16 + lane / 4 + (e >> 1) * 8)) & 1u;
                    s[x][e] = seen ? s[x][e] : -INFINITY;
                    top[e & 1] = fmaxf(top[e & 1], s[x][e]);
                }
            }
        if constexpr (kAllSeen) {
            if (live != 0xffffffffu >> (32 - 16 * S)) {
#pragma unroll
                for (int x = 0; x < S; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!((live >> (x * 16 + lane / 4 + (e >> 1) * 8)) & 1u)) s[x][e] = -INFINITY;
            }
#pragma unroll
            for (int x = 0; x < S; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e) top[e & 1] = fmaxf(top[e & 1], s[x][e]);
        }
        if (scores) {
            const int h = 2 * (lane % 4);
#pragma unroll
            for (int x = 0; x < 2 * S; ++x) {
                const int r = x * 8 + lane / 4;
                if (h < a.heads2 && r < rows)
                    *reinterpret_cast<float2 *>(scores + r * a.heads2 + h) = make_float2(s[x / 2][(x & 1) * 2], s[x / 2][(x & 1) * 2 + 1]);
            }
        }
        bool grown = false;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 4; i < 32; i <<= 1) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], i));
            top[h] = fmaxf(top[h] - kLift, m[h]);
            grown |= top[h] > m[h];
            ref[h] = top[h] == -INFINITY ? 0.f : top[h];
        }
        if (__any_sync(0xffffffffu, grown)) {
            const float c0 = ex2(m[0] - ref[0]), c1 = ex2(m[1] - ref[1]);
            l[0] *= c0;
            l[1] *= c1;
#pragma unroll
            for (int b = 0; b < TILES; ++b) {
                o[b][0] *= c0;
                o[b][1] *= c1;
                o[b][2] *= c0;
                o[b][3] *= c1;
            }
            m[0] = top[0];
            m[1] = top[1];
        }
    }
    // The weights of 16 rows as two operands P^T, the first part b0, b1 and what its rounding left c0, c1 (a second
    // product): one part alone would add as much error again as the output's rounding, and an eighth of it where
    // float16 weights make bfloat16 results.
    __device__ __forceinline__ void weigh(const float (&s)[4], const float (&ref)[2], uint32_t &b0, uint32_t &b1, uint32_t &c0,
                                          uint32_t &c1) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            p[e] = ex2(s[e] - ref[e & 1]);
            l[e & 1] += p[e];
        }
        const uint32_t h0 = pack2(p[0], p[1], T()), h1 = pack2(p[2], p[3], T());
        b0 = transposed(h0);
        b1 = transposed(h1);
        const float2 r0 = unpack2(h0, T()), r1 = unpack2(h1, T());
        c0 = transposed(pack2(p[0] - r0.x, p[1] - r0.y, T()));
        c1 = transposed(pack2(p[2] - r1.x, p[3] - r1.y, T()));
    }

    // Sums over the warp; false if a value is not finite.
    __device__ __forceinline__ bool finish() {
        bool finite = true;
#pragma unroll
        for (int b = 0; b < TILES; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) finite &= fabsf(o[b][e]) < INFINITY;
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int i = 4; i < 32; i <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], i);
        return __all_sync(0xffffffffu, finite);
    }
    __device__ __forceinline__ void put_lse(float *lse) const {
        const int lane = threadIdx.x % 32;
        if (lane < 4)
#pragma unroll
            for (int e = 0; e < 2; ++e) lse[2 * lane + e] = log_sum(m[e], l[e]);
    }
};

// A warp's row copies, some steps ahead of its work: the same pieces walked by
// itself, a step's page ids read when the step before it is copied.
template <typename M, typename Next>
struct Feed {
    using R = typename M::R;
    static constexpr int STEP = M::STEP, kCopies = STEP * R::kPieces / 32;
    Next next;             // steps a walk on; false behind its last piece
    int i, to;             // rows of the step looked up: i .. , and the piece's end
    bool more;             // such a step is there
    int id, row;           // lane's row of it: page (-1: hidden) and place there
    int64_t k, v;          // its head's offset
    __device__ __forceinline__ explicit Feed(const Next &n) : next(n) {}
    __device__ __forceinline__ void piece() {
        do {
            more = next();
            i = next.walk.t0 * STEP;
            to = min(next.walk.t1 * STEP, next.walk.seen.rows);
        } while (more && i >= to);
    }
    __device__ __forceinline__ void look(const PagedArgs &a) {
        const int at = i + static_cast<int>(threadIdx.x % 32);
        id = -1;
        row = 0;
        if (more && threadIdx.x % 32 < STEP && at < to) {
            const int t = next.walk.seen.at(at), page = a.pages.page.div(t);
            const int found = __ldg(a.pages.table + next.walk.s * a.pages.table_stride + page);
            row = t - page * a.pages.page.d;
            id = static_cast<unsigned>(found) < static_cast<unsigned>(a.pages.pages) ? found : -1;
        }
        const int kh = next.walk.u / a.blocks;
        k = kh * a.k_head;
        v = kh * a.v_head;
    }
    // Queues the copies of the step looked up into `stage` and looks up the next.
    // Returns the rows that are seen, a bit each.
    __device__ __forceinline__ uint32_t issue(const PagedArgs &a, uint32_t stage) {
        const uint32_t live = __ballot_sync(0xffffffffu, id >= 0);
        if (more) {
            each(a, stage);
            i += STEP;
            if (i >= to) piece();
            look(a);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        return live;
    }
    // The step's copies, with every row's own place.
    __device__ __forceinline__ void each(const PagedArgs &a, uint32_t stage) const {
        const int lane = threadIdx.x % 32;
        const int pieces = R::pieces(a);
        const char *kb = a.k + k, *vb = a.v + v;
#pragma unroll
        for (int c = 0; c < kCopies; ++c) {
            const int e = c * 32 + lane, r = e / R::kPieces, p = e % R::kPieces;
            const int page = __shfl_sync(0xffffffffu, id, r), at = __shfl_sync(0xffffffffu, row, r);
            const bool there = page >= 0 && p < pieces;
            const uint64_t n = there ? page : 0, t = there ? at : 0;
            const int q = there ? p : 0;
            const uint32_t to_shared = stage + R::offset(r, p);
            copy_piece<R::kUnit>(to_shared, kb + (n * a.k_page + t * a.k_row + q * R::kUnit), there);
            copy_piece<R::kUnit>(to_shared + STEP * R::kRowBytes, vb + (n * a.v_page + t * a.v_row + q * R::kUnit), there);
        }
    }
};

// The same for steps of 32 short rows, where looking up and addressing each 16 bytes would cost as much as the
// products (227 instructions a step of 760 in all): most steps' rows lie one after the other in one page, or on both sides
// of one border between two pages.  Then the first and the last row's addresses do for all, and where rows follow
// each other without gaps (heads before rows in a page) the copies' addresses differ by constants.
template <typename M, typename Next>
struct RunFeed : Feed<M, Next> {
    using Base = Feed<M, Next>;
    using R = typename M::R;
    using Base::STEP, Base::kCopies, Base::next, Base::i, Base::to, Base::more, Base::id, Base::row;
    static_assert(STEP == 32, "a row a lane");
    const char *kb, *vb;  // the piece's head in the pools
    const int *table;     // its sequence's pages
    __device__ __forceinline__ explicit RunFeed(const Next &n) : Base(n) {}
    __device__ __forceinline__ void begin(const PagedArgs &a) {
        if (!more) return;
        const int kh = next.walk.u / a.blocks;
        kb = a.k + kh * a.k_head;
        vb = a.v + kh * a.v_head;
        table = a.pages.table + next.walk.s * a.pages.table_stride;
    }
    __device__ __forceinline__ void look(const PagedArgs &a) {
        const int at = i + static_cast<int>(threadIdx.x % 32);
        id = -1;
        row = 0;
        if (more && at < to) {
            const int t = next.walk.seen.at(at), page = a.page_shift >= 0 ? t >> a.page_shift : a.pages.page.div(t);
            const int found = __ldg(table + page);
            row = t - page * a.pages.page.d;
            id = static_cast<unsigned>(found) < static_cast<unsigned>(a.pages.pages) ? found : -1;
        }
    }
    static __device__ __forceinline__ const char *place(const char *base, uint32_t page, uint32_t stride, int n, int r) {
        return base + static_cast<uint64_t>(static_cast<uint32_t>(n)) * page + static_cast<int64_t>(r) * stride;
    }
    __device__ __forceinline__ bool runs(const PagedArgs &a, uint32_t stage, uint32_t live) const {
        if (live != 0xffffffffu) return false;
        const int lane = threadIdx.x % 32, first = row - lane;
        const int id0 = __shfl_sync(0xffffffffu, id, 0), row0 = __shfl_sync(0xffffffffu, first, 0);
        const uint32_t begin = __ballot_sync(0xffffffffu, id == id0 && first == row0);
        const bool tight = a.k_row == R::kRow && a.v_row == R::kRow;
        const char *k0 = place(kb, a.k_page, a.k_row, id0, row0), *v0 = place(vb, a.v_page, a.v_row, id0, row0);
        if (begin == live && tight) {
            k0 += lane * R::kUnit;
            v0 += lane * R::kUnit;
#pragma unroll
            for (int c = 0; c < kCopies; ++c) {
                const uint32_t to_shared = stage + R::place(c * 32 + lane);
                copy_piece<R::kUnit>(to_shared, k0 + c * 32 * R::kUnit, true);
                copy_piece<R::kUnit>(to_shared + STEP * R::kRowBytes, v0 + c * 32 * R::kUnit, true);
            }
            return true;
        }
        const int id1 = __shfl_sync(0xffffffffu, id, STEP - 1), row1 = __shfl_sync(0xffffffffu, first, STEP - 1);
        const uint32_t end = __ballot_sync(0xffffffffu, id == id1 && first == row1);
        // a prefix of the rows in the first run, all the others in the last
        if ((begin & (begin + 1)) || (begin | end) != live) return false;
        const char *k1 = place(kb, a.k_page, a.k_row, id1, row1), *v1 = place(vb, a.v_page, a.v_row, id1, row1);
        const int border = __popc(begin);
#pragma unroll
        for (int c = 0; c < kCopies; ++c) {
            const int e = c * 32 + lane, r = e / R::kPieces, p = (e - r * R::kPieces) * R::kUnit;
            const uint32_t to_shared = stage + R::place(e);
            const bool low = r < border;
            copy_piece<R::kUnit>(to_shared, (low ? k0 : k1) + (static_cast<uint64_t>(r) * a.k_row + p), true);
            copy_piece<R::kUnit>(to_shared + STEP * R::kRowBytes, (low ? v0 : v1) + (static_cast<uint64_t>(r) * a.v_row + p), true);
        }
        return true;
    }
    __device__ __forceinline__ uint32_t issue(const PagedArgs &a, uint32_t stage) {
        const uint32_t live = __ballot_sync(0xffffffffu, id >= 0);
        if (more) {
            if (!runs(a, stage, live)) {
                this->k = kb - a.k;
                this->v = vb - a.v;
                this->each(a, stage);
            }
            i += STEP;
            if (i >= to) {
                this->piece();
                begin(a);
            }
            look(a);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        return live;
    }
};

// A piece whose values are not all finite, again and row by row: an infinite value
// meets the second part of a weight as 0 x inf or inf - inf on the tensor cores.
template <typename T, typename M>
__device__ __noinline__ void piece_by_rows(const PagedArgs &a, const Piece &walk, const char *q, char *out, float *partial,
                                           float2 *sums, int64_t stride, int heads) {
    constexpr int DP = M::DP;
    const int lane = threadIdx.x % 32, kh = walk.u / a.blocks;
    const int from = walk.t0 * M::STEP, to = min(walk.t1 * M::STEP, walk.seen.rows);
    auto load = [&](const char *src, float (&x)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            x[j] = 4 * lane + j < a.dim ? widen(reinterpret_cast<const T *>(src) + 4 * lane + j) : 0.f;
    };
    for (int h = 0; h < heads; ++h) {
        float x[4], o[4] = {}, m = -INFINITY, l = 0.f;
        load(q + h * a.q_head, x);
        for (int i = from; i < to; ++i) {
            const int t = walk.seen.at(i);
            const int64_t kr = a.pages.row(walk.s, t, a.k_page, a.k_row), vr = a.pages.row(walk.s, t, a.v_page, a.v_row);
            if (kr < 0) continue;
            float k[4], v[4];
            load(a.k + kr + kh * a.k_head, k);
            load(a.v + vr + kh * a.v_head, v);
            const float y = warp_sum(x[0] * k[0] + x[1] * k[1] + x[2] * k[2] + x[3] * k[3]) * a.scale;
            const float top = fmaxf(m, y), ref = top == -INFINITY ? 0.f : top;
            const float c = ex2(m - ref), p = ex2(y - ref);
            l = fmaf(l, c, p);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = fmaf(o[j], c, p * v[j]);
            m = top;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int d = 4 * lane + j;
            if (out && d < a.dim) narrow(l != 0.f ? o[j] / l : 0.f, reinterpret_cast<T *>(out + h * a.o_head) + d);
            if (partial && d < DP) partial[h * DP + d] = o[j];
        }
        if (partial && lane == 0) sums[h * stride] = make_float2(m, l);
    }
}

// The same where a way to work needs it.
template <typename T, typename M>
__device__ __forceinline__ void again(const PagedArgs &a, const Piece &walk, const char *q, char *out, float *partial,
                                      float2 *sums, int64_t stride, int heads) {
    if constexpr (M::kAgain) piece_by_rows<T, M>(a, walk, q, out, partial, sums, stride, heads);
}

// The shares of a block of heads in a head's weights: rows i = from + first, + step, .. of those seen; N
// query heads' scores a row.  A row's shares are added up before they meet what is there, which may be
// so much larger that each alone would be lost in its rounding: of several blocks (kBlocks), block b
// leaves the sum so far where the first one's first score was, and the last adds it to the weight.
template <int N, int H, bool kBlocks>
__device__ __forceinline__ void add_rows(const PagedArgs &a, const Piece &walk, int64_t unit, int kh, int from, int to,
                                         int first, int step, const float (&lse)[H], int b) {
    constexpr int kRows = 4;  // in flight
    const bool last = !kBlocks || b == a.blocks - 1;
    float *weights = a.weights + walk.s * a.w_batch + kh * a.w_head;
    float *scores = a.scores + unit * a.seen_max * N;
    const int64_t block = b * a.seen_max * N;
#pragma unroll 1
    for (int i0 = from + first; i0 < to; i0 += step * kRows) {
        alignas(16) float2 x[kRows][N / 2];
        float was[kRows], sum[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const int i = min(i0 + r * step, to - 1);
            float *row = scores + static_cast<int64_t>(i) * N;
            was[r] = last ? weights[walk.seen.at(i)] : 0.f;
            sum[r] = kBlocks && b ? __ldcg(row) : 0.f;
            if (kBlocks) row += block;
            if constexpr (N % 4 == 0) {
#pragma unroll
                for (int h = 0; h < N / 2; h += 2)
                    *reinterpret_cast<float4 *>(&x[r][h]) = __ldcg(reinterpret_cast<const float4 *>(row + 2 * h));
            } else {
#pragma unroll
                for (int h = 0; h < N / 2; ++h) x[r][h] = __ldcg(reinterpret_cast<const float2 *>(row + 2 * h));
            }
        }
        // A hidden row's score is -inf, and adds nothing whatever the sum is; nor does a head past the
        // group (lse infinite), whatever its score is: of an infinite key, 0 x inf.
        auto share = [&](float score, int h) {
            return score == -INFINITY || lse[h] == INFINITY ? 0.f : ex2(score - lse[h]);
        };
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const int i = i0 + r * step;
#pragma unroll
            for (int h = 0; h < N / 2; ++h) {
                sum[r] += share(x[r][h].x, 2 * h);
                sum[r] += share(x[r][h].y, 2 * h + 1);
            }
            if (i >= to) continue;
            if (last) weights[walk.seen.at(i)] = was[r] + sum[r];
            else scores[static_cast<int64_t>(i) * N] = sum[r];
        }
    }
}
template <int H>
__device__ __forceinline__ void add_weights(const PagedArgs &a, const Piece &walk, int64_t unit, int kh, int from, int to,
                                            int first, int step, const float (&lse)[H]) {
    if (a.heads2 == 2) return add_rows<2, H, false>(a, walk, unit, kh, from, to, first, step, lse, 0);
    if constexpr (H == 8) {
        if (a.heads2 == 4) return add_rows<4, H, false>(a, walk, unit, kh, from, to, first, step, lse, 0);
        if (a.heads2 == 6) return add_rows<6, H, false>(a, walk, unit, kh, from, to, first, step, lse, 0);
    }
    add_rows<H, H, false>(a, walk, unit, kh, from, to, first, step, lse, 0);
}

// Works through pieces; `done(math, piece, q, unit, heads, kh, h0)` takes each one's results.
template <typename T, typename M, typename Next, typename Done>
__device__ __forceinline__ void work_through(const PagedArgs &a, uint32_t ring, const Next &start, const Done &done) {
    using R = typename M::R;
    constexpr int H = M::kHeads, STEP = M::STEP, STAGES = M::STAGES;
    Next next(start);
    std::conditional_t<M::kRuns, RunFeed<M, Next>, Feed<M, Next>> feed(start);
    feed.piece();
    if constexpr (M::kRuns) feed.begin(a);
    feed.look(a);
    uint32_t live[STAGES - 1];  // of the steps in flight, the oldest first
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) live[i] = feed.issue(a, ring + i * R::kBytes);
    int slot = 0;
    while (next()) {
        const Piece &walk = next.walk;
        const int kh = walk.u / a.blocks, h0 = walk.u % a.blocks * H, heads = min(H, a.group - h0);
        const int64_t unit = static_cast<int64_t>(walk.s) * (a.kv_heads * a.blocks) + walk.u;
        const char *q = a.q + walk.s * a.q_batch + (kh * a.group + h0) * a.q_head;
        const int to = min(walk.t1 * STEP, walk.seen.rows);
        M math;
        math.begin(a, q, heads);
        const int64_t score0 = unit * a.seen_max + walk.t0 * STEP;
        float *scores = a.scores ? a.scores + score0 * a.heads2 : nullptr;  // of the step's first row
        for (int i = walk.t0 * STEP; i < to; i += STEP) {
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
            __syncwarp();  // every lane's copies of the step have landed, and all are done with the slot filled next
            const uint32_t seen = live[0];
#pragma unroll
            for (int j = 0; j + 1 < STAGES - 1; ++j) live[j] = live[j + 1];
            live[STAGES - 2] = feed.issue(a, ring + (slot == 0 ? STAGES - 1 : slot - 1) * R::kBytes);
            math.step(a, ring + slot * R::kBytes, seen, to - i, scores);
            if (scores) scores += STEP * a.heads2;
            slot = slot == STAGES - 1 ? 0 : slot + 1;
        }
        done(math, walk, q, unit, heads, kh, h0);
    }
}

template <int STEP>
struct NextStretch {
    Walk walk;
    const PagedArgs &a;
    const Plan<STEP> &plan;
    __device__ __forceinline__ bool operator()() { return walk.next(a, plan); }
};
template <int STEP>
struct NextQuarter {
    Quarters<STEP> walk;
    const PagedArgs &a;
    __device__ __forceinline__ bool operator()() { return walk.next(a); }
};

template <typename T, typename M>
__global__ void __launch_bounds__(kThreads, M::kCtas) k_paged(const __grid_constant__ PagedArgs a) {
    extern __shared__ __align__(128) char smem[];
    constexpr int H = M::kHeads, DP = M::DP, STEP = M::STEP;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, worker = blockIdx.x * kWarps + warp;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // sequences that see nothing give zeros
    for (int s = worker; s < a.batch; s += gridDim.x * kWarps) {
        if (seen_of(a, s).rows > 0) continue;
        const int heads = a.kv_heads * a.group;
        for (int e = lane; e < heads * a.dim; e += 32)
            narrow(0.f, reinterpret_cast<T *>(a.out + s * a.o_batch + e / a.dim * a.o_head) + e % a.dim);
    }
    Plan<STEP> plan;
    plan.init(a);
    Walk walk = {};
    if (!walk.init(a, plan, worker)) return;
    int part = 0;
    work_through<T, M>(a, shared_address(smem + warp * M::R::kWarpBytes), NextStretch<STEP>{walk, a, plan},
                       [&](M &math, const Piece &piece, const char *q, int64_t unit, int heads, int kh, int h0) {
        const bool whole = piece.t0 == 0 && piece.t1 == piece.steps;
        char *out = whole ? a.out + piece.s * a.o_batch + (kh * a.group + h0) * a.o_head : nullptr;
        float *partial = whole ? nullptr : a.partial + (worker * 2 + part) * static_cast<int64_t>(H * DP);
        const int64_t warps = a.warps;
        float2 *sums = a.sums + part * H * warps + worker;
        if (!math.finish()) again<T, M>(a, piece, q, out, partial, sums, warps, heads);
        else if (whole) math.put_out(a, out, heads);
        else math.put_partial(partial, sums, warps, heads);
        if (whole && a.lse) math.put_lse(a.lse + unit * H);
        part = 1;
    });
}

// The same with a unit a CTA.
template <typename T, typename M>
__global__ void __launch_bounds__(kThreads, M::kCtas) k_paged_few(const __grid_constant__ PagedArgs a) {
    extern __shared__ __align__(128) char smem[];
    constexpr int H = M::kHeads, DP = M::DP, STEP = M::STEP, kPart = H * (DP + 2);
    const int tid = threadIdx.x, warp = tid / 32;
    float *parts = reinterpret_cast<float *>(smem + kWarps * M::R::kWarpBytes);
    Quarters<STEP> walk = {};
    walk.unit = blockIdx.x;
    work_through<T, M>(a, shared_address(smem + warp * M::R::kWarpBytes), NextQuarter<STEP>{walk, a},
                       [&](M &math, const Piece &piece, const char *q, int64_t unit, int heads, int kh, int h0) {
        float *mine = parts + warp * kPart;
        float2 *sums = reinterpret_cast<float2 *>(mine + H * DP);
        if (!math.finish()) again<T, M>(a, piece, q, nullptr, mine, sums, 1, heads);
        else math.put_partial(mine, sums, 1, heads);
        __syncthreads();
        char *out = a.out + piece.s * a.o_batch + (kh * a.group + h0) * a.o_head;
        for (int e = tid; e < heads * DP; e += kThreads) {
            const int h = e / DP, j = e % DP;
            Partial all = {-INFINITY, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float *p = parts + w * kPart;
                all.add(p[H * DP + 2 * h], p[H * DP + 2 * h + 1], p[e]);
            }
            if (j < a.dim)
                narrow(all.sum != 0.f ? all.x / all.sum : 0.f, reinterpret_cast<T *>(out + h * a.o_head) + j);
        }
        if (a.weights) {
            float lse[H];
#pragma unroll
            for (int h = 0; h < H; ++h) {
                Partial all = {-INFINITY, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float *p = parts + w * kPart + H * DP;
                    if (h < heads) all.add(p[2 * h], p[2 * h + 1], 0.f);
                }
                lse[h] = log_sum(all.top, all.sum);
            }
            add_weights<H>(a, piece, unit, kh, 0, piece.seen.rows, tid, kThreads, lse);
        }
        __syncthreads();  // the partials have been read
    });
}

// Whether there are weights to add, and for groups of several blocks of heads (in one kernel with the other case
// some of its registers spill).
enum { kNoWeights, kWeights, kBlockWeights };
// Warps for each of k_paged's, to hide the latency of the little that each reads.  One is enough for the short way
// there is without weights over pages of 4 bits (one sequence of 32768 rows: 1.6 us less than two; with weights,
// 24 sequences to 8192 rows: 37.8 and 36.0).
template <typename M, int MODE>
constexpr int kJoiners = M::kRuns && MODE == kNoWeights ? 1 : 2;

// Joins the units that were cut: the warps whose stretch starts inside a unit
// share its columns, four at a time.  With weights, every warp then adds up its
// own stretch's rows.  All of it is latency: what needs no partials (whose columns, in whole-number divisions;
// the weights on their way to L2) comes before the wait, and loads of a kind are issued together.
template <typename T, typename M, int MODE>
__global__ void __launch_bounds__(kThreads, 5) k_join(const __grid_constant__ PagedArgs a) {
    constexpr int H = M::kHeads, DP = M::DP, STEP = M::STEP;
    constexpr int64_t kPart = H * DP;
    constexpr int kJoin = kJoiners<M, MODE>;
    constexpr bool kBlocks = MODE == kBlockWeights;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int id = blockIdx.x * kWarps + warp, worker = id / kJoin, share = id % kJoin;
    Plan<STEP> plan;
    plan.init(a);
    Walk walk = {};
    const bool work = walk.init(a, plan, worker);
    if (MODE != kNoWeights && work) {
        // the weights that this warp adds to, which k_paged leaves alone, into L2
        Walk ahead = walk;
        while (ahead.next(a, plan)) {
            const int rows = min(ahead.t1 * STEP, ahead.seen.rows) - ahead.t0 * STEP;
            const int from = ahead.t0 * STEP + rows * share / kJoin, to = ahead.t0 * STEP + rows * (share + 1) / kJoin;
            const float *weights = a.weights + ahead.s * a.w_batch + ahead.u / a.blocks * a.w_head;
            for (int i = from + 32 * lane; i < to + 31; i += 32 * 32)
                if (to > from) asm volatile("prefetch.global.L2 [%0];" ::"l"(weights + ahead.seen.at(min(i, to - 1))));
        }
    }
    // The partials of a unit cut between workers b0 ..: a worker's first piece is in its
    // slot 0, so only b0's may be its last one, in slot 1.
    struct Parts {
        const float *at;
        int b0, slot0;
        __device__ __forceinline__ const float *operator()(int b) const {
            return at + (b * 2 + (b == b0 ? slot0 : 0)) * kPart;
        }
    };
    const int64_t warps = a.warps;
    auto sums_of = [&](const Parts &part, int b, int h) {
        return __ldcg(a.sums + ((b == part.b0 ? part.slot0 : 0) * H + h) * warps + b);
    };
    // this warp's columns of a unit that its stretch starts in
    int kh = 0, h0 = 0, n = 0, c0 = 0, c1 = 0;
    Parts part = {a.partial, 0, 0};
    if (work) {
        const int cut = (walk.x - walk.base) / walk.steps, first = walk.base + cut * walk.steps;
        if (first < walk.x) {
            part.b0 = plan.worker_of(first);
            part.slot0 = plan.start(part.b0) >= first ? 0 : 1;
            n = plan.worker_of(first + walk.steps - 1) - part.b0 + 1;
            kh = cut / a.blocks;
            h0 = cut % a.blocks * H;
            const int columns = min(H, a.group - h0) * (DP / 4), sharers = (n - 1) * kJoin;
            const int me = (worker - part.b0 - 1) * kJoin + share;
            c0 = columns * me / sharers;
            c1 = columns * (me + 1) / sharers;
        }
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (!work) return;
    if (c0 < c1) {
        const int b0 = part.b0;
        // head by head of its columns
        for (int h = c0 / (DP / 4); h * (DP / 4) < c1; ++h) {
            const int lo = max(c0, h * (DP / 4)), hi = min(c1, (h + 1) * (DP / 4));
            // 2^shift lanes side by side over the columns, the rest over the partials
            const int shift = hi - lo > 1 ? min(32 - __clz(hi - lo - 1), 5) : 0;
            const int wide = 1 << shift, step = 32 >> shift, beside = lane & (wide - 1), behind = lane >> shift;
            constexpr int kFlight = 5;
            float4 v[kFlight];  // the first columns' values are under way while the softmax is worked out
            float top_of[kFlight];
            auto load = [&](int c, int i, int b) {
                v[i] = b < n ? __ldcg(reinterpret_cast<const float4 *>(part(b0 + b) + 4 * c)) : float4{};
                top_of[i] = b < n ? sums_of(part, b0 + b, h).x : -INFINITY;
            };
#pragma unroll
            for (int i = 0; i < kFlight; ++i) load(min(lo + beside, hi - 1), i, behind + i * step);
            float top = -INFINITY, sum = 0.f;
            for (int base = 0; base < n; base += 32 * kFlight) {
                float2 x[kFlight];
#pragma unroll
                for (int i = 0; i < kFlight; ++i) {
                    const int b = base + lane + 32 * i;
                    x[i] = b < n ? sums_of(part, b0 + b, h) : make_float2(-INFINITY, 0.f);
                }
#pragma unroll
                for (int i = 0; i < kFlight; ++i) {
                    const float t = fmaxf(top, x[i].x), ref = t == -INFINITY ? 0.f : t;
                    sum = fmaf(sum, ex2(top - ref), x[i].y * ex2(x[i].x - ref));
                    top = t;
                }
            }
            const float most = warp_max(top), ref = most == -INFINITY ? 0.f : most;
            sum = warp_sum(sum * ex2(top - ref));
            const float f = sum != 0.f ? 1.f / sum : 0.f;
            for (int base = lo; base < hi; base += wide) {
                const int c = min(base + beside, hi - 1);
                float4 x = {};
                for (int b = 0; b < n; b += kFlight * step) {
                    if (base != lo || b)
#pragma unroll
                        for (int i = 0; i < kFlight; ++i) load(c, i, b + behind + i * step);
#pragma unroll
                    for (int i = 0; i < kFlight; ++i) {
                        const float w = ex2(top_of[i] - ref) * f;
                        x.x = fmaf(w, v[i].x, x.x);
                        x.y = fmaf(w, v[i].y, x.y);
                        x.z = fmaf(w, v[i].z, x.z);
                        x.w = fmaf(w, v[i].w, x.w);
                    }
                }
                for (int w = 16; w >= wide; w >>= 1) {
                    x.x += __shfl_xor_sync(0xffffffffu, x.x, w);
                    x.y += __shfl_xor_sync(0xffffffffu, x.y, w);
                    x.z += __shfl_xor_sync(0xffffffffu, x.z, w);
                    x.w += __shfl_xor_sync(0xffffffffu, x.w, w);
                }
                const int j = c % (DP / 4) * 4;
                if (lane < wide && base + lane < hi && j < a.dim) {
                    T *out = reinterpret_cast<T *>(a.out + walk.s * a.o_batch + (kh * a.group + h0 + h) * a.o_head) + j;
                    narrow(x.x, out);
                    narrow(x.y, out + 1);
                    narrow(x.z, out + 2);
                    narrow(x.w, out + 3);
                }
            }
        }
    }
    if (MODE == kNoWeights) return;
    // A cut unit's softmax over its partials: each head's maximum and sum, in every lane.
    auto softmax_of = [&](const Parts &part, int b1, float (&top)[H], float (&sum)[H]) {
#pragma unroll
        for (int h = 0; h < H; ++h) {
            top[h] = -INFINITY;
            sum[h] = 0.f;
        }
#pragma unroll 2
        for (int b = part.b0 + lane; b <= b1; b += 32) {
            float2 x[H];
#pragma unroll
            for (int h = 0; h < H; ++h) x[h] = h < a.heads2 ? sums_of(part, b, h) : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int h = 0; h < H; ++h) {
                const float t = fmaxf(top[h], x[h].x), ref = t == -INFINITY ? 0.f : t;
                sum[h] = fmaf(sum[h], ex2(top[h] - ref), x[h].y * ex2(x[h].x - ref));
                top[h] = t;
            }
        }
#pragma unroll
        for (int h = 0; h < H; ++h) {
            if (h >= a.heads2) continue;
            const float t = warp_max(top[h]), ref = t == -INFINITY ? 0.f : t;
            sum[h] = warp_sum(sum[h] * ex2(top[h] - ref));
            top[h] = t;
        }
    };
    // Its logarithm, of head lane / each in a group of `each` lanes: all heads at once.
    const int each = a.heads2 == 2 ? 16 : a.heads2 == 4 ? 8 : 4;
    auto log_sum_of = [&](const Parts &part, int b1) {
        const int h = lane / each;
        float top = -INFINITY, sum = 0.f;
        if (h < a.heads2) {
#pragma unroll 4
            for (int b = part.b0 + lane % each; b <= b1; b += each) {
                const float2 x = sums_of(part, b, h);
                const float t = fmaxf(top, x.x), ref = t == -INFINITY ? 0.f : t;
                sum = fmaf(sum, ex2(top - ref), x.y * ex2(x.x - ref));
                top = t;
            }
        }
        float most = top;
        for (int o = each / 2; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        sum *= ex2(top - (most == -INFINITY ? 0.f : most));
        for (int o = each / 2; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        return log_sum(most, sum);
    };
    while (walk.next(a, plan)) {
        if (walk.u % a.blocks) continue;  // the group's first block of heads adds up for all of them
        const int lo = walk.t0 * STEP, rows = min(walk.t1 * STEP, walk.seen.rows) - lo;
        const int from = lo + rows * share / kJoin, to = lo + rows * (share + 1) / kJoin;
        const int64_t unit = static_cast<int64_t>(walk.s) * plan.units + walk.u;
        const int kh = walk.u / a.blocks;
        for (int b = 0; b < (kBlocks ? a.blocks : 1); ++b) {
            const int start = walk.base + (walk.u + b) * walk.steps;
            const int b0 = plan.worker_of(start), b1 = plan.worker_of(start + walk.steps - 1);
            float lse[H];
            const Parts part = {a.partial, b0, plan.start(b0) >= start ? 0 : 1};
            if constexpr (M::kRuns) {
                const float mine = b0 != b1 ? log_sum_of(part, b1) : 0.f;
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    const float joined = __shfl_sync(0xffffffffu, mine, h * each % 32);
                    lse[h] = h >= a.group - b * H ? INFINITY : b0 == b1 ? __ldcg(a.lse + (unit + b) * H + h) : joined;
                }
            } else {
                float top[H], sum[H];
                if (b0 != b1) softmax_of(part, b1, top, sum);
#pragma unroll
                for (int h = 0; h < H; ++h)
                    lse[h] = h >= a.group - b * H ? INFINITY : b0 == b1 ? __ldcg(a.lse + (unit + b) * H + h) : log_sum(top[h], sum[h]);
            }
            if constexpr (kBlocks) add_rows<H, H, true>(a, walk, unit, kh, from, to, lane, 32, lse, b);
            else add_weights<H>(a, walk, unit, kh, from, to, lane, 32, lse);
        }
    }
}

template <typename T, typename M>
int launch(mr_context *ctx, PagedArgs &a) {
    constexpr int H = M::kHeads, STEP = M::STEP;
    a.blocks = (a.group - 1) / H + 1;
    a.heads2 = (std::min(a.group, H) + 1) / 2 * 2;
    a.page_shift = -1;
    for (int n = 0; n < 31; ++n)
        if (a.pages.page.d == 1 << n) a.page_shift = n;
    // the most rows a token can see, and the most steps there can be
    a.seen_max = a.window ? std::min<int64_t>(a.capacity, static_cast<int64_t>(a.window) + a.sinks) : a.capacity;
    const int64_t units = static_cast<int64_t>(a.batch) * a.kv_heads * a.blocks;
    const int64_t steps = (a.seen_max + STEP - 1) / STEP;
    MR_REQUIRE(units <= kMaxSteps && units * steps <= kMaxSteps, "the sequences' rows and heads are too many for one call");
    // weights of a group in several blocks are added up by one warp, which only k_join can
    const bool few = steps <= kFewSteps && (!a.weights || a.blocks == 1);
    const int64_t ctas = few ? units : (units * steps + kWarps - 1) / kWarps;
    const int grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(ctas, M::ctas(units * steps, ctx->sm_count, a.weights) * ctx->sm_count)));
    a.warps = grid * kWarps;
    const size_t partial = few ? 0 : sizeof(float) * 2 * a.warps * H * M::DP;
    const size_t sums = few ? 0 : sizeof(float2) * 2 * a.warps * H;
    const size_t lse = a.weights && !few ? sizeof(float) * units * H : 0;
    const size_t scores = a.weights ? sizeof(float) * units * a.seen_max * a.heads2 : 0;
    auto up = [](size_t n) { return (n + 255) & ~size_t(255); };
    Scratch scratch(ctx);
    MR_CHECK(scratch.take(up(partial) + up(sums) + up(lse) + scores));
    char *base = static_cast<char *>(scratch.data);
    a.partial = reinterpret_cast<float *>(base);
    base += up(partial);
    a.sums = reinterpret_cast<float2 *>(base);
    base += up(sums);
    a.lse = lse ? reinterpret_cast<float *>(base) : nullptr;
    a.scores = scores ? reinterpret_cast<float *>(base + up(lse)) : nullptr;
    constexpr int kRings = kWarps * M::R::kWarpBytes;
    if (few) {
        constexpr int kSmem = kRings + kWarps * H * (M::DP + 2) * 4;
        static std::atomic<uint64_t> allowed{0};
        MR_CHECK(allow_shared(ctx->device, reinterpret_cast<const void *>(k_paged_few<T, M>), kSmem, allowed));
        k_paged_few<T, M><<<grid, kThreads, kSmem, ctx->stream>>>(a);
        MR_CUDA_TRY(cudaGetLastError());
        return MR_OK;
    }
    static std::atomic<uint64_t> allowed{0};
    MR_CHECK(allow_shared(ctx->device, reinterpret_cast<const void *>(k_paged<T, M>), kRings, allowed));
    k_paged<T, M><<<grid, kThreads, kRings, ctx->stream>>>(a);
    MR_CUDA_TRY(cudaGetLastError());
    auto join = [&](auto mode) {
        constexpr int MODE = decltype(mode)::value;
        return launch_early(ctx, dim3(grid * kJoiners<M, MODE>), dim3(kThreads), k_join<T, M, MODE>, a);
    };
    return !a.weights      ? join(std::integral_constant<int, kNoWeights>())
           : a.blocks == 1 ? join(std::integral_constant<int, kWeights>())
                           : join(std::integral_constant<int, kBlockWeights>());
}

}  // namespace
}  // namespace cache
}  // namespace mr
