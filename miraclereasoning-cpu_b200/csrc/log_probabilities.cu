// Log probabilities of given tokens, the entropy and the most likely tokens of rows
// of logits x:
//
//   S = sum e^(x - m),  log p_t = x_t - m - log S,  H = log S - sum e^(x - m) (x - m) / S
//
// (m: about the maximum; differences, so that logits far from 0 cost no digits).
//
// One pass: every logit is read once, at about seven operations, and each thread
// keeps a running maximum, S and the entropy's sum of its own elements.  A row is a
// team's: a CTA's; a warp's where rows are short; or where rows are few and long a
// cluster's of up to 4 CTAs, whose sums and candidates meet in the first one's
// shared memory.
//
// The most likely tokens come from maxima of 256 parts of the row (a CTA's threads; eight of a
// warp's lane).  The k-th largest of them, T, is a lower bound of the k-th largest logit, and only a part
// whose maximum reaches T can have such logits: about k parts' elements are read
// again, from cache, and the few that reach T are ranked by counting.  No work is
// added to the pass, and the list's does not depend on the order of the logits.  Where
// more of them reach T than there is room for (rows that allow fewer tokens than are asked for beside
// a mask of -inf, constant rows), the row is read once more for the larger ones alone, and the
// rest filled with the first ones that equal T, looked for by one warp.  That is slow: 20 alternatives of rows that
// allow 5 tokens take 25 us instead of 7.3 (1 row of 64000 float32), 27 instead of 9.1 (64 of 64000 bfloat16), 255
// instead of 37 (4096 of 8000 float32, where a warp counts every masked logit).
//
// 4096 rows of 32000 float32, 2 given tokens and 5 alternatives (525 MB): 92 us, 5.7 TB/s.  What a row costs once
// (its sums joined, its list) leaves a CTA without loads under way, so that the start of a later row is fetched
// to L2 meanwhile: 99.5 without it; 95 with 16 KB, 91 with 64, which other sizes lose again; all of each row ahead of its
// loads 89, but 1000 rows 10% slower.  Rows through rings of asynchronous copies in shared memory took 8% more than
// registers, CTAs of 128 or 512 threads 115 and 126 us.  16-bit rows are bound by their instructions and the
// exponentials' unit (60% and 47% busy; 2000 rows of 64000 bfloat16 66 us, 4096 of 32000 62, 60 to 66% of the copy
// rate); whole groups without bounds checks and sums kept in pairs gained nothing there.  Short rows, a warp's, have nothing
// fetched ahead: 4096 of 4000, 8000 and 12000 float32 20.6, 32.0 and 43.0 us where the copy rate has 10.2, 20.4 and 30.5.
// One row of 64000 takes 7.3 us: most of it is the list, whose steps follow each other.
#include <cooperative_groups.h>

#include <type_traits>

#include "cache_ops.cuh"

namespace mr {
namespace cache {
namespace {

namespace cg = cooperative_groups;

constexpr int kMostTop = 128, kMostCtas = 4, kParts = 256;
constexpr int kResident = 4;             // CTAs of an SM
constexpr uint32_t kAhead = 32 << 10;    // bytes of a later row, fetched to L2
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
    int64_t rows;
    int vocab, given, top, ctas;  // ctas: of a row
    int ahead;                    // CTAs that run at once
};

// Logits in rising order as unsigned numbers; both zeros equal, NaN the lowest.
__device__ __forceinline__ uint32_t order_of(float x) {
    if (x != x) return 0;
    const uint32_t bits = __float_as_uint(x + 0.f);
    return bits ^ (static_cast<uint32_t>(static_cast<int32_t>(bits) >> 31) | 0x80000000u);
}
constexpr uint32_t kLowest = 0x007fffffu;  // of -inf
constexpr uint32_t kZero = 0x80000000u;    // of both zeros; no logit has the order below it, -0's by its bits
// The logit of an order from kLowest on; NaN of 0.
__device__ __forceinline__ float value_of(uint32_t order) {
    return order ? __uint_as_float(order & 0x80000000u ? order ^ 0x80000000u : ~order) : __uint_as_float(0x7fffffffu);
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
};

// Two float32 operations in one instruction.
union Pair {
    float2 f;
    uint64_t bits;
};
__device__ __forceinline__ Pair both(float x) {
    Pair p;
    p.f = make_float2(x, x);
    return p;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair c;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(c.bits) : "l"(a.bits), "l"(b.bits));
    return c;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair c;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(c.bits) : "l"(a.bits), "l"(b.bits));
    return c;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.bits) : "l"(a.bits), "l"(b.bits), "l"(c.bits));
    return d;
}

template <typename T>
struct Vector {
    static constexpr int kValues = 16 / sizeof(T);
    union {
        uint4 raw;
        T v[kValues];
    };
    __device__ __forceinline__ Vector() {}
    // -inf everywhere, which adds nothing
    __device__ __forceinline__ void clear() {
        const uint32_t low = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
        raw = make_uint4(low, low, low, low);
    }
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

// P threads of a row (or of a CTA's share of it): a CTA or a warp.
template <int P>
struct Shared {
    static constexpr int kWarps = P / 32, kRoom = P == 32 ? 256 : 1024, kLists = P == 32 ? 1 : kMostCtas;
    uint64_t found[kRoom];           // candidates
    uint64_t best[kMostTop];         // of them the largest, falling; 0 behind
    uint64_t all[kMostTop * kLists - (P == 32) * (kMostTop - 1)];  // of the first CTA: every CTA's best
    Sums parts[kWarps * kLists];     // and every warp's sums
    Sums sums[kWarps];               // this team's
    Sums total;
    uint32_t maxima[kParts];
    uint8_t reaching[kParts];        // parts whose maximum reaches the bound; of a CTA, 32 of each warp
    uint32_t bound;
    int count;
    int tally[kWarps];
};
template <int P>
__device__ __forceinline__ void team_sync() {
    if (P == 32) __syncwarp();
    else __syncthreads();
}

// Candidates of the slice: elements from `bound` on, or past it.
template <typename T, int P>
__device__ __forceinline__ void collect(const Slice<T> &slice, Shared<P> &sh, int tid, uint32_t bound, bool past) {
    constexpr int V = Slice<T>::V, kFlight = 4;
    const int warp = tid / 32, lane = tid % 32;
    const float limit = value_of(bound);
    // as the orders compare; with 0, the order of NaN, all elements, or all others
    auto reaches = [&](float x) { return past ? x > limit || (!bound && x == x) : x >= limit || !bound; };
    auto push = [&](int token, float x) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < Shared<P>::kRoom) sh.found[at] = candidate(order_of(x), token);
    };
    slice.singles(tid, [&](int token, float x) {
        if (reaches(x)) push(token, x);
    });
    // the elements of the warp's parts that reach the bound, read by all its lanes: 128 vectors at once
    uint8_t *reaching = sh.reaching + warp * 32;
    int parts = 0;
#pragma unroll
    for (int i = 0; i < kParts / P; ++i) {
        const int part = warp * 32 + i * P + lane;
        const bool is = sh.maxima[part] >= bound;
        const uint32_t mask = __ballot_sync(0xffffffffu, is);
        if (is) reaching[parts + __popc(mask & ((1u << lane) - 1))] = static_cast<uint8_t>(part);
        parts += __popc(mask);
    }
    __syncwarp();
    const int each = (slice.v1 - slice.v0 + kParts - 1) / kParts, all = parts * each;
    const float per = 1.f / static_cast<float>(each);
#pragma unroll 1
    for (int e0 = lane; e0 < all; e0 += 32 * kFlight) {
        Vector<T> x[kFlight];
        int v[kFlight];
#pragma unroll
        for (int f = 0; f < kFlight; ++f) {
            const int e = min(e0 + 32 * f, all - 1);
            int t = min(static_cast<int>(static_cast<float>(e) * per), parts - 1);  // e / each, or one beside it
            t -= t * each > e;
            t += (t + 1) * each <= e;
            v[f] = e0 + 32 * f < all ? slice.v0 + reaching[t] + (e - t * each) * kParts : slice.v1;
            if (v[f] < slice.v1) x[f] = slice.load(v[f]);
            else x[f].clear();
        }
#pragma unroll
        for (int f = 0; f < kFlight; ++f) {
            uint32_t hits = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) hits |= reaches(x[f][j]) ? 1u << j : 0u;
            if (v[f] >= slice.v1) hits = 0;
            for (; hits; hits &= hits - 1) {
                const int token = slice.head + v[f] * V + __ffs(hits) - 1;
                push(token, widen(slice.row + token));
            }
        }
    }
}

// How many elements of the slice are from `bound` on; all threads have it.
template <typename T, int P>
__device__ int count_from(const Slice<T> &slice, Shared<P> &sh, int tid, uint32_t bound) {
    int n = 0;
    auto add = [&](int, float x) { n += order_of(x) >= bound; };
    slice.singles(tid, add);
    for (int v = slice.v0 + tid; v < slice.v1; v += P) {
        const Vector<T> x = slice.load(v);
#pragma unroll
        for (int j = 0; j < Slice<T>::V; ++j) add(0, x[j]);
    }
    n = __reduce_add_sync(0xffffffffu, n);
    if (P == 32) return n;
    __syncthreads();
    if (tid % 32 == 0) sh.tally[tid / 32] = n;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int w = 0; w < P / 32; ++w) n += sh.tally[w];
    return n;
}

// The slice's `want` largest elements into sh.best.  largest: of the thread's parts.
template <typename T, int P>
__device__ __forceinline__ void choose(const Slice<T> &slice, Shared<P> &sh, int tid, const float (&largest)[kParts / P], int want) {
    constexpr int V = Slice<T>::V, kKeys = kParts / 32, kRoom = Shared<P>::kRoom;
    const int lane = tid % 32;
#pragma unroll
    for (int i = 0; i < kParts / P; ++i) {
        const bool some = slice.v0 + tid + i * P < slice.v1 || (i == 0 && (tid < slice.head_count || tid < slice.tail_count));
        sh.maxima[tid + i * P] = some ? max(order_of(largest[i]), 1u) : 0u;  // at least 1, of NaN alone too: has elements
    }
    if (tid == 0) sh.count = 0;
    team_sync<P>();
    if (tid < 32) {
        // the want-th largest of the maxima, or a number below it that not many more reach: halving
        uint32_t key[kKeys], low = 0xffffffffu, high = 0;
#pragma unroll
        for (int w = 0; w < kKeys; ++w) {
            key[w] = sh.maxima[w * 32 + lane];
            low = min(low, key[w]);
            high = max(high, key[w]);
        }
        low = __reduce_min_sync(0xffffffffu, low);
        high = __reduce_max_sync(0xffffffffu, high);
        int reach = kParts;
        ++high;  // order_of(+inf) at most: does not wrap
        while (high - low > 1 && reach > want + 4 + want / 4) {
            const uint32_t mid = low + (high - low) / 2;
            int n = 0;
#pragma unroll
            for (int w = 0; w < kKeys; ++w) n += key[w] >= mid;
            n = __reduce_add_sync(0xffffffffu, n);
            if (n >= want) low = mid, reach = n;
            else high = mid;
        }
        // Fewer parts with elements than wanted, or among them NaN alone: everything counts.  Otherwise an order whose
        // number compares alike: the one below zero's reads as -0, which zeros reach but do not pass.
        if (lane == 0) sh.bound = low <= 1 ? 0u : low == kZero - 1 ? kZero : max(low, kLowest);
    }
    team_sync<P>();
    uint32_t bound = sh.bound;
    auto collected = [&](bool past) {
        collect<T, P>(slice, sh, tid, bound, past);
        team_sync<P>();
        const int n = sh.count;
        team_sync<P>();
        if (tid == 0) sh.count = 0;
        team_sync<P>();
        return n;
    };
    int n = collected(false);
    bool enough = n >= want;  // from the bound on (parts of NaN alone have less than their maximum says)
    if (enough && n > kRoom) n = collected(true);
    if (!enough || n > kRoom) {
        // the want-th largest itself, bit by bit
        bound = 0;
        for (int bit = 31; bit >= 0; --bit)
            if (count_from<T, P>(slice, sh, tid, bound | 1u << bit) >= want) bound |= 1u << bit;
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
        team_sync<P>();
    }
    if (slice.count() < kMostTop) {  // a list of fewer than are asked for ends in zeros
        for (int i = tid; i < kMostTop; i += P) sh.best[i] = 0;
        team_sync<P>();
    }
    for (int i = tid; i < n; i += P) {
        const uint64_t c = sh.found[i];
        int above = 0;
        for (int j = 0; j < n; ++j) above += sh.found[j] > c;
        if (above < want) sh.best[above] = c;
    }
}

// All CTAs of the cluster have started: said at the start, waited for before their memory is written.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

template <typename T, int P>
__global__ void __launch_bounds__(P == 32 ? 128 : P, P == 32 ? 0 : kResident) k_log_probabilities(const __grid_constant__ ScoreArgs a) {
    constexpr int V = Slice<T>::V, kEach = kParts / P, kWarps = P / 32, kTeams = P == 32 ? 4 : 1;
    // vectors of a thread under way: one of each of its parts, or some of its only one
    constexpr int kFlight = P == 32 ? kEach : sizeof(T) == 4 ? 4 : 2;
    __shared__ Shared<P> teams[kTeams];
    Shared<P> &sh = teams[P == 32 ? threadIdx.x / 32 : 0];
    const int tid = P == 32 ? threadIdx.x % 32 : threadIdx.x, warp = tid / 32, lane = tid % 32;
    if (P > 32 && a.ctas > 1) cluster_arrive();
    const int rank = P == 32 || a.ctas == 1 ? 0 : static_cast<int>(cg::this_cluster().block_rank());
    const int64_t r = P == 32 ? static_cast<int64_t>(blockIdx.x) * kTeams + threadIdx.x / 32 : blockIdx.x / a.ctas;
    if (P == 32 && r >= a.rows) return;
    const Slice<T> slice(a, r, rank);
    Sums mine = {-INFINITY, 0.f, 0.f};
    float largest[kEach];  // of the parts
#pragma unroll
    for (int i = 0; i < kEach; ++i) largest[i] = -INFINITY;
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
    // a group of vectors is under way while the one before it is worked on
    Vector<T> now[kFlight];
    auto load = [&](int v) {
#pragma unroll
        for (int f = 0; f < kFlight; ++f) {
            if (v + f * P < slice.v1) now[f] = slice.load(v + f * P);
            else now[f].clear();
        }
    };
    load(slice.v0 + tid);
    // the given tokens' logits come early too
    int given = -1;
    float given_logit = 0.f;
    if (rank == 0 && tid < a.given) {
        given = a.tokens[r * a.token_row + tid];
        if (static_cast<unsigned>(given) < static_cast<unsigned>(a.vocab)) given_logit = widen(slice.row + given);
    }
    slice.singles(tid, [&](int, float x) {
        largest[0] = fmaxf(largest[0], x);
        grow(x);
        add(x);
    });
#pragma unroll 1
    for (int v = slice.v0 + tid; v - tid < slice.v1; v += kFlight * P) {
        Vector<T> x[kFlight];
#pragma unroll
        for (int f = 0; f < kFlight; ++f) x[f].raw = now[f].raw;
        load(v + kFlight * P);
        float all = -INFINITY;
#pragma unroll
        for (int f = 0; f < kFlight; ++f) {
            float top = x[f][0];
#pragma unroll
            for (int j = 1; j < V; ++j) top = fmaxf(top, x[f][j]);
            if (kEach > 1) largest[f % kEach] = fmaxf(largest[f % kEach], top);
            all = fmaxf(all, top);
        }
        grow(all);
        Pair s = {make_float2(mine.s, 0.f)}, sa = {make_float2(mine.a, 0.f)};
        const Pair minus = both(-from), log2e = both(kLog2e);
#pragma unroll
        for (int f = 0; f < kFlight; ++f)
#pragma unroll
            for (int j = 0; j < V; j += 2) {
                Pair d = add2({make_float2(x[f][j], x[f][j + 1])}, minus), e = mul2(d, log2e);
                e.f = make_float2(ex2(e.f.x), ex2(e.f.y));
                s = add2(s, e);
                d.f = make_float2(fmaxf(d.f.x, -kFar), fmaxf(d.f.y, -kFar));
                sa = fma2(e, d, sa);
            }
        mine.s = s.f.x + s.f.y;
        mine.a = sa.f.x + sa.f.y;
    }
    if (kEach == 1) largest[0] = mine.top;
    if (P > 32 && a.ctas == 1 && tid == 0 && r + a.ahead < a.rows) {
        // the start of the row that the next CTA here will read, to L2 while this one's is worked out
        const uintptr_t next = (reinterpret_cast<uintptr_t>(a.logits + (r + a.ahead) * a.row_bytes) + 15) / 16 * 16;
        const uint32_t bytes = min(kAhead, (static_cast<uint32_t>(a.vocab) * static_cast<uint32_t>(sizeof(T)) - 15) / 16 * 16);
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(next), "r"(bytes) : "memory");
    }
    // the row's sums: of a warp, all against its maximum
    auto reduce = [](Sums &x) {
        const float top = warp_max(x.top), by = x.top - top, c = ex2(by * kLog2e);
        const bool none = x.top == -INFINITY;  // nothing to move; s may be the NaN of a NaN
        x.a = warp_sum(none ? x.a : c * fmaf(x.s, fmaxf(by, -kFar), x.a));
        x.s = warp_sum(none ? x.s : x.s * c);
        x.top = top;
    };
    reduce(mine);
    if (lane == 0) sh.sums[warp] = mine;
    if (a.top) choose<T, P>(slice, sh, tid, largest, min(a.top, slice.count()));
    team_sync<P>();
    Sums *parts = sh.sums;
    if (P > 32 && a.ctas > 1) {
        // every CTA's results to the first one's memory; all have started
        cluster_wait();
        Shared<P> *root = cg::this_cluster().map_shared_rank(&sh, 0);
        for (int i = tid; i < a.top; i += P) root->all[rank * a.top + i] = sh.best[i];
        if (tid < kWarps) root->parts[rank * kWarps + tid] = sh.sums[tid];
        cg::this_cluster().sync();
        if (rank) return;
        parts = sh.parts;
        // the place of each among all: how many of each falling list are larger, by halving, all lists at once
        int widest = 1;
        while (widest * 2 <= a.top) widest *= 2;
        for (int i = tid; i < a.ctas * a.top; i += P) {
            const uint64_t c = sh.all[i];
            int larger[kMostCtas] = {};
            for (int w = widest; w; w >>= 1)
#pragma unroll
                for (int l = 0; l < kMostCtas; ++l)
                    if (l < a.ctas && larger[l] + w <= a.top && sh.all[l * a.top + larger[l] + w - 1] > c) larger[l] += w;
            int above = 0;
#pragma unroll
            for (int l = 0; l < kMostCtas; ++l) above += larger[l];
            if (c && above < a.top) sh.best[above] = c;
        }
    }
    if (warp == kWarps - 1 && P > 32) {
        static_assert(kWarps * kMostCtas <= 32, "a sum a lane");
        Sums x = {-INFINITY, 0.f, 0.f};
        if (lane < kWarps * a.ctas) x = parts[lane];
        reduce(x);
        if (lane == 0) sh.total = x;
    }
    team_sync<P>();
    const Sums all = P == 32 ? mine : sh.total;
    const float log_s = logf(all.s);
    // a row of -inf alone: -inf, and no entropy
    auto log_p = [&](float x) { return all.s == 0.f ? -INFINITY : x - all.top - log_s; };
    if (a.entropy && tid == 0) a.entropy[r * a.entropy_row] = all.s == 0.f ? 0.f : log_s - all.a / all.s;
    auto put = [&](int i, int token, float x) {
        a.logprobs[r * a.logprob_row + i] = static_cast<unsigned>(token) < static_cast<unsigned>(a.vocab) ? log_p(x) : 0.f;
    };
    if (tid < a.given) put(tid, given, given_logit);
    for (int i = tid + P; i < a.given; i += P) {
        const int t = a.tokens[r * a.token_row + i];
        put(i, t, static_cast<unsigned>(t) < static_cast<unsigned>(a.vocab) ? widen(slice.row + t) : 0.f);
    }
    for (int i = tid; i < a.top; i += P) {
        const uint64_t c = sh.best[i];
        a.top_tokens[r * a.top_token_row + i] = token_of(c);
        a.top_logprobs[r * a.top_logprob_row + i] = log_p(value_of(static_cast<uint32_t>(c >> 32)));
    }
}

template <typename T>
int launch(mr_context *ctx, ScoreArgs &a) {
    // Short rows are a warp's, and where there are more than four an SM those of up to 64 KB, in float32 52, and 32 bytes
    // for each row that there is (us of a warp and of a CTA each: 4096 rows of 4000 float32 23 and 41, of 12000 52 and 55, of
    // 16000 69 and 64; of 32000 bfloat16 72 and 83; 1000 of 8000 float32 13.1 and 14.4, of 32000 bfloat16 28.2 and 25.5).
    // A longer one's CTAs: as many as give the GPU four an SM, each with two vectors a thread at least.
    a.ctas = 1;
    a.ahead = kResident * ctx->sm_count;
    const int64_t bytes = a.vocab * static_cast<int64_t>(sizeof(T)), most = (sizeof(T) == 4 ? 52 : 64) << 10;
    if (a.vocab <= 1024 || (a.rows > 4 * ctx->sm_count && bytes <= std::min(most, 32 * a.rows))) {
        k_log_probabilities<T, 32><<<static_cast<unsigned>((a.rows + 3) / 4), 128, 0, ctx->stream>>>(a);
        MR_CUDA_TRY(cudaGetLastError());
        return MR_OK;
    }
    while (a.ctas < kMostCtas && a.rows * a.ctas * 2 <= 4 * ctx->sm_count &&
           a.vocab / Slice<T>::V >= 2 * kParts * a.ctas * 2)
        a.ctas *= 2;
    cudaLaunchAttribute cluster;
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = a.ctas;
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(a.rows * a.ctas));
    config.blockDim = dim3(256);
    config.stream = ctx->stream;
    config.attrs = &cluster;
    config.numAttrs = a.ctas > 1;
    MR_CUDA_TRY(cudaLaunchKernelEx(&config, k_log_probabilities<T, 256>, a));
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
    a.rows = rows;
    return logits->dtype == MR_DTYPE_F32   ? launch<float>(ctx, a)
           : logits->dtype == MR_DTYPE_F16 ? launch<__half>(ctx, a)
                                           : launch<__nv_bfloat16>(ctx, a);
}
