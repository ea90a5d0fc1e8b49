// Attention of packed prompts: causal, optionally in a sliding window with a few
// first rows that stay visible.
//
//   p = m - n + i   (query i of a sequence of n queries and m keys)
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j  over the j that query i sees:
//           j <= p and (no window, or p - j < window, or j < sinks).
//
// 16-bit types run on the 5th-generation tensor cores (k_window).  A CTA works on
// two tiles of 128 query rows (128 / group tokens x the group's heads: the heads
// share their keys, and a tile of few tokens wastes little at the mask's edges)
// over the 128-key tiles that any of their rows sees; keys between the sinks and
// the windows are skipped.  Warp roles: warps 0-3 and 4-7 the softmax of one query
// tile each (a thread a row, so a row's maximum and sum need no exchange), warp 8
// the TMA loads, warps 9 and 10 the products of one query tile each.  S = Q K^T and
// O += P V accumulate in TMEM (S of both tiles 2 x 128 columns, O of both behind); P,
// rounded to the operands' type, goes back to TMEM over its own S and is the first
// operand of the second product, V the second one as it lies in memory (MN-major).
// O is rescaled only where a row's maximum grows by more than 2^8: until then the
// weights are taken against the old maximum, which the sum shares, so nothing is lost
// but headroom (Headroom: float16 has less of it).
//
// What bounds it: a 128 x 128 tile's exponentials (head dim 128) take the special-function
// unit 1024 cycles, its two products the tensor cores as many.  One tile's softmax runs
// beside the other's products; with two softmax warps a scheduler, each unit is busy 57% of
// the time (ncu, flashlite's 8192-token context; 239 us in a CUDA graph, 1.15 PFLOP/s).  Measured and left out:
// a quarter of the exponentials by polynomials (no faster at head dim 64, 15% slower at 128),
// key tiles of 64 with the next scores worked out ahead (290 us), two threads a row (314 us),
// P beside S where TMEM has room (head dim 64: no difference).
//
// A weight is 0 where the mask hides a key, but 0 x NaN is NaN: a row whose values are
// not all finite at the end is worked out again from the visible keys alone
// (row_alone), so that what a mask hides, also in other sequences, never matters.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <cmath>
#include <type_traits>

#include "cache_ops.cuh"
#include "tcgen05.cuh"

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
    int *gave_up;    // host word of the context
    uint64_t limit;  // of a wait: the context's, and what a warp may take to work 32 rows out again alone
    int withhold;    // fault injection: no values are loaded
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

// One query row's attention by one warp, four values of a row a lane: row i of the
// sequence, head h.
template <typename T>
__device__ void row_alone(const WindowArgs &a, const Span &x, int i, int h) {
    const int lane = threadIdx.x % 32;
    auto load = [&](const char *row, float (&y)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            y[j] = 4 * lane + j < a.dim ? widen(reinterpret_cast<const T *>(row) + 4 * lane + j) : 0.f;
    };
    const int p = x.m - x.n + i, kh = h / a.group;
    float q[4], o[4] = {}, m = -INFINITY, l = 0.f;
    load(a.q + (x.q0 + i) * a.q_row + h * a.q_head, q);
    for (int j = 0; j <= p; ++j) {
        if (a.window && p - j >= a.window && j >= a.sinks) {
            j = p - a.window;
            continue;
        }
        float k[4], v[4];
        load(a.k + (x.k0 + j) * a.k_row + kh * a.k_head, k);
        load(a.v + (x.k0 + j) * a.v_row + kh * a.v_head, v);
        const float y = warp_sum(q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3]) * a.scale;
        const float top = fmaxf(m, y), ref = top == -INFINITY ? 0.f : top, c = expf(m - ref), w = expf(y - ref);
        l = l * c + w;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = o[e] * c + w * v[e];
        m = top;
    }
    T *out = reinterpret_cast<T *>(a.out + (x.q0 + i) * a.o_row + h * a.o_head);
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (4 * lane + j < a.dim) narrow(l != 0.f ? o[j] / l : 0.f, out + 4 * lane + j);
}

// A warp per (query row, head).
template <typename T>
__global__ void __launch_bounds__(128) k_rows(const __grid_constant__ WindowArgs a) {
    const int64_t id = blockIdx.x * static_cast<int64_t>(4) + threadIdx.x / 32;
    const int i = static_cast<int>(id / a.heads), h = static_cast<int>(id % a.heads);
    if (i >= a.tokens) return;
    int s = 0;
    Span x = {};
    for (; s < a.batch; ++s) {
        x = span_of(a, s);
        if (i >= x.q0 && i < x.q0 + x.n) break;
    }
    if (s < a.batch) row_alone<T>(a, x, i - x.q0, h);
}

// ---- tensor cores -----------------------------------------------------------------
// Powers of two: how far a weight may pass its reference, and the reference below the maximum
// that it was taken from.  A float16 weight ends at 2^16, and half its smallest step is
// 2^-25: against a reference of 2^-11 of the maximum, small weights are off by 2^-36 of the largest
// (2^-25 without: 8192 rows of 2^-25.2 beside one, 2e-4 of the sum, were lost).  The less a weight may
// grow, the more often O is rescaled: flashlite's 8192 tokens take 242.9 us with 2^8 and 2^7, 246.8
// with 2^4 and 2^11, 258.7 with 2^2 and 2^13.
template <typename T>
struct Headroom {
    static constexpr float kGrows = std::is_same<T, __half>::value ? 4.f : 8.f;
    static constexpr float kLift = std::is_same<T, __half>::value ? 11.f : 0.f;
};
constexpr int kTile = 128, kKeys = 128;  // query rows and keys of a tile
constexpr int kLoadWarp = 8, kMathWarp = 9, kTcThreads = 384;  // warp 11 fills the third warpgroup
// bytes of 64 dims of a tile's queries, and of its keys
constexpr uint32_t kHalfQ = kTile * 128, kHalfK = kKeys * 128;

template <int DP>
struct Shape {
    static constexpr int kHalves = DP / 64;
    static constexpr uint32_t kQBytes = kHalves * kHalfQ, kStageBytes = kHalves * kHalfK;
    static constexpr int kStages = DP == 128 ? 5 : 8;
    static constexpr uint32_t kSmem = 1024 + 2 * kQBytes + kStages * kStageBytes + 512;
    static constexpr uint32_t kO = 2 * kTile;  // TMEM columns: S0, S1, O0, O1
};

struct Maps {
    CUtensorMap q, k, v;
};

// Shared memory behind the tiles.
struct Barriers {
    uint64_t q_full, q_empty, kv_full[8], kv_empty[8], s_full[2], p_half[2], p_full[2], o_done[2], turn[2], drained[2];
    uint32_t tmem;
    int stop;  // a wait gave up: every role leaves
};

// A bounded wait; false when it gives up, or another role has.
__device__ __forceinline__ bool wait_for(uint64_t *bar, int parity, Barriers *b, int *gave_up, uint64_t limit) {
    if (tc::try_wait(bar, parity)) return true;
    const uint64_t start = tc::now();
    for (unsigned spin = 1;; ++spin) {
        if (tc::try_wait(bar, parity)) return true;
        if (spin % 64 == 0) {
            if (*reinterpret_cast<volatile int *>(&b->stop)) return false;
            if (tc::now() - start > limit) {
                *reinterpret_cast<volatile int *>(&b->stop) = 1;
                *reinterpret_cast<volatile int *>(gave_up) = 1;
                return false;
            }
        }
    }
}
// The same by a whole warp, which goes on or gives up together.
__device__ __forceinline__ bool warp_wait_for(uint64_t *bar, int parity, Barriers *b, int *gave_up, uint64_t limit) {
    return __all_sync(0xffffffffu, wait_for(bar, parity, b, gave_up, limit));
}
// A bounded wait for what is in flight, whoever has given up; `unless`: where it may not come.
__device__ __forceinline__ void wait_in_flight(uint64_t *bar, int parity, uint64_t start, volatile int *unless = nullptr) {
    while (!tc::try_wait(bar, parity) && !(unless && *unless) && tc::now() - start < tc::kWaitNs) {
    }
}
// One lane of a converged warp.
__device__ __forceinline__ bool elect() {
    uint32_t yes;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(yes));
    return yes != 0;
}
__device__ __forceinline__ void arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tc::saddr(bar)) : "memory");
}
__device__ __forceinline__ void expect(uint64_t *bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(tc::saddr(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap *map, int x, int head, int row, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(head), "r"(row), "r"(tc::saddr(bar))
        : "memory");
}
// D (+)= A B^T with A in TMEM (two 16-bit values a column).
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
}
// An operand tile as rows of 64 contiguous values of the operand's outer (not summed)
// dimension, 128-byte swizzle: 8-row groups 1024 bytes apart, the next 64 values a half on.
__device__ __forceinline__ uint64_t mn_desc(uint32_t addr) {
    return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(kHalfK >> 4) << 16) |
           (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}
// Instruction descriptor: D float32, A and B of one 16-bit type; A negated; B MN-major.
__device__ __forceinline__ uint32_t mma_desc(bool bf16, int n, bool negate, bool b_mn) {
    const uint32_t type = bf16 ? 1u : 0u;
    return (1u << 4) | (type << 7) | (type << 10) | ((negate ? 1u : 0u) << 13) | ((b_mn ? 1u : 0u) << 16) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kTile >> 4) << 24);
}
#define MR_R8(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]), "=r"(v[i + 4]), "=r"(v[i + 5]), "=r"(v[i + 6]), "=r"(v[i + 7])
#define MR_I8(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]), "r"(v[i + 4]), "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7])
// 32 columns of this thread's lane, not waited for (settle).
__device__ __forceinline__ void tmem_get(uint32_t addr, uint32_t *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : MR_R8(v, 0), MR_R8(v, 8), MR_R8(v, 16), MR_R8(v, 24)
        : "r"(addr));
}
__device__ __forceinline__ void tmem_put(uint32_t addr, const uint32_t *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::MR_I8(v, 0),
        MR_I8(v, 8), MR_I8(v, 16), MR_I8(v, 24), "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_get16(uint32_t addr, uint32_t *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : MR_R8(v, 0), MR_R8(v, 8)
        : "r"(addr));
}
__device__ __forceinline__ void tmem_put16(uint32_t addr, const uint32_t *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::MR_I8(v, 0),
        MR_I8(v, 8), "r"(addr)
        : "memory");
}
// Waits for the loads before it; the values may be used behind it only.
template <int N>
__device__ __forceinline__ void settle(uint32_t (&v)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(v[i]));
}
__device__ __forceinline__ float pow2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two float32 operations as one instruction.
__device__ __forceinline__ uint64_t bits_of(float2 x) {
    uint64_t y;
    asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(x.x), "f"(x.y));
    return y;
}
__device__ __forceinline__ float2 floats_of(uint64_t x) {
    float2 y;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(y.x), "=f"(y.y) : "l"(x));
    return y;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(bits_of(a)), "l"(bits_of(b)), "l"(bits_of(c)));
    return floats_of(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits_of(a)), "l"(bits_of(b)));
    return floats_of(d);
}
// The lowest n of 32 bits.
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }
__device__ __forceinline__ float max_nan(float x, float y) {  // NaN if one is
    float z;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
    return z;
}
__device__ __forceinline__ uint32_t pair_of(float x, float y, __nv_bfloat16) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&p);
}
__device__ __forceinline__ uint32_t pair_of(float x, float y, __half) {
    const __half2 p = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&p);
}

// A CTA's work: queries t0 .. of sequence `x`, KV head `kh`, and the tiles of KEYS keys they see:
// `front` tiles of the sinks, keys 0 .. edge - 1, and from key `first` on, where their windows
// begin (no tile boundary: a window of 512 over 64 queries is five tiles of 128 wherever it lies).
template <int KEYS>
struct Item {
    Span x;
    int kh, t0, count;         // first query, queries
    int front, edge, first, tiles;
    __device__ __forceinline__ int key(int j) const { return j < front ? j * KEYS : first + (j - front) * KEYS; }
    // Past the last key of tile j that any query may see there.
    __device__ __forceinline__ int past(int j) const { return j < front ? edge : INT32_MAX; }
};
// The items of a call, in falling order of their tiles' numbers, so that the longest of a
// causal prompt start first; `most` queries each.  Whole warps.
template <int KEYS>
struct Items {
    int most, pairs;   // items of one KV head
    int64_t total;
    int mine, sum;     // of sequence `lane`, and of those up to it (32 sequences at most; else found again for each item)
    __device__ __forceinline__ int of(const WindowArgs &a, int s) const {
        return s < a.batch ? (span_of(a, s).n + most - 1) / most : 0;
    }
    static __device__ __forceinline__ int scan(int x) {
        const int lane = threadIdx.x % 32;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int below = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += below;
        }
        return x;
    }
    __device__ __forceinline__ void init(const WindowArgs &a, int queries) {
        const int lane = threadIdx.x % 32;
        most = queries;
        mine = of(a, lane);
        pairs = mine;
        for (int s = lane + 32; s < a.batch; s += 32) pairs += of(a, s);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) pairs += __shfl_xor_sync(0xffffffffu, pairs, o);
        total = static_cast<int64_t>(max(pairs, 0)) * a.kv_heads;
        sum = scan(mine);
    }
    __device__ __forceinline__ bool get(const WindowArgs &a, int64_t index, Item<KEYS> &it) const {
        if (index >= total) return false;
        const int lane = threadIdx.x % 32;
        const int pair = pairs - 1 - static_cast<int>(index / a.kv_heads);
        it.kh = static_cast<int>(index % a.kv_heads);
        int base = 0, s = -1;
        for (int s0 = 0; s0 < a.batch; s0 += 32) {
            const int here = a.batch <= 32 ? mine : of(a, s0 + lane), upto = a.batch <= 32 ? sum : scan(here);
            const uint32_t past = __ballot_sync(0xffffffffu, base + upto > pair);
            if (past) {
                const int l = __ffs(past) - 1;
                s = s0 + l;
                base += __shfl_sync(0xffffffffu, upto - here, l);
                break;
            }
            base += __shfl_sync(0xffffffffu, upto, 31);
        }
        if (s < 0) return false;  // offsets that overlap so far that their sum wraps
        it.x = span_of(a, s);
        it.t0 = (pair - base) * most;
        it.count = min(most, it.x.n - it.t0);
        const int low = it.x.m - it.x.n + it.t0, high = low + it.count - 1;  // their positions
        it.front = it.edge = it.first = it.tiles = 0;
        if (high < 0) return true;
        const int start = a.window ? max(0, low - a.window + 1) : 0;  // the first key in a window
        if (a.sinks < start) {  // keys between that no query sees
            it.edge = a.sinks;
            it.front = (a.sinks + KEYS - 1) / KEYS;
            it.first = start;
        }
        it.tiles = it.front + (high - it.first) / KEYS + 1;
        return true;
    }
};

// ---- float32 ------------------------------------------------------------------------
// On the CUDA cores, in float32 throughout (the tensor cores would need three parts of
// every operand): a CTA takes ROWS query rows (ROWS / group tokens x the group's heads) over
// tiles of 32 keys.  A thread has ROWS / 8 rows x 2 keys of the scores, and as many rows x
// DP / 16 dims of the values; the weights pass through shared memory between the two.  A
// tile's values arrive while its scores are worked out, the next keys while the values are
// mixed.  64 rows read shared memory least often for a product; where they would leave SMs
// without a CTA, 32 rows, with the next keys asked for a tile earlier (two buffers).
// Rows ty, ty + 8, ..: the two rows that a warp reads at once lie in different banks.
constexpr int kKeys32 = 32, kThreads32 = 128;

__device__ __forceinline__ void copy16(void *dst, const void *src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tc::saddr(dst)), "l"(src), "r"(live ? 16 : 0) : "memory");
}

template <int DP, int ROWS>
struct Shared32 {
    static constexpr int kBuffers = ROWS == 32 ? 2 : 1;
    float q[ROWS][DP + 4], k[kBuffers][kKeys32][DP + 4], v[kKeys32][DP], p[kKeys32][ROWS + 4];
};

template <int DP, int ROWS>
__global__ void __launch_bounds__(kThreads32, 3) k_window32(const __grid_constant__ WindowArgs a) {
    extern __shared__ __align__(16) char raw32[];
    using Shared = Shared32<DP, ROWS>;
    Shared &sm = *reinterpret_cast<Shared *>(raw32);
    constexpr int kMine = ROWS / 8, kAhead = Shared::kBuffers - 1;  // a thread's rows; tiles the keys run ahead
    constexpr int kVec = DP >= 64 ? 4 : 2, kVecs = DP / 16 / kVec;  // a thread's dims: kVecs pieces of kVec
    const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
    const int per = ROWS / a.group;
    Items<kKeys32> items;
    items.init(a, per);
    Item<kKeys32> it;
    if (!items.get(a, blockIdx.x, it)) return;
    auto rows_in = [&](auto &to, const char *base, int64_t stride, int tile) {  // a tile's keys or values; zeros past the end
        for (int e = tid; e < kKeys32 * DP / 4; e += kThreads32) {
            const int r = e / (DP / 4), c = e % (DP / 4), row = it.key(tile) + r;
            const bool live = row < it.x.m && 4 * c < a.dim;
            copy16(&to[r][4 * c], live ? base + (it.x.k0 + row) * stride + c * 16 : base, live);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const char *kb = a.k + it.kh * a.k_head, *vb = a.v + it.kh * a.v_head;
    for (int e = tid; e < ROWS * DP / 4; e += kThreads32) {
        const int r = e / (DP / 4), c = e % (DP / 4), t = r / a.group, g = r - t * a.group;
        const bool live = t < per && t < it.count && 4 * c < a.dim;
        copy16(&sm.q[r][4 * c],
               live ? a.q + (it.x.q0 + it.t0 + t) * a.q_row + (it.kh * a.group + g) * a.q_head + c * 16 : a.q, live);
    }
    if (it.tiles > 0) rows_in(sm.k[0], kb, a.k_row, 0);
    const float scale = a.scale * 1.4426950408889634f;
    float m[kMine], l[kMine];
    float2 o[kMine][DP / 32];
    int pos[kMine];  // the rows' positions; -1: no row
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        const int r = ty + 8 * i, t = r / a.group;
        pos[i] = t < per && t < it.count ? it.x.m - it.x.n + it.t0 + t : -1;
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) o[i][d] = make_float2(0.f, 0.f);
    }
    for (int j = 0; j < it.tiles; ++j) {
        rows_in(sm.v, vb, a.v_row, j);
        if (kAhead) {
            if (j + 1 < it.tiles) rows_in(sm.k[(j + 1) % Shared::kBuffers], kb, a.k_row, j + 1);
            else asm volatile("cp.async.commit_group;" ::: "memory");
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(1 + kAhead) : "memory");
        __syncthreads();  // the keys are there
        const auto &keys = sm.k[j % Shared::kBuffers];
        float2 dot[kMine][2] = {};  // of the even and the odd pairs' dims
#pragma unroll 2
        for (int d = 0; d < DP; d += 4) {
            float4 k[2];
#pragma unroll
            for (int y = 0; y < 2; ++y) k[y] = *reinterpret_cast<const float4 *>(&keys[tx + 16 * y][d]);
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const float4 q = *reinterpret_cast<const float4 *>(&sm.q[ty + 8 * i][d]);
#pragma unroll
                for (int y = 0; y < 2; ++y)
                    dot[i][y] = fma2(make_float2(q.z, q.w), make_float2(k[y].z, k[y].w),
                                     fma2(make_float2(q.x, q.y), make_float2(k[y].x, k[y].y), dot[i][y]));
            }
        }
        float s[kMine][2];
        const int first = it.key(j) + tx, past = it.past(j);
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            float top = -INFINITY;
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const int key = first + 16 * y;
                const bool seen = key <= pos[i] && key < past && (a.window == 0 || pos[i] - key < a.window || key < a.sinks);
                s[i][y] = seen ? (dot[i][y].x + dot[i][y].y) * scale : -INFINITY;
                top = fmaxf(top, s[i][y]);
            }
#pragma unroll
            for (int w = 8; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
            top = fmaxf(top, m[i]);
            const float ref = top == -INFINITY ? 0.f : top, c = pow2(m[i] - ref);
            m[i] = top;
#pragma unroll
            for (int y = 0; y < 2; ++y) s[i][y] = pow2(s[i][y] - ref);
            l[i] = fmaf(l[i], c, s[i][0] + s[i][1]);
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) o[i][d] = make_float2(o[i][d].x * c, o[i][d].y * c);
        }
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int i = 0; i < kMine; i += 4)
                *reinterpret_cast<float4 *>(&sm.p[tx + 16 * y][ty * kMine + i]) = make_float4(s[i][y], s[i + 1][y], s[i + 2][y], s[i + 3][y]);
        asm volatile("cp.async.wait_group %0;" ::"n"(kAhead) : "memory");
        __syncthreads();  // the values and all weights are there, the keys are done with
        if (!kAhead && j + 1 < it.tiles) rows_in(sm.k[0], kb, a.k_row, j + 1);
#pragma unroll 4
        for (int key = 0; key < kKeys32; ++key) {
            float p[kMine];
            float2 v[DP / 32];
#pragma unroll
            for (int i = 0; i < kMine; i += 4)
                *reinterpret_cast<float4 *>(p + i) = *reinterpret_cast<const float4 *>(&sm.p[key][ty * kMine + i]);
#pragma unroll
            for (int d = 0; d < kVecs; ++d) {
                const float *at = &sm.v[key][d * 16 * kVec + tx * kVec];
                if (kVec == 4) {
                    const float4 x = *reinterpret_cast<const float4 *>(at);
                    v[2 * d] = make_float2(x.x, x.y);
                    v[2 * d + 1] = make_float2(x.z, x.w);
                } else {
                    v[d] = *reinterpret_cast<const float2 *>(at);
                }
            }
#pragma unroll
            for (int i = 0; i < kMine; ++i)
#pragma unroll
                for (int d = 0; d < DP / 32; ++d) o[i][d] = fma2(make_float2(p[i], p[i]), v[d], o[i][d]);
        }
        __syncthreads();  // the values and weights are done with
    }
    uint32_t again = 0;  // rows with values that are not finite
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], w);
        const int r = ty + 8 * i, t = r / a.group, g = r - t * a.group;
        const float f = l[i] != 0.f ? 1.f / l[i] : 0.f;
        bool finite = true;
        float *out = reinterpret_cast<float *>(a.out + (it.x.q0 + it.t0 + t) * a.o_row + (it.kh * a.group + g) * a.o_head);
#pragma unroll
        for (int d = 0; d < kVecs; ++d)
#pragma unroll
            for (int e = 0; e < kVec; e += 2) {
                const float2 y = o[i][(d * kVec + e) / 2], x = make_float2(y.x * f, y.y * f);
                const int dim = d * 16 * kVec + tx * kVec + e;
                finite &= fabsf(x.x) < INFINITY && fabsf(x.y) < INFINITY;
                if (t < per && t < it.count && dim < a.dim) *reinterpret_cast<float2 *>(out + dim) = x;
            }
        if (!finite && t < per && t < it.count) again |= 1u << i;
    }
    // the rows of both halves of the warp, as any lane of a half says
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) again |= __shfl_xor_sync(0xffffffffu, again, w);
    __syncwarp();  // the rows' first stores come before their second ones, which other lanes make
    for (int half = 0; half < 2; ++half)
        for (uint32_t left = __shfl_sync(0xffffffffu, again, half * 16); left; left &= left - 1) {
            const int r = tid / 32 * 2 + half + 8 * (__ffs(left) - 1), t = r / a.group;
            row_alone<float>(a, it.x, it.t0 + t, it.kh * a.group + r - t * a.group);
        }
}

// A CTA's items: one of each round of as many as there are CTAs, forwards and backwards in
// turn, so that who has a round's longest has the next one's shortest.
__device__ __forceinline__ int64_t item_of(int round) {
    return static_cast<int64_t>(round) * gridDim.x + (round & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}

// kRounds: a CTA takes items of several rounds; else one.  (A body of its own: the loop around
// everything cost 6% where items are long.)
template <typename T, int DP, bool kRounds>
__global__ void __launch_bounds__(kTcThreads, 1) k_window(const __grid_constant__ WindowArgs a,
                                                          const __grid_constant__ Maps maps) {
    using S = Shape<DP>;
    extern __shared__ uint8_t raw[];
    uint8_t *tiles = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    Barriers *b = reinterpret_cast<Barriers *>(tiles + 2 * S::kQBytes + S::kStages * S::kStageBytes);
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const int per = kTile / a.group;  // tokens of a query tile
    if (tid == 0) {
        auto init = [](uint64_t *bar, int count) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(tc::saddr(bar)), "r"(count) : "memory");
        };
        init(&b->q_full, 1);
        init(&b->q_empty, 2);
        for (int i = 0; i < S::kStages; ++i) {
            init(&b->kv_full[i], 1);
            init(&b->kv_empty[i], 2);
        }
        for (int i = 0; i < 2; ++i) {
            init(&b->s_full[i], 1);
            init(&b->p_half[i], 4);
            init(&b->p_full[i], 4);
            init(&b->o_done[i], 1);
            init(&b->turn[i], 4);
            init(&b->drained[i], 1);
        }
        b->stop = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMathWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tc::saddr(&b->tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == kLoadWarp && lane < 3)
        asm volatile("prefetch.tensormap [%0];" ::"l"(lane == 0 ? &maps.q : lane == 1 ? &maps.k : &maps.v) : "memory");
    Items<kKeys> items;
    items.init(a, 2 * per);
    const uint64_t limit = a.limit;
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = b->tmem, q_tiles = tc::saddr(tiles), stages = q_tiles + 2 * S::kQBytes;
    Item<kKeys> it;
    bool ok = true;
    // 384 threads start with 168 registers each; a softmax thread holds a row of 128 scores
    // and takes 216, of what the third warpgroup gives: 2 x 216 + 72 = 3 x 168.
    if (warp >= kLoadWarp) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == kLoadWarp) {
        int issued = 0, count = 0;  // stages and items with tiles so far
        for (int round = 0; (kRounds || round == 0) && ok && items.get(a, item_of(round), it); ++round) {
            if (it.tiles == 0) continue;
            if (lane == 0) {
                // Q once the last item's products with it are done
                ok = count == 0 || wait_for(&b->q_empty, (count - 1) & 1, b, a.gave_up, limit);
                if (ok) {
                    expect(&b->q_full, 2 * S::kHalves * per * a.group * 128);
                    for (int w = 0; w < 2; ++w)
                        for (int h = 0; h < S::kHalves; ++h)
                            load_box(q_tiles + w * S::kQBytes + h * kHalfQ, &maps.q, h * 64, it.kh * a.group,
                                     it.x.q0 + it.t0 + w * per, &b->q_full);
                    ++count;
                }
                // K0, V0, K1, V1, ... through the stages
                auto load = [&](const CUtensorMap *map, int j) {
                    const int st = issued % S::kStages, use = issued / S::kStages;
                    if (use > 0 && !wait_for(&b->kv_empty[st], (use - 1) & 1, b, a.gave_up, limit)) return false;
                    expect(&b->kv_full[st], S::kStageBytes);
                    for (int h = 0; h < S::kHalves; ++h)
                        load_box(stages + st * S::kStageBytes + h * kHalfK, map, h * 64, it.kh,
                                 it.x.k0 + it.key(j), &b->kv_full[st]);
                    ++issued;
                    return true;
                };
                for (int j = 0; j < it.tiles && ok; ++j) ok = load(&maps.k, j) && !a.withhold && load(&maps.v, j);
            }
            ok = __shfl_sync(0xffffffffu, ok, 0);
        }
        if (lane == 0) {
            // no copy may land after the CTA has left (the last stages; those before were waited for by the products),
            // and no arrival of the products
            const uint64_t start = tc::now();
            if (count > 0) wait_in_flight(&b->q_full, (count - 1) & 1, start);
            for (int i = max(0, issued - S::kStages); i < issued; ++i)
                wait_in_flight(&b->kv_full[i % S::kStages], (i / S::kStages) & 1, start);
            if (count > 0) wait_in_flight(&b->q_empty, (count - 1) & 1, start, &b->stop);
            for (int i = max(0, issued - S::kStages); i < issued; ++i)
                wait_in_flight(&b->kv_empty[i % S::kStages], (i / S::kStages) & 1, start, &b->stop);
        }
    } else if (warp == kMathWarp || warp == kMathWarp + 1) {
        // A warp for each query tile, so that one's waits do not hold up the other's products.
        // All of it walks through them and one lane issues: descriptors stay in uniform
        // registers, where the instruction wants them.  A lane whose wait gave up issues nothing more
        // but walks on; the warp leaves together, by a vote once a step (0.3% of the time; a vote a wait: 1.5%).
        {
            constexpr bool kBf16 = sizeof(T) == 2 && !__is_same(T, __half);
            const uint32_t qk = mma_desc(kBf16, kKeys, a.scale < 0.f, false), pv = mma_desc(kBf16, DP, false, true);
            const int w = warp - kMathWarp;
            const uint64_t q = tc::sw128_desc(q_tiles + w * S::kQBytes), k_desc = tc::sw128_desc(stages), v_desc = mn_desc(stages);
            const uint32_t s_at = tmem + w * kTile, o_at = tmem + S::kO + w * DP;
            const bool leader = elect();
            int st = 0, fill = 0;  // the next stage, and the parity of its fill
            bool mine = true;      // none of this lane's waits gave up
            auto take = [&] {
                mine = mine && wait_for(&b->kv_full[st], fill, b, a.gave_up, limit);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            };
            auto leave = [&] {
                if (leader) tc::commit(&b->kv_empty[st]);
                __syncwarp();
                if (++st == S::kStages) {
                    st = 0;
                    fill ^= 1;
                }
            };
            auto scores = [&] {
                const uint64_t k = k_desc + st * (S::kStageBytes >> 4);
                if (leader && mine) {
#pragma unroll
                    for (int i = 0; i < DP / 16; ++i)
                        tc::mma(s_at, q + ((i / 4) * kHalfQ + (i % 4) * 32) / 16, k + ((i / 4) * kHalfK + (i % 4) * 32) / 16, qk,
                                i > 0);
                    tc::commit(&b->s_full[w]);
                }
                __syncwarp();
            };
            int count = 0, g = 0;  // items and steps so far
            for (int round = 0; (kRounds || round == 0) && ok && items.get(a, item_of(round), it); ++round) {
                const int n = it.tiles;
                if (n == 0) continue;
                mine = mine && wait_for(&b->q_full, count++ & 1, b, a.gave_up, limit);
                take();
                scores();
                if (n == 1 && leader) tc::commit(&b->q_empty);
                leave();
                for (int j = 0; j < n && ok; ++j, ++g) {
                    take();
                    const uint64_t v = v_desc + st * (S::kStageBytes >> 4);
                    // P comes in two halves; the first is multiplied while the second is worked out
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        mine = mine && wait_for(half ? &b->p_full[w] : &b->p_half[w], g & 1, b, a.gave_up, limit);
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        if (leader && mine) {
#pragma unroll
                            for (int i = half * kKeys / 32; i < (half + 1) * kKeys / 32; ++i)
                                mma_ts(o_at, s_at + i * 8, v + i * 128, pv, j > 0 || i > 0);
                            if (half) tc::commit(&b->o_done[w]);
                        }
                        __syncwarp();
                    }
                    leave();
                    if (j + 1 < n) {
                        take();
                        scores();
                        if (j + 2 == n && leader) tc::commit(&b->q_empty);
                        leave();
                    }
                    ok = __all_sync(0xffffffffu, mine);
                }
            }
            // no product may still run when the CTA gives its memory back, whatever made the warp leave
            if (leader) tc::commit(&b->drained[w]);
            __syncwarp();
            wait_in_flight(&b->drained[w], 0, tc::now());
            __syncwarp();
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        }
    } else if (warp < kLoadWarp) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int w = warp / 4, r = (warp & 3) * 32 + lane, tt = r / a.group, g = r - tt * a.group;
        int done = 0;  // steps so far
        for (int round = 0; (kRounds || round == 0) && ok && items.get(a, item_of(round), it); ++round) {
            const int n = it.tiles;
            const int i = it.t0 + w * per + tt;  // query of the sequence
            const bool live = tt < per && w * per + tt < it.count;
            const int p = live ? it.x.m - it.x.n + i : -1;
            // every row's position of this tile, for the tiles that need no mask
            const int p_low = it.x.m - it.x.n + it.t0 + w * per, p_high = p_low + min(per, it.count - w * per) - 1;
            const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
            const uint32_t s_at = tmem + lanes + w * kTile, o_at = tmem + lanes + S::kO + w * DP;
            const float scale = fabsf(a.scale) * 1.4426950408889634f;
            constexpr float kNone = -3.4028235e38f;  // no key seen yet
            // Rows of no query of the sequence (another's, or what shared memory held) have no say in when the
            // others' values are rescaled, and so rounded anew: their maximum cannot grow.
            float m = live ? kNone : INFINITY, l = 0.f;
            // A tile's step; where the mask hides some of its keys, its quarters of 32 keys that no row of
            // the warp sees are left out.  Two bodies: the scores of either stay in registers of its own.
            auto step = [&](int j, auto hides) {
                constexpr bool kHides = decltype(hides)::value;
                if (!warp_wait_for(&b->s_full[w], done & 1, b, a.gave_up, limit)) return false;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                uint32_t s[kKeys];
#pragma unroll
                for (int c = 0; c < kKeys; c += 32) tmem_get(s_at + c, s + c);
                settle(s);
                uint32_t used = 0;  // the quarters to work on
                if (kHides) {
                    const int kb = it.key(j), low = a.window ? p - kb - a.window + 1 : 0, front = a.sinks - kb;
                    const int high = min(p, it.past(j) - 1) - kb;
#pragma unroll
                    for (int c = 0; c < kKeys; c += 32) {
                        // a bit for each key that is seen: up to `high`, and from `low` on or in the sinks
                        const uint32_t seen = below(high + 1 - c) & (~below(low - c) | below(front - c));
                        if (__any_sync(0xffffffffu, seen)) used |= 1u << (c / 32);
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (!(seen & (1u << e))) s[c + e] = 0xff800000u;
                    }
                }
                float tops[8];
#pragma unroll
                for (int c = 0; c < 8; ++c) tops[c] = __uint_as_float(s[c]);
#pragma unroll
                for (int c = 8; c < kKeys; ++c) tops[c % 8] = max_nan(tops[c % 8], __uint_as_float(s[c]));
                const float top = max_nan(max_nan(max_nan(tops[0], tops[1]), max_nan(tops[2], tops[3])),
                                          max_nan(max_nan(tops[4], tops[5]), max_nan(tops[6], tops[7])));
                // (never of a NaN, whose row's values all become NaN)
                if (__any_sync(0xffffffffu, (top - m) * scale > Headroom<T>::kGrows)) {
                    const float grown = max_nan(m, top);
                    if (j > 0) {
                        // done already, since the scores came behind it
                        if (!warp_wait_for(&b->o_done[w], (done - 1) & 1, b, a.gave_up, limit)) return false;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const float c = m == grown ? 1.f : pow2((m - grown) * scale);
                        l *= c;
#pragma unroll
                        for (int d = 0; d < DP; d += 16) {
                            uint32_t o[16];
                            tmem_get16(o_at + d, o);
                            settle(o);
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * c);
                            tmem_put16(o_at + d, o);
                        }
                    }
                    m = grown;
                }
                const float shift = m == kNone ? 0.f : fmaf(-m, scale, Headroom<T>::kLift);
                // The two tiles take the special-function unit in turns, a quarter overlapping; otherwise both
                // settle into doing their exponentials, and then their products, at the same time
                // (chunked flashnano-1.7 prompts 35.1 us without, 34.0 with).
                if ((w == 1 || done > 0) && !warp_wait_for(&b->turn[w], (w == 1 ? done : done - 1) & 1, b, a.gave_up, limit))
                    return false;
                float2 sum[2] = {};
                // The weights, rounded to the operands' type: half a step each, at random, of sums
                // whose result is rounded to that type again.  The sum takes them unrounded.
                auto weigh = [&](int c) {
                    float2 x = fma2(make_float2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), make_float2(scale, scale),
                                    make_float2(shift, shift));
                    x.x = pow2(x.x);
                    x.y = pow2(x.y);
                    sum[c / 2 % 2] = add2(sum[c / 2 % 2], x);
                    s[c / 2] = pair_of(x.x, x.y, T());
                };
                auto hand_half = [&] {
                    tmem_put(s_at, s);
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) arrive(&b->p_half[w]);
                };
#pragma unroll
                for (int c0 = 0; c0 < kKeys; c0 += 32) {
                    if (!kHides || used & (1u << (c0 / 32))) {
#pragma unroll
                        for (int c = c0; c < c0 + 32; c += 2) weigh(c);
                    } else {
#pragma unroll
                        for (int c = c0; c < c0 + 32; c += 2) s[c / 2] = 0;
                    }
                    if (c0 + 32 == kKeys / 2) hand_half();
                    if (c0 + 32 == kKeys * 3 / 4) {
                        __syncwarp();
                        if (lane == 0) arrive(&b->turn[w ^ 1]);
                    }
                }
                sum[0] = add2(sum[0], sum[1]);
                l += sum[0].x + sum[0].y;
                tmem_put(s_at + kKeys / 4, s + kKeys / 4);
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) arrive(&b->p_full[w]);
                return true;
            };
            for (int j = 0; j < n && ok; ++j, ++done) {
                const int kb = it.key(j);
                ok = kb + kKeys - 1 > min(p_low, it.past(j) - 1) || (a.window && kb <= p_high - a.window && kb + kKeys > a.sinks)
                         ? step(j, std::true_type())
                         : step(j, std::false_type());
            }
            if (n > 0 && ok) ok = warp_wait_for(&b->o_done[w], (done - 1) & 1, b, a.gave_up, limit);
            if (ok) {
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const int h = it.kh * a.group + g;
                char *out = a.out + (it.x.q0 + i) * a.o_row + h * a.o_head;
                const float f = m == kNone ? 0.f : 1.f / l;
                // (The maximum's own weight is 2^kLift, but for how far m * scale was rounded: by powers of two where scores
                // pass 2^25.  Float16 loses its bits where that made it small; such rows are worked out again too.)
                bool finite = !std::is_same<T, __half>::value || m == kNone || l >= 0x1p10f;
                static_assert(!std::is_same<T, __half>::value || Headroom<T>::kLift > 10.f, "a usual sum is above that");
#pragma unroll
                for (int d = 0; d < DP; d += 32) {
                    uint32_t o[32] = {};
                    if (n > 0) {
                        tmem_get(o_at + d, o);
                        settle(o);
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        uint4 x;
                        uint32_t *y = &x.x;
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const float u = __uint_as_float(o[e + 2 * c]) * f, v = __uint_as_float(o[e + 2 * c + 1]) * f;
                            finite &= fabsf(u) < INFINITY && fabsf(v) < INFINITY;
                            y[c] = pair_of(u, v, T());
                        }
                        if (live && d + e < a.dim) *reinterpret_cast<uint4 *>(out + (d + e) * 2) = x;
                    }
                }
                __syncwarp();  // the rows' first stores come before their second ones, which other lanes make
                for (uint32_t again = __ballot_sync(0xffffffffu, live && !finite); again; again &= again - 1) {
                    const int from = __ffs(again) - 1;
                    row_alone<T>(a, it.x, __shfl_sync(0xffffffffu, i, from), __shfl_sync(0xffffffffu, h, from));
                }
            }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    }
    __syncthreads();
    if (warp == kMathWarp) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

PFN_cuTensorMapEncodeTiled_v12000 map_encoder() {
    static const auto fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }();
    return fn;
}

// Rows [rows][heads][dim] as boxes of 64 dims x `heads_box` heads x `rows_box` rows; dims past the end read as zeros.
int encode(CUtensorMap *map, const void *data, bool bf16, int64_t dim, int64_t heads, int64_t rows, int64_t head_stride,
           int64_t row_stride, int heads_box, int rows_box) {
    auto fn = map_encoder();
    if (!fn) return set_error(MR_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
    const cuuint64_t size[3] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows)};
    // a dimension of one element may come with any stride, also none
    const cuuint64_t stride[2] = {static_cast<cuuint64_t>(heads == 1 ? 16 : head_stride),
                                  static_cast<cuuint64_t>(rows == 1 ? 16 : row_stride)};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(heads_box), static_cast<cuuint32_t>(rows_box)}, one[3] = {1, 1, 1};
    const CUresult r = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                          const_cast<void *>(data), size, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(MR_ERR_ARGUMENT, "the rows' layout cannot be loaded by tiles (%d)", static_cast<int>(r));
    return MR_OK;
}

template <typename T, int DP>
int launch(mr_context *ctx, WindowArgs &a) {
    using S = Shape<DP>;
    constexpr bool kBf16 = !__is_same(T, __half);
    const int per = kTile / a.group;
    Maps maps;
    MR_CHECK(encode(&maps.q, a.q, kBf16, a.dim, a.heads, a.tokens, a.q_head, a.q_row, a.group, per));
    MR_CHECK(encode(&maps.k, a.k, kBf16, a.dim, a.kv_heads, a.rows, a.k_head, a.k_row, 1, kKeys));
    MR_CHECK(encode(&maps.v, a.v, kBf16, a.dim, a.kv_heads, a.rows, a.v_head, a.v_row, 1, kKeys));
    const int64_t pairs = a.tokens / (2 * per) + static_cast<int64_t>(a.batch);  // no sequence has more than one that is not full
    const int64_t items = pairs * a.kv_heads;
    MR_REQUIRE(items <= INT32_MAX, "too many rows and heads for one call");
    // Short items: a CTA an SM that loads the next while it finishes one (40 prompts of 100 tokens:
    // 23.0 us, 28.5 with a CTA each).  Long ones: a CTA each, whose order the GPU balances as they end
    // (one flashlite context: 229 us, 239 in fixed rounds).
    const int64_t keys = std::min<int64_t>(a.rows / a.batch, a.window ? static_cast<int64_t>(a.window) + a.sinks : a.rows);
    const bool rounds = keys <= 1024;
    const auto kernel = rounds ? k_window<T, DP, true> : k_window<T, DP, false>;
    static std::atomic<uint64_t> allowed[2] = {};
    MR_CHECK(allow_shared(ctx->device, reinterpret_cast<const void *>(kernel), S::kSmem, allowed[rounds]));
    const int64_t grid = rounds ? std::min<int64_t>(items, ctx->sm_count) : items;
    kernel<<<static_cast<unsigned>(grid), kTcThreads, S::kSmem, ctx->stream>>>(a, maps);
    MR_CUDA_TRY(cudaGetLastError());
    return MR_OK;
}

template <typename T>
int launch_rows(mr_context *ctx, const WindowArgs &a) {
    const int64_t warps = static_cast<int64_t>(a.tokens) * a.heads;
    MR_REQUIRE((warps + 3) / 4 <= INT32_MAX, "too many rows and heads for one call");
    k_rows<T><<<static_cast<unsigned>((warps + 3) / 4), 128, 0, ctx->stream>>>(a);
    MR_CUDA_TRY(cudaGetLastError());
    return MR_OK;
}

template <int DP, int ROWS>
int launch32(mr_context *ctx, const WindowArgs &a) {
    using Shared = Shared32<DP, ROWS>;
    const int per = ROWS / a.group;
    const int64_t items = (a.tokens / per + static_cast<int64_t>(a.batch)) * a.kv_heads;
    MR_REQUIRE(items <= INT32_MAX, "too many rows and heads for one call");
    static std::atomic<uint64_t> allowed{0};
    MR_CHECK(allow_shared(ctx->device, reinterpret_cast<const void *>(k_window32<DP, ROWS>), sizeof(Shared), allowed));
    k_window32<DP, ROWS><<<static_cast<unsigned>(items), kThreads32, sizeof(Shared), ctx->stream>>>(a);
    MR_CUDA_TRY(cudaGetLastError());
    return MR_OK;
}
template <int DP>
int launch32(mr_context *ctx, const WindowArgs &a) {
    // fewer than two CTAs of 64 rows an SM: the smaller ones (short flashnano-1.5 prompts, 745
    // tokens in 53 or 106 CTAs: 12.1 us against 17.3)
    const bool few = static_cast<int64_t>(a.tokens) * a.heads < int64_t(2) * 64 * ctx->sm_count;
    return a.group <= 32 && few ? launch32<DP, 32>(ctx, a) : launch32<DP, 64>(ctx, a);
}
int launch32(mr_context *ctx, WindowArgs &a) {
    if (a.group > 64) return launch_rows<float>(ctx, a);
    return a.dim <= 32 ? launch32<32>(ctx, a) : a.dim <= 64 ? launch32<64>(ctx, a) : launch32<128>(ctx, a);
}

template <typename T>
int launch16(mr_context *ctx, WindowArgs &a) {
    // Under the smallest scales a tile's maximum would not leave `none seen`, and 0 would not leave the hidden
    // keys' -inf alone.  Float16 scores are below 2^40, and a scale of 2^-100 weighs them all alike as 0 does.
    constexpr float kLeast = 1e-36f;
    if (a.scale == 0.f && std::is_same<T, __half>::value) a.scale = 0x1p-100f;
    // A tile holds whole groups; a group of more heads than it has rows goes by rows, as no rows of keys do,
    // and those scales.
    if (a.group > kTile || a.rows == 0 || fabsf(a.scale) < kLeast) return launch_rows<T>(ctx, a);
    return a.dim <= 64 ? launch<T, 64>(ctx, a) : launch<T, 128>(ctx, a);
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
    MR_REQUIRE(is_float(query->dtype) && keys->dtype == query->dtype && values->dtype == query->dtype &&
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
    MR_CHECK(mr::check_waits(ctx));
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
    // A window of all rows hides nothing; a shorter one is below 2^30, as positions are in size, so that
    // their differences stay within 32 bits.
    a.window = window < keys->shape[0] ? window : 0;
    a.sinks = sinks;
    a.scale = scale;
    a.gave_up = ctx->wait_error;
    a.limit = ctx->wait_limit + std::min<uint64_t>(uint64_t(4000) * a.rows, 8 * mr::tc::kWaitNs);
    a.withhold = ctx->withhold;
    return query->dtype == MR_DTYPE_F32   ? launch32(ctx, a)
           : query->dtype == MR_DTYPE_F16 ? launch16<__half>(ctx, a)
                                          : launch16<__nv_bfloat16>(ctx, a);
}
