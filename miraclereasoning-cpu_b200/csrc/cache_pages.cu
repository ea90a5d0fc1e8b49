// Rows of a paged key / value cache: appending new ones, and eviction (the rows
// of largest accumulated weight kept and copied to other pages).
//
// Both move whole rows and are bound by memory: an append reads and writes every
// new row once; an eviction reads every weight once to choose, then reads and
// writes the kept rows.  Rows move as 16-byte pieces, consecutive threads taking
// consecutive pieces of a row and then the next key / value head, so that both
// sides touch whole 32-byte sectors whatever the head dim.
#include "packed.cuh"

namespace mr {
namespace cache {
namespace {

// A pool's base and strides in bytes.
struct Pool {
    char *base;
    int64_t page, row, head;
};
Pool make_pool(const mr_array *a) {
    const int64_t size = dtype_bytes(a->dtype);
    return Pool{static_cast<char *>(a->data), a->stride[0] * size, a->stride[1] * size, a->stride[2] * size};
}

// ---- append -----------------------------------------------------------------------
struct AppendArgs {
    const char *keys, *values;  // new rows; strides in bytes
    int64_t key_token, key_head, value_token, value_head;
    Pool k, v;
    Pages pages;
    const int *lengths, *offsets;
    int64_t length_stride, offset_stride;
    int tokens, batch, heads, pieces;  // pieces: 16-byte pieces of a row
    int team, share;  // warps that work together, and their tokens
};

// The sequence that owns packed row i: the last s with offsets[s] <= i; -1 if its
// end is not behind i (offsets that do not rise own nothing twice: one s a row).
__device__ int sequence_of(const int *offsets, int64_t stride, int batch, int i) {
    int lo = -1, hi = batch;  // offsets[lo] <= i < offsets[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(offsets + mid * stride) <= i) lo = mid;
        else hi = mid;
    }
    return lo >= 0 && __ldg(offsets + (lo + 1) * stride) > i ? lo : -1;
}

// `team` warps take `share` tokens (kOne: one), few where rows are long: a lane finds one token's
// place, then all copy the rows' pieces, four of the keys and four of the values in flight a lane.
template <bool kOne>
__global__ void __launch_bounds__(256, 4) k_append(const __grid_constant__ AppendArgs a) {
    const int lane = threadIdx.x % 32, warp = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    const int first = warp / a.team * a.share;
    const int mine = first + lane, n = a.heads * a.pieces;
    if (first >= a.tokens) return;
    int64_t kr = -1, vr = -1;
    if (lane < a.share && mine < a.tokens) {
        int s = mine, behind = 1;  // rows from this one to the sequence's end
        if (a.offsets) {
            s = sequence_of(a.offsets, a.offset_stride, a.batch, mine);
            if (s >= 0) behind = __ldg(a.offsets + (s + 1) * a.offset_stride) - mine;
        }
        const int t = s >= 0 ? max(0, __ldg(a.lengths + s * a.length_stride)) - behind : -1;
        if (t >= 0) {
            kr = a.pages.row(s, t, a.k.page, a.k.row);
            vr = a.pages.row(s, t, a.v.page, a.v.row);
        }
    }
    constexpr int kFlight = 4;
    const int all = min(a.share, a.tokens - first) * n;
    if (kOne) {
        kr = __shfl_sync(0xffffffffu, kr, 0);
        vr = __shfl_sync(0xffffffffu, vr, 0);
        if (kr < 0) return;
    }
    for (int e0 = lane + warp % a.team * 32 * kFlight; e0 - lane < all; e0 += 32 * kFlight * a.team) {
        uint4 x[kFlight], y[kFlight];
        char *to_k[kFlight], *to_v[kFlight];
#pragma unroll
        for (int f = 0; f < kFlight; ++f) {
            const int e = min(e0 + 32 * f, all - 1), token = kOne ? 0 : e / n, i = e - token * n;
            const int h = i / a.pieces, c = (i - h * a.pieces) * 16;
            const int64_t k = kOne ? kr : __shfl_sync(0xffffffffu, kr, token);
            const int64_t v = kOne ? vr : __shfl_sync(0xffffffffu, vr, token);
            const bool there = k >= 0 && e0 + 32 * f < all;
            to_k[f] = there ? a.k.base + k + h * a.k.head + c : nullptr;
            to_v[f] = a.v.base + v + h * a.v.head + c;
            x[f] = y[f] = make_uint4(0, 0, 0, 0);
            if (there) {
                x[f] = *reinterpret_cast<const uint4 *>(a.keys + (first + token) * a.key_token + h * a.key_head + c);
                y[f] = *reinterpret_cast<const uint4 *>(a.values + (first + token) * a.value_token + h * a.value_head + c);
            }
        }
#pragma unroll
        for (int f = 0; f < kFlight; ++f)
            if (to_k[f]) {
                *reinterpret_cast<uint4 *>(to_k[f]) = x[f];
                *reinterpret_cast<uint4 *>(to_v[f]) = y[f];
            }
    }
}

// ---- eviction -----------------------------------------------------------------------
struct EvictArgs {
    Pool k, v, tk, tv;
    Pages from, to;
    const int *lengths;
    int64_t length_stride;
    const float *weights;
    int64_t w_batch, w_head;
    int *kept, *new_lengths;
    int64_t kept_batch, kept_head, new_length_stride;
    float *new_weights;
    int64_t nw_batch, nw_head;
    int batch, heads, capacity, target_rows, budget, sinks, recent, pieces;
};

// Weights in rising order as unsigned numbers; both zeros equal, NaN the lowest.
__device__ __forceinline__ uint32_t rank_key(float w) {
    if (w != w) return 0;
    const uint32_t bits = __float_as_uint(w + 0.f);  // -0 becomes 0
    return bits ^ (static_cast<uint32_t>(static_cast<int32_t>(bits) >> 31) | 0x80000000u);
}

template <int BYTES>
__device__ __forceinline__ void cp_async(void *to, const void *from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))),
                 "l"(from), "n"(BYTES)
                 : "memory");
}

constexpr int kSelectThreads = 1024, kSelectWarps = kSelectThreads / 32, kBins = 2048, kCached = 48 << 10;
constexpr int kMarked = 28;  // rows that a thread marks at once

// CTA = (sequence, head).  The sinks and the recent rows take part as the largest of all, so
// the `budget` largest stay: the value of the last of them is found digit by digit, 11, 11
// and 10 bits of the weights' order: counts of a digit among the rows that match the digits
// found so far, and the highest digit that has the wanted row.  (The first 11 bits are sign,
// exponent and two bits of the fraction, so that weights of all sizes fall on many counters; a
// warp's rows that all fall on one, as after a reset, are counted at once.)  Rows above that
// value stay, and the first few equal to it.  Then each thread marks a few rows of its own, and
// the kept ones go in order behind those of the threads before it.
//
// The weights come to shared memory where they fit, by asynchronous copies, and are their order
// from the first count on.  20000 weights are 625 issues of the SM for each instruction that is
// written once a weight: 3.1 us until they are there, 7.5 for the digits, 3.2 for the rows that
// stay and 1.5 for their weights.  (Votes and counts of bits for every 32 rows in turn took 5.4 us
// instead of the 3.2, whether the rows were stored one by one or in lines.)  What runs only a few
// times costs the fetch of its code, hundreds of cycles a line: the loops stay rolled (loads
// unrolled by eight took 6.0 us instead of 3.1, and by eight everywhere 12000 weights took 40).
__global__ void __launch_bounds__(kSelectThreads) k_select(const __grid_constant__ EvictArgs a) {
    __shared__ int counts[kBins];
    __shared__ int above[kSelectWarps];
    __shared__ uint32_t s_digit;
    __shared__ int s_need;
    extern __shared__ __align__(16) uint32_t cached[];
    const int s = blockIdx.x / a.heads, h = blockIdx.x % a.heads;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int n = sequence_rows(a.lengths, a.length_stride, s, a.capacity);
    for (int i = tid; i < kBins; i += kSelectThreads) counts[i] = 0;
    const float *w = a.weights + s * a.w_batch + h * a.w_head;
    int *kept = a.kept + s * a.kept_batch + h * a.kept_head;
    float *nw = a.new_weights + s * a.nw_batch + h * a.nw_head;
    const int total = min(n, a.budget);
    if (tid == 0 && h == 0) a.new_lengths[s * a.new_length_stride] = total;
    const bool in_shared = a.capacity <= kCached;
    const uint32_t ranked = max(n - a.recent, a.sinks) - a.sinks;  // rows behind the sinks, before the recent ones
    auto order = [&](int t, float x) { return static_cast<uint32_t>(t - a.sinks) < ranked ? rank_key(x) : 0xffffffffu; };
    // rows past the end: 0, and told apart by their number
    auto read = [&](int t) { return t < n ? order(t, __ldg(w + t)) : 0u; };
    auto four = [&](int t) {
        return in_shared ? *reinterpret_cast<const uint4 *>(cached + t)
                         : make_uint4(read(t), read(t + 1), read(t + 2), read(t + 3));
    };
    if (in_shared && n > a.budget) {
        const int fours = reinterpret_cast<uintptr_t>(w) % 16 ? 0 : n & ~3;
#pragma unroll 1
        for (int t = 4 * tid; t < fours; t += 4 * kSelectThreads) cp_async<16>(cached + t, w + t);
#pragma unroll 1
        for (int t = fours + tid; t < n; t += kSelectThreads) cp_async<4>(cached + t, w + t);
        asm volatile("cp.async.wait_all;" ::: "memory");
    }
    __syncthreads();
    if (n > a.budget) {
        uint32_t cut = 0;  // rows of a larger key stay, and `need` of those equal to it
        int need = a.budget;
#pragma unroll 1
        for (int shift = 21; shift >= 0; shift = shift == 21 ? 10 : shift == 10 ? 0 : -1) {
            const int bits = shift ? 11 : 10, bins = 1 << bits;
            if (shift != 21) {
                for (int i = tid; i < bins; i += kSelectThreads) counts[i] = 0;
                __syncthreads();
            }
#pragma unroll 1
            for (int t = 4 * tid; t - 4 * lane < n; t += 4 * kSelectThreads) {
                uint4 x = make_uint4(0, 0, 0, 0);
                if (t < n) x = four(t);
                if (shift == 21 && in_shared && t < n) {  // weights as they came: their order from here on
                    auto key_of = [&](int i, uint32_t raw) { return t + i < n ? order(t + i, __uint_as_float(raw)) : 0u; };
                    x = make_uint4(key_of(0, x.x), key_of(1, x.y), key_of(2, x.z), key_of(3, x.w));
                    *reinterpret_cast<uint4 *>(cached + t) = x;
                }
                const uint32_t key[4] = {x.x, x.y, x.z, x.w};
                const uint32_t one = __shfl_sync(0xffffffffu, x.x >> shift, 0);
                if (__all_sync(0xffffffffu, t + 3 < n && x.x >> shift == one && x.y >> shift == one &&
                                                x.z >> shift == one && x.w >> shift == one)) {
                    if (lane == 0 && (shift == 21 || one >> bits == cut)) atomicAdd(&counts[one & (bins - 1)], 128);
                    continue;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (t + i < n && (shift == 21 || key[i] >> (shift + bits) == cut))
                        atomicAdd(&counts[key[i] >> shift & (bins - 1)], 1);
            }
            __syncthreads();
            // each warp's bins summed, then the warp that has the row looks into its own
            const int mine = bins / kSelectWarps, base = warp * mine;  // 64 or 32 bins
            const int low = counts[base + lane], high = mine == 64 ? counts[base + 32 + lane] : 0;
            const int sum = __reduce_add_sync(0xffffffffu, low + high);
            if (lane == 0) above[warp] = sum;
            __syncthreads();
            const int over = __reduce_add_sync(0xffffffffu, lane > warp ? above[lane] : 0);  // rows of higher warps' bins
            if (over < need && over + sum >= need) {
                int left = need - over;
                auto find = [&](int count, int at) {  // in 32 bins from the highest: the one that has the row
                    int from = count;  // rows in this bin and the higher ones
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const int up = __shfl_down_sync(0xffffffffu, from, o);
                        if (lane + o < 32) from += up;
                    }
                    const uint32_t reach = __ballot_sync(0xffffffffu, from >= left);
                    if (!reach) {
                        left -= __shfl_sync(0xffffffffu, from, 0);
                        return false;
                    }
                    const int bin = 31 - __clz(reach);
                    if (lane == bin) {
                        s_digit = at + bin;
                        s_need = left - (from - count);
                    }
                    return true;
                };
                if (mine == 32 || !find(high, base + 32)) find(low, base);
            }
            __syncthreads();
            cut = cut << bits | s_digit;
            need = s_need;
        }
        // Rows that stay, in order: a thread's own few rows become two masks, larger than the cut and
        // equal to it, whose counts (below 2^15 in a part of the rows) are added up over the CTA in
        // the halves of one number.  From shared memory, a warp's kept rows are gathered where its
        // keys were, and stored in whole lines.
        int kept_before = 0, equal_before = 0;
#pragma unroll 1
        for (int part = 0; part < n; part += kSelectThreads * kMarked) {
            // vectors of four a thread: an odd number, so that eight threads' meet all banks
            const int mine = min(((n - part + kSelectThreads - 1) / kSelectThreads + 3) / 4 | 1, kMarked / 4) * 4;
            const int lo = part + warp * 32 * mine, from = lo + lane * mine;
            uint32_t stay = 0, same = 0;
#pragma unroll 1
            for (int i = 0; i < mine && from + i < n; i += 4) {
                const uint4 x = four(from + i);
                const uint32_t key[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    stay |= (key[e] > cut ? 1u << e : 0u) << i;
                    same |= (key[e] == cut && from + i + e < n ? 1u << e : 0u) << i;
                }
            }
            const int count = __popc(stay) + (__popc(same) << 16);
            int sum = count;  // of the lanes up to this one
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int under = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += under;
            }
            __syncthreads();  // above[] of the part before, or of the last digit, has been read
            if (lane == 31) above[warp] = sum;
            __syncthreads();
            const int warps = above[lane], under = __reduce_add_sync(0xffffffffu, lane < warp ? warps : 0);
            const int all = __reduce_add_sync(0xffffffffu, warps);
            const int first = kept_before + (under & 0xffff) + min(equal_before + (under >> 16), need);
            sum += under - count;
            const int equals = equal_before + (sum >> 16);  // rows equal to the cut before this thread's
            int at = kept_before + (sum & 0xffff) + min(equals, need);
            for (int room = need - equals; same && room > 0; same &= same - 1, --room) stay |= same & -same;
            kept_before += all & 0xffff;
            equal_before += all >> 16;
#pragma unroll 1
            for (; stay; stay &= stay - 1, ++at) {
                const int row = from + __ffs(stay) - 1;
                if (in_shared) cached[lo + at - first] = row;
                else if (at < a.budget) kept[at] = row;
            }
            if (in_shared) {
                at = __shfl_sync(0xffffffffu, at, 31);
                __syncwarp();
#pragma unroll 1
                for (int i = first + lane; i < min(at, a.budget); i += 32) kept[i] = static_cast<int>(cached[lo + i - first]);
            }
        }
    } else {
        for (int i = tid; i < n; i += kSelectThreads) kept[i] = i;
    }
#pragma unroll 1
    for (uint32_t i = total + tid; i < static_cast<uint32_t>(a.budget); i += kSelectThreads) kept[i] = -1;  // to 2^31 - 1
    __syncthreads();
    constexpr int kFlight = 4;
#pragma unroll 1
    for (int i = tid; i < a.target_rows; i += kSelectThreads * kFlight) {
        int t[kFlight];
        float x[kFlight];
#pragma unroll
        for (int e = 0; e < kFlight; ++e) t[e] = i + e * kSelectThreads < total ? __ldcg(kept + i + e * kSelectThreads) : -1;
#pragma unroll
        for (int e = 0; e < kFlight; ++e) x[e] = t[e] >= 0 ? __ldg(w + t[e]) : 0.f;
#pragma unroll
        for (int e = 0; e < kFlight; ++e)
            if (i + e * kSelectThreads < a.target_rows) nw[i + e * kSelectThreads] = x[e];
    }
}

// Kept rows to their target pages: a warp takes 32 rows of a head, a lane looks up one row's two
// places, and all copy the rows piece by piece (16 bytes, or what rows of 4-bit values are whole
// multiples of), four loads of each pool in flight a lane.  16 sequences of 8192 rows of 4 bits to 2048 with
// their selection: 8 heads of 128 35 us, 10 of 96 45, 16 of 64 48, 32 of 32 72 (at the copy rate 13 to 17): pieces of 8 and 4 bytes.
constexpr int kCopyWarps = 4;
template <typename Bytes>
__global__ void __launch_bounds__(kCopyWarps * 32) k_copy_kept(const __grid_constant__ EvictArgs a) {
    const int s = blockIdx.z, h = blockIdx.y, lane = threadIdx.x % 32;
    const int at = (blockIdx.x * kCopyWarps + threadIdx.x / 32) * 32 + lane;
    const int total = min(sequence_rows(a.lengths, a.length_stride, s, a.capacity), min(a.budget, a.target_rows));
    if (at - lane >= total) {
        // waits too: with no rows anywhere, this grid would end, and what is queued behind it start,
        // while the selection still writes
        asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    // the target's page is found before the selection is waited for
    int64_t to_k = -1, to_v = -1, k = -1, v = -1;
    if (at < total) {
        to_k = a.to.row(s, at, a.tk.page, a.tk.row);
        to_v = a.to.row(s, at, a.tv.page, a.tv.row);
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (at < total) {
        const int t = __ldcg(a.kept + s * a.kept_batch + h * a.kept_head + at);
        k = a.from.row(s, t, a.k.page, a.k.row);
        v = a.from.row(s, t, a.v.page, a.v.row);
    }
    const char *kb = a.k.base + h * a.k.head, *vb = a.v.base + h * a.v.head;
    char *tk = a.tk.base + h * a.tk.head, *tv = a.tv.base + h * a.tv.head;
    const int n = 32 * a.pieces;
    constexpr int kFlight = 4;
    for (int e0 = lane; e0 < n; e0 += 32 * kFlight) {
        Bytes x[kFlight], y[kFlight];
        int64_t tks[kFlight], tvs[kFlight];
#pragma unroll
        for (int i = 0; i < kFlight; ++i) {
            const int e = min(e0 + 32 * i, n - 1), r = e / a.pieces, c = (e - r * a.pieces) * static_cast<int>(sizeof(Bytes));
            const int64_t from_k = __shfl_sync(0xffffffffu, k, r), from_v = __shfl_sync(0xffffffffu, v, r);
            tks[i] = __shfl_sync(0xffffffffu, to_k, r);
            tvs[i] = __shfl_sync(0xffffffffu, to_v, r);
            if (e0 + 32 * i >= n) tks[i] = -1;
            x[i] = y[i] = Bytes{};
            if (from_k >= 0 && tks[i] >= 0) {
                x[i] = __ldcs(reinterpret_cast<const Bytes *>(kb + from_k + c));
                y[i] = __ldcs(reinterpret_cast<const Bytes *>(vb + from_v + c));
            }
            tks[i] += c;
            tvs[i] += c;
            if (tks[i] < c) tks[i] = -1;
        }
#pragma unroll
        for (int i = 0; i < kFlight; ++i)
            if (tks[i] >= 0) {
                *reinterpret_cast<Bytes *>(tk + tks[i]) = x[i];
                *reinterpret_cast<Bytes *>(tv + tvs[i]) = y[i];
            }
    }
}

}  // namespace
}  // namespace cache
}  // namespace mr

using namespace mr::cache;

extern "C" int mr_append_pages(mr_context *ctx, const mr_array *keys, const mr_array *values, const mr_array *key_pages,
                               const mr_array *value_pages, const mr_array *page_table, const mr_array *lengths,
                               const mr_array *offsets) {
    if (key_pages && key_pages->dtype == MR_DTYPE_U8)
        return mr_append_rotated(ctx, nullptr, keys, values, key_pages, value_pages, page_table, lengths, offsets, nullptr,
                                 nullptr, nullptr, 0);
    MR_CHECK(check_array(keys, "keys", 3, true, false));
    MR_CHECK(check_array(values, "values", 3, true, false));
    MR_CHECK(check_pools(key_pages, value_pages, "key_pages", "value_pages", true));
    MR_REQUIRE(keys->dtype == key_pages->dtype && values->dtype == key_pages->dtype,
               "keys, values and the pages must be of one type");
    for (int i = 0; i < 3; ++i) MR_REQUIRE(keys->shape[i] == values->shape[i], "keys and values differ in shape");
    MR_REQUIRE(keys->shape[1] == key_pages->shape[2] && keys->shape[2] == key_pages->shape[3],
               "keys must be [tokens, %lld, %lld], as the pages' heads and dim",
               static_cast<long long>(key_pages->shape[2]), static_cast<long long>(key_pages->shape[3]));
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
    MR_REQUIRE(ctx, "ctx is NULL");
    MR_CHECK(mr::check_waits(ctx));
    if (!keys->shape[0] || !batch || !key_pages->shape[0] || !page_table->shape[1]) return MR_OK;
    DeviceGuard guard(ctx->device);
    const int64_t size = dtype_bytes(keys->dtype);
    AppendArgs a;
    a.keys = static_cast<const char *>(keys->data);
    a.values = static_cast<const char *>(values->data);
    a.key_token = keys->stride[0] * size;
    a.key_head = keys->stride[1] * size;
    a.value_token = values->stride[0] * size;
    a.value_head = values->stride[1] * size;
    a.k = make_pool(key_pages);
    a.v = make_pool(value_pages);
    a.pages = make_pages(key_pages, page_table);
    a.lengths = static_cast<const int *>(lengths->data);
    a.length_stride = lengths->stride[0];
    a.offsets = offsets ? static_cast<const int *>(offsets->data) : nullptr;
    a.offset_stride = offsets ? offsets->stride[0] : 0;
    a.tokens = static_cast<int>(keys->shape[0]);
    a.batch = static_cast<int>(batch);
    a.heads = static_cast<int>(keys->shape[1]);
    a.pieces = static_cast<int>(keys->shape[2] * size / 16);
    // Few tokens: a CTA each, its warps sharing the row.  Else as many to a warp as make about 128
    // pieces of each pool (79000 tokens of 18 pieces: 19 us, 62 with one each).
    const int pieces = a.heads * a.pieces;
    const bool few = a.tokens < 4 * ctx->sm_count;
    a.share = few ? 1 : std::max(1, std::min(32, 128 / pieces));
    a.team = few ? std::max(1, std::min(8, pieces / 128)) : 1;
    const int warps = few ? a.team : 8, each = warps / a.team * a.share;
    (a.share == 1 ? k_append<true> : k_append<false>)<<<(a.tokens - 1) / each + 1, warps * 32, 0, ctx->stream>>>(a);
    MR_CUDA_TRY(cudaGetLastError());
    return MR_OK;
}

extern "C" int mr_evict_pages(mr_context *ctx, const mr_array *key_pages, const mr_array *value_pages,
                              const mr_array *page_table, const mr_array *lengths, const mr_array *weights,
                              const mr_array *target_keys, const mr_array *target_values, const mr_array *target_table,
                              const mr_array *kept, const mr_array *new_lengths, const mr_array *new_weights,
                              int budget, int sinks, int recent) {
    const bool packed = key_pages && key_pages->dtype == MR_DTYPE_U8;
    if (packed) {
        MR_CHECK(check_packed(key_pages, value_pages, "key_pages", "value_pages", false));
        MR_CHECK(check_packed(target_keys, target_values, "target_keys", "target_values", true));
    } else {
        MR_CHECK(check_pools(key_pages, value_pages, "key_pages", "value_pages", false));
        MR_CHECK(check_pools(target_keys, target_values, "target_keys", "target_values", true));
    }
    MR_REQUIRE(target_keys->dtype == key_pages->dtype, "the target pages must be of the pages' type");
    for (int i = 1; i < 4; ++i)
        MR_REQUIRE(target_keys->shape[i] == key_pages->shape[i],
                   "the target pages must have the pages' rows, heads and dim");
    MR_CHECK(check_ints(lengths, "lengths", 1));
    const int64_t batch = lengths->shape[0], page = key_pages->shape[1], heads = key_pages->shape[2];
    MR_CHECK(check_table(page_table, "page_table", batch, page));
    MR_CHECK(check_table(target_table, "target_table", batch, page));
    MR_REQUIRE(sinks >= 0 && recent >= 0 && budget > 0, "budget must be positive, sinks and recent not negative");
    MR_REQUIRE(static_cast<int64_t>(sinks) + recent <= budget, "budget %d is less than sinks %d and recent %d", budget,
               sinks, recent);
    const int64_t capacity = page_table->shape[1] * page, room = target_table->shape[1] * page;
    MR_REQUIRE(room >= std::min<int64_t>(budget, capacity),
               "target_table has room for %lld rows of the %lld that may be kept", static_cast<long long>(room),
               static_cast<long long>(std::min<int64_t>(budget, capacity)));
    MR_CHECK(check_weights(weights, "weights", batch, heads, capacity, false));
    MR_CHECK(check_weights(new_weights, "new_weights", batch, heads, room, true));
    MR_CHECK(check_ints(kept, "kept", 3, true));
    MR_REQUIRE(kept->shape[0] == batch && kept->shape[1] == heads && kept->shape[2] == budget,
               "kept must be [%lld, %lld, %d] (batch, kv heads, budget)", static_cast<long long>(batch),
               static_cast<long long>(heads), budget);
    MR_CHECK(check_ints(new_lengths, "new_lengths", 1, true));
    MR_REQUIRE(new_lengths->shape[0] == batch, "new_lengths must have %lld values", static_cast<long long>(batch));
    MR_CHECK(check_apart(weights, "weights", new_weights, "new_weights"));
    MR_CHECK(check_apart(lengths, "lengths", new_lengths, "new_lengths"));
    MR_REQUIRE(batch <= 65535, "more than 65535 sequences");
    MR_REQUIRE(heads <= 65535 && batch * heads <= INT32_MAX, "too many heads");
    MR_REQUIRE(ctx, "ctx is NULL");
    MR_CHECK(mr::check_waits(ctx));
    if (!batch) return MR_OK;
    DeviceGuard guard(ctx->device);
    EvictArgs a;
    a.k = make_pool(key_pages);
    a.v = make_pool(value_pages);
    a.tk = make_pool(target_keys);
    a.tv = make_pool(target_values);
    a.from = make_pages(key_pages, page_table);
    a.to = make_pages(target_keys, target_table);
    a.lengths = static_cast<const int *>(lengths->data);
    a.length_stride = lengths->stride[0];
    a.weights = static_cast<const float *>(weights->data);
    a.w_batch = weights->stride[0];
    a.w_head = weights->stride[1];
    a.kept = static_cast<int *>(kept->data);
    a.kept_batch = kept->stride[0];
    a.kept_head = kept->stride[1];
    a.new_lengths = static_cast<int *>(new_lengths->data);
    a.new_length_stride = new_lengths->stride[0];
    a.new_weights = static_cast<float *>(new_weights->data);
    a.nw_batch = new_weights->stride[0];
    a.nw_head = new_weights->stride[1];
    a.batch = static_cast<int>(batch);
    a.heads = static_cast<int>(heads);
    a.capacity = static_cast<int>(capacity);
    a.target_rows = static_cast<int>(room);
    a.budget = budget;
    a.sinks = sinks;
    a.recent = recent;
    const int unit = packed ? packed_unit(key_pages->shape[3]) : 16;
    a.pieces = static_cast<int>(key_pages->shape[3] * dtype_bytes(key_pages->dtype) / unit);
    static std::atomic<uint64_t> allowed{0};
    MR_CHECK(allow_shared(ctx->device, reinterpret_cast<const void *>(k_select), kCached * 4, allowed));
    const int cached = capacity <= kCached ? (static_cast<int>(capacity) + 3) / 4 * 16 : 0;
    k_select<<<a.batch * a.heads, kSelectThreads, cached, ctx->stream>>>(a);
    MR_CUDA_TRY(cudaGetLastError());
    const int64_t rows = std::min<int64_t>(budget, capacity);
    if (rows) {
        const dim3 grid(static_cast<unsigned>((rows - 1) / (32 * kCopyWarps) + 1), a.heads, a.batch);
        MR_CHECK(launch_early(ctx, grid, dim3(kCopyWarps * 32),
                              unit == 16 ? k_copy_kept<uint4> : unit == 8 ? k_copy_kept<uint2> : k_copy_kept<uint32_t>, a));
    }
    return MR_OK;
}
