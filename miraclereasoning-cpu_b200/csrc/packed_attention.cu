// One-token attention over pages of 4 bits a value (packed.cuh has the format,
// paged_core.cuh the work's division, the copies and the kernels).
//
// Rows of 80 bytes instead of 256 leave a third of the time for the same products, so
// what bounds this is no longer memory alone but the instructions that turn codes
// into operands.  Two codes become two float16 values by one logical operation and
// one fused multiply-add; nothing moves between lanes.  For the keys, a lane's
// share of a row's 16 bytes is a word of eight neighbouring dims, and the
// products' inner dims may come in any order as long as the queries' come in the same.  For the values,
// ldmatrix transposes 16-bit units (four codes) of eight rows, so that each register
// holds the same four dims of two rows, and the four results of a word go to rows of
// different product tiles.
//
// A step of 32 rows of 128 dims is 706 instructions: 210 and 236 for the two products' operands and issue, 120
// for the softmax and the weights' two parts, 120 for the copies of two steps on.  32 sequences ragged to 32768 rows
// at 8 heads of 128 (668 MB): 160 us in bfloat16 and float16, 178 in float32, of which about 20 are the start, the uneven
// end and the join; the copies alone take 113.  (Weights in one float16 part, off by 2^-11, took 142: they were as much as an
// eighth of a bfloat16 result's rounding, which moved several results in a hundred to the next bfloat16 number.)
// Smaller dims have less of a row for what a step costs once, and copies of 4 or 8 bytes: 16 sequences ragged to 16384 rows,
// four query heads each (170 MB): 8 heads of 128 62.5 us, 10 of 96 75.6, 16 of 64 83.6, 32 of 32 125; with rows before
// heads in a page, where every 16 bytes have an address of their own, 70, 92, 95 and 152.
// Logical operations and float16 multiply-adds each issue every other cycle, and 1.5 cycles each when
// mixed, so that moving work between the two gains nothing.  Tried beside one part of each weight, at 145 us:
// 8-bit floating-point products of the codes as they stand (e4m3 0 .. 15 are linear) need fewer masks, but that
// type is widened in software here, 790 instructions a step, 175 us; four CTAs an SM spill (150); of
// all 16 warps' stretches joined in shared memory first, one long sequence gains 1 us and the batch loses 8.
#include "packed.cuh"
#include "paged_core.cuh"

namespace mr {
namespace cache {
namespace {

template <int DP>
struct Ring4 {
    static constexpr int kRow = DP * 5 / 8, kUnit = kRow & -kRow;  // 80: 16, 60: 4, 40: 8, 20: 4
    static constexpr int kPieces = kRow / kUnit;
    static constexpr int kRowBytes = DP <= 64 ? 48 : 80;  // odd multiples of 16: eight rows' pieces lie in different banks
    static __device__ __forceinline__ int pieces(const PagedArgs &) { return kPieces; }
    static __device__ __forceinline__ uint32_t offset(int row, int piece) { return row * kRowBytes + piece * kUnit; }
    // of piece e of a step's rows
    static __device__ __forceinline__ uint32_t place(int e) {
        return kRowBytes == kRow ? e * kUnit : offset(e / kPieces, e % kPieces);
    }
};

__device__ __forceinline__ void ldmatrix2(uint32_t (&r)[4], uint32_t address) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(address));
}
__device__ __forceinline__ void ldmatrix2_t(uint32_t (&r)[4], uint32_t address) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(address));
}
// A row's G pairs of step and base.
template <int G>
__device__ __forceinline__ void load_pairs(uint32_t (&p)[G], uint32_t address) {
    if constexpr (G == 1) {
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(p[0]) : "r"(address));
    } else if constexpr (G == 2) {
        asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(p[0]), "=r"(p[1]) : "r"(address));
    } else {
        uint32_t last;
        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(p[0]), "=r"(p[1]), "=r"(p[2]), "=r"(last) : "r"(address));
        if constexpr (G == 4) p[3] = last;
    }
}
__device__ __forceinline__ __half2 halves(uint32_t x) { return *reinterpret_cast<const __half2 *>(&x); }

template <typename T, int DP_>
struct Math4 : Heads8<__half, DP_ / 16> {
    using Base = Heads8<__half, DP_ / 16>;
    using Base::o;
    using Base::m;
    using Base::l;
    static constexpr bool kRuns = true, kAgain = false;  // what is not finite here is NaN, and stays it
    static constexpr int kCtas = 3, DP = DP_, G = DP / kShared, kHeads = 8, STEP = 32;
    // CTAs of an SM.  Three have more steps under way, two leave room for the joining kernel's CTAs to start beside
    // them and fewer partials to join: from about 9 steps a warp on (by the tables; with weights, which the joining
    // kernel adds up, 48) three are faster (us at 32768 rows of 8 heads of 128, two and three: 1 sequence 21.0 and 22.5,
    // 2 31.9 and 31.4, 4 52.3 and 49.9, 16 171 and 157; with weights 8 sequences 111.3 and 111.4, 16 207 and 199).
    static int ctas(int64_t steps, int sms, bool weights) {
        return steps >= (weights ? 48 : 9) * static_cast<int64_t>(3 * kWarps) * sms ? 3 : 2;
    }
    struct R : Ring4<DP> {
        static constexpr int kBytes = 2 * STEP * Ring4<DP>::kRowBytes;
        static constexpr int kWarpBytes = kBytes * 3;
    };
    static constexpr int STAGES = 3;
    // Queries of 16 bits are one float16 operand, those of 32 two, scaled by a power of 2 for each head so that
    // the largest is in [2^14, 2^15): what is lost is below 2^-39 of it, or 2^-22 of the value itself.
    static constexpr int kParts = sizeof(T) == 4 ? 2 : 1;
    uint32_t qf[kParts][G][2][2];
    float f[2];  // of heads 2 (lane % 4), + 1: products to scores

    __device__ __forceinline__ void begin(const PagedArgs &a, const char *q, int heads) {
        const int lane = threadIdx.x % 32, h = lane / 4, c = lane % 4;
        float x[G][8], most = 0.f;
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[g][i] = h < heads ? widen(reinterpret_cast<const T *>(q + h * a.q_head) + 32 * g + 8 * c + i) : 0.f;
                most = fmaxf(most, fabsf(x[g][i]));
            }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // 2^n: 14 less the exponent of the largest; 1 where that is 0 or not finite
        const int exponent = min(max(static_cast<int>(__float_as_uint(most) >> 23) - 127, -100), 127);
        const int n = most > 0.f && most < INFINITY ? 14 - exponent : 0;
        const float up = __uint_as_float(static_cast<uint32_t>(127 + n) << 23);  // n: -113 .. 114
        const float down = __uint_as_float(static_cast<uint32_t>(127 - n) << 23);
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    // codes 2 j + e of a word's two halves
                    const float u = x[g][2 * j + e] * up, w = x[g][4 + 2 * j + e] * up;
                    qf[0][g][j][e] = pack2(u, w, __half());
                    if constexpr (kParts == 2) {
                        const float2 r = unpack2(qf[0][g][j][e], __half());
                        qf[1][g][j][e] = pack2(u - r.x, w - r.y, __half());
                    }
                }
#pragma unroll
        for (int e = 0; e < 2; ++e) f[e] = __shfl_sync(0xffffffffu, down, (2 * c + e) * 4) * a.scale;
        this->clear();
    }

    // S^T of 16 rows at `tile`.
    __device__ __forceinline__ void products(float (&s)[4], uint32_t tile) const {
        const int lane = threadIdx.x % 32, r = lane / 4;
        const uint32_t part = (lane % 16) * R::kRowBytes + lane / 16 * 16;
        s[0] = s[1] = s[2] = s[3] = 0.f;
        uint32_t p0[G], p1[G];
        load_pairs<G>(p0, tile + r * R::kRowBytes + DP / 2);
        load_pairs<G>(p1, tile + (r + 8) * R::kRowBytes + DP / 2);
#pragma unroll
        for (int g = 0; g < G; g += 2) {
            uint32_t w[4];
            if (g + 1 < G) ldmatrix(w, tile + part + g * 16);
            else ldmatrix2(w, tile + part + g * 16 - lane / 16 * 16);
#pragma unroll
            for (int i = 0; i < (g + 1 < G ? 2 : 1); ++i) {
                const __half2 s0 = __low2half2(halves(p0[g + i])), z0 = __high2half2(halves(p0[g + i]));
                const __half2 s1 = __low2half2(halves(p1[g + i])), z1 = __high2half2(halves(p1[g + i]));
                uint32_t u[4], v[4];
                word_codes(w[2 * i], u);
                word_codes(w[2 * i + 1], v);
                const uint32_t k0[4] = {fma2(u[0], s0, z0), fma2(v[0], s1, z1), fma2(u[1], s0, z0), fma2(v[1], s1, z1)};
                const uint32_t k1[4] = {fma2(u[2], s0, z0), fma2(v[2], s1, z1), fma2(u[3], s0, z0), fma2(v[3], s1, z1)};
#pragma unroll
                for (int part_of = kParts - 1; part_of >= 0; --part_of) {
                    mma16(s, k0, qf[part_of][g + i][0][0], qf[part_of][g + i][0][1], __half());
                    mma16(s, k1, qf[part_of][g + i][1][0], qf[part_of][g + i][1][1], __half());
                }
            }
        }
    }

    __device__ __forceinline__ void step(const PagedArgs &a, uint32_t stage, uint32_t live, int rows, float *scores) {
        const int lane = threadIdx.x % 32, c = lane % 4;
        constexpr int S = STEP / 16;
        // this lane's row and piece for ldmatrix: 16 rows of two groups' codes
        const uint32_t part = (lane % 16) * R::kRowBytes + lane / 16 * 16;
        float s[S][4];
#pragma unroll
        for (int x = 0; x < S; ++x) products(s[x], stage + x * 16 * R::kRowBytes);
        float ref[2];
        this->template settle<true>(a, s, f[0], f[1], live, rows, scores, ref);
#pragma unroll
        for (int x = 0; x < S; ++x) {
            uint32_t b0, b1, c0, c1;
            this->weigh(s[x], ref, b0, b1, c0, c1);
            const uint32_t tile = stage + (STEP + x * 16) * R::kRowBytes;
            uint32_t p[4][G];  // of rows 2 c, 2 c + 1, 2 c + 8, 2 c + 9
#pragma unroll
            for (int i = 0; i < 4; ++i) load_pairs<G>(p[i], tile + (2 * c + (i & 1) + (i >> 1) * 8) * R::kRowBytes + DP / 2);
#pragma unroll
            for (int g = 0; g < G; g += 2) {
                uint32_t w[4];
                if (g + 1 < G) ldmatrix_t(w, tile + part + g * 16);
                else ldmatrix2_t(w, tile + part + g * 16 - lane / 16 * 16);
#pragma unroll
                for (int i = 0; i < (g + 1 < G ? 2 : 1); ++i) {
                    const __half2 s0 = halves(__byte_perm(p[0][g + i], p[1][g + i], 0x5410));
                    const __half2 z0 = halves(__byte_perm(p[0][g + i], p[1][g + i], 0x7632));
                    const __half2 s1 = halves(__byte_perm(p[2][g + i], p[3][g + i], 0x5410));
                    const __half2 z1 = halves(__byte_perm(p[2][g + i], p[3][g + i], 0x7632));
                    const uint32_t u = w[2 * i], v = w[2 * i + 1];
                    uint32_t uc[4], vc[4];
                    word_codes(u, uc);
                    word_codes(v, vc);
                    const uint32_t v0[4] = {fma2(uc[0], s0, z0), fma2(uc[1], s0, z0), fma2(vc[0], s1, z1), fma2(vc[1], s1, z1)};
                    const uint32_t v1[4] = {fma2(uc[2], s0, z0), fma2(uc[3], s0, z0), fma2(vc[2], s1, z1), fma2(vc[3], s1, z1)};
                    mma16(o[2 * (g + i)], v0, b0, b1, __half());
                    mma16(o[2 * (g + i)], v0, c0, c1, __half());
                    mma16(o[2 * (g + i) + 1], v1, b0, b1, __half());
                    mma16(o[2 * (g + i) + 1], v1, c0, c1, __half());
                }
            }
        }
    }

    __device__ __forceinline__ bool finish() {
        Base::finish();
        return true;
    }
    // Four values of consecutive dims of a head, times its head's factor: put(head, dim, values).
    template <typename Put>
    __device__ __forceinline__ void each(float f0, float f1, const Put &put) const {
        const int lane = threadIdx.x % 32, h = 2 * (lane % 4);
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float by = e ? f1 : f0;
                put(h + e, 32 * g + lane / 4 * 4, make_float4(o[2 * g][e] * by, o[2 * g][2 + e] * by, o[2 * g + 1][e] * by,
                                                              o[2 * g + 1][2 + e] * by));
            }
    }
    __device__ __forceinline__ void put_out(const PagedArgs &a, char *out, int heads) const {
        each(l[0] != 0.f ? 1.f / l[0] : 0.f, l[1] != 0.f ? 1.f / l[1] : 0.f, [&](int h, int dim, float4 x) {
            if (h >= heads) return;
            char *to = out + h * a.o_head + dim * sizeof(T);
            if constexpr (sizeof(T) == 4) *reinterpret_cast<float4 *>(to) = x;
            else *reinterpret_cast<uint2 *>(to) = make_uint2(pack2(x.x, x.y, T()), pack2(x.z, x.w, T()));
        });
    }
    __device__ __forceinline__ void put_partial(float *to, float2 *sums, int64_t stride, int heads) const {
        const int lane = threadIdx.x % 32;
        each(1.f, 1.f, [&](int h, int dim, float4 x) {
            if (h < heads) *reinterpret_cast<float4 *>(to + h * DP + dim) = x;
        });
        if (lane < 4)
#pragma unroll
            for (int e = 0; e < 2; ++e) sums[(2 * lane + e) * stride] = make_float2(m[e], l[e]);
    }
};

template <typename T>
int launch_dims(mr_context *ctx, PagedArgs &a) {
    return a.dim == 32   ? launch<T, Math4<T, 32>>(ctx, a)
           : a.dim == 64 ? launch<T, Math4<T, 64>>(ctx, a)
           : a.dim == 96 ? launch<T, Math4<T, 96>>(ctx, a)
                         : launch<T, Math4<T, 128>>(ctx, a);
}

}  // namespace

int launch_packed(mr_context *ctx, PagedArgs &a, int dtype) {
    return dtype == MR_DTYPE_F32   ? launch_dims<float>(ctx, a)
           : dtype == MR_DTYPE_F16 ? launch_dims<__half>(ctx, a)
                                   : launch_dims<__nv_bfloat16>(ctx, a);
}

}  // namespace cache
}  // namespace mr
