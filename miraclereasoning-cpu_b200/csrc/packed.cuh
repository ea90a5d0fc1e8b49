// Rows of a cache held in 4 bits a value.
//
// A row of a page, of one key / value head, is 5 dim / 8 bytes: dim / 2 bytes of
// codes, the even dim in a byte's low half, and behind them two float16 numbers for
// each 32 dims, a step s and a base z.  Code c stands for s (64 + c) + z, rounded to
// float16 once.  The base is that of code -64, not of code 0, because a code ored
// into the fraction of float16's 64 is the number 64 + c: a pair of a word's codes becomes
// an operand of one fused multiply-add by a logical operation, behind a shift for
// three pairs of the four.  (The base's own rounding,
// 2^-11 of about 4.8 times the spread of the 32 values, moves a value by 4% of a step.)
#pragma once

#include "cache_ops.cuh"

namespace mr {
namespace cache {

constexpr int kShared = 32;  // values that share a step and a base

inline int64_t packed_dim(int64_t bytes) { return bytes * 8 / 5; }
// What the start of every row is a multiple of: a row's own bytes, up to 16.
inline int packed_unit(int64_t bytes) { return static_cast<int>(std::min<int64_t>(bytes & -bytes, 16)); }

// A key and a value pool of 4-bit rows.
inline int check_packed(const mr_array *k, const mr_array *v, const char *kn, const char *vn, bool written) {
    MR_CHECK(check_array(k, kn, 4, false, written));
    MR_CHECK(check_array(v, vn, 4, false, written));
    MR_REQUIRE(k->dtype == MR_DTYPE_U8 && v->dtype == MR_DTYPE_U8, "%s and %s must be of one type", kn, vn);
    for (int i = 0; i < 4; ++i) MR_REQUIRE(k->shape[i] == v->shape[i], "%s and %s differ in shape", kn, vn);
    MR_REQUIRE(k->shape[1] > 0 && k->shape[2] > 0, "%s: an empty page row", kn);
    const int64_t bytes = k->shape[3];
    MR_REQUIRE(bytes == 20 || bytes == 40 || bytes == 60 || bytes == 80,
               "%s: rows of 4-bit values must be 20, 40, 60 or 80 bytes (head dims 32, 64, 96, 128), not %lld", kn,
               static_cast<long long>(bytes));
    const int unit = packed_unit(bytes);
    for (const mr_array *a : {k, v}) {
        const char *name = a == k ? kn : vn;
        MR_REQUIRE(reinterpret_cast<uintptr_t>(a->data) % unit == 0, "%s must start on a %d-byte boundary", name, unit);
        for (int i = 0; i < 3; ++i)
            MR_REQUIRE(a->shape[i] == 1 || a->stride[i] % unit == 0, "%s: stride %d is not a multiple of %d bytes", name, i,
                       unit);
    }
    return MR_OK;
}

// Two codes of a word, those of bits 4 .. 7 of each half, as the numbers 64 + c.
__device__ __forceinline__ uint32_t codes64(uint32_t word) {
    uint32_t x;
    asm("lop3.b32 %0, %1, 0x00f000f0, 0x54005400, 0xea;" : "=r"(x) : "r"(word));
    return x;
}
// All eight codes of a word, those n and n + 4 of the natural order in c[n].
__device__ __forceinline__ void word_codes(uint32_t word, uint32_t (&c)[4]) {
    c[0] = codes64(word << 4);
    c[1] = codes64(word);
    c[2] = codes64(word >> 4);
    c[3] = codes64(word >> 8);
}
// s (64 + c) + z of two codes.
__device__ __forceinline__ uint32_t fma2(uint32_t codes, __half2 s, __half2 z) {
    const __half2 x = __hfma2(*reinterpret_cast<const __half2 *>(&codes), s, z);
    return *reinterpret_cast<const uint32_t *>(&x);
}

}  // namespace cache
}  // namespace mr
