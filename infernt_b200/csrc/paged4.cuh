// paged4.cuh — pages that hold K and V in 4 bits: the format, and what the
// operators over it share (paged4.cu, paged4_attention.cu,
// paged_attention_tc.cu).
//
// The vector x of a KV head at a position is held as D codes of 4 bits and a
// scale word of 16:
//   s = (max(x, 0) - min(x, 0)) / 15, rounded up to four significant bits,
//   z = round(-min(x, 0) / s),  c_i = round(x_i / s) + z, held to 0..15,
//   value = (c_i - z) s.
// c - z has at most four bits and s has four, so a value has eight: it is a
// number of bf16 and of fp16 as it is.  So a product on the tensor cores may
// take either the values or the whole numbers c - z with s applied to the
// sums, and both are exact (with a scale of bf16's eight bits the values would
// be rounded in one kernel and not in the other).  The step is at most 1/8
// wider than the range needs, or kLeastScale4.  |x_i - value| <= s / 2, but up to
// s where the nearest multiple of s is past the largest number of T.
// The word: the upper twelve bits of s as a bf16, z in the low four.  A vector
// with a value that is NaN or past the largest number of T has a scale of NaN.
#pragma once

#include "paged.cuh"

namespace infernt {

// Largest finite value, and the least scale: below it products of the whole
// numbers would not be numbers of the type (fp16: 2^-24 is its last bit).
template <typename T>
constexpr float kLargest4 = Half16<T>::kBf16 ? 3.3895313892515355e38f : 65504.0f;
template <typename T>
constexpr float kLeastScale4 = Half16<T>::kBf16 ? 7.888609052210118e-31f : 4.76837158203125e-07f;  // 2^-100, 2^-21
constexpr uint32_t kNotFinite4 = 0x7ff0u;

__device__ __forceinline__ float scale4(uint32_t word) { return __uint_as_float((word & 0xfff0u) << 16); }

// (w & mask) | one, in one operation.
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t one) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(one));
    return r;
}

// Pairs of codes as 16-bit floats: the exponent of 2^m puts a code in the last
// bits of the mantissa (bf16: m = 7; fp16: 10), and what is taken off after it,
// 2^m + z, leaves c - z exactly.  The mask and 2^m come out of registers that
// the compiler cannot see through: as immediates they take two operations.
template <typename T>
struct Codes4;
template <>
struct Codes4<__nv_bfloat16> {
    static constexpr uint32_t kOne = 0x43004300u;
    static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ uint32_t mul(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
};
template <>
struct Codes4<__half> {
    static constexpr uint32_t kOne = 0x64006400u;
    static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ uint32_t mul(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
};
struct Masks4 {
    uint32_t low, one;
};
template <typename T>
__device__ __forceinline__ Masks4 make_masks4() {
    Masks4 k;
    asm volatile("mov.b32 %0, 0x000f000f;" : "=r"(k.low));
    asm volatile("mov.b32 %0, %1;" : "=r"(k.one) : "n"(Codes4<T>::kOne));
    return k;
}
// 2^m + z in both halves, of a scale word.
__device__ __forceinline__ uint32_t zeros4(uint32_t word, const Masks4& k) {
    return and_or(__byte_perm(word, word, 0x1010), k.low, k.one);
}

// Eight values, element j in bits 4 j ... of w, as pairs (j, j + 4); s2: the
// scale as a T in both halves.
template <typename T>
__device__ __forceinline__ void pairs4(uint32_t w, uint32_t z2, uint32_t s2, const Masks4& k, uint32_t (&p)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
        p[j] = Codes4<T>::mul(Codes4<T>::sub(and_or(w >> (4 * j), k.low, k.one), z2), s2);
}
// In their order, as the 16 bytes of a row of T.
template <typename T>
__device__ __forceinline__ uint4 values4(uint32_t w, uint32_t z2, uint32_t s2, const Masks4& k) {
    uint32_t p[4];
    pairs4<T>(w, z2, s2, k, p);
    // (0, 4) (1, 5) (2, 6) (3, 7) -> (0, 1) (2, 3) (4, 5) (6, 7)
    return make_uint4(__byte_perm(p[0], p[1], 0x5410), __byte_perm(p[2], p[3], 0x5410),
                      __byte_perm(p[0], p[1], 0x7632), __byte_perm(p[2], p[3], 0x7632));
}
template <typename T>
__device__ __forceinline__ uint32_t scale_pair4(uint32_t word) {
    const float s = scale4(word);
    return Half16<T>::pack(s, s);
}

// Checks of a 4-bit cache (paged4.cu), and its geometry as that of 16-bit
// pools for the checks and the batch of the kernels.
int check_paged_cache4(const char* op, const infernt_paged_cache4* c);
inline infernt_paged_cache geometry4(const infernt_paged_cache4& c) {
    return {c.k, c.v, c.num_pages, c.num_kv_heads, c.page_size, c.head_dim, c.dtype};
}

}  // namespace infernt
