// paged.cuh — what the operators over paged caches share (paged_rope.cu,
// paged_attention.cu): the ragged batch on the device, the way from a token
// row to its sequence, the argument checks, and the two 16-bit types.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "common.cuh"
#include "internal.h"

namespace infernt {

// Positions and rows stay below it, so that sums of two of them fit an int.
constexpr int kMaxPositions = 1 << 30;

// n / d for 0 <= n < 2^31 by a product: with 2^(L - 1) < d <= 2^L the factor
// ceil(2^(31 + L) / d) is off by less than d / 2^(31 + L), which the quotient
// of such an n does not see (Granlund and Montgomery 1994).
struct FastDiv {
    uint32_t factor;
    int shift;
    __device__ __forceinline__ int operator()(int n) const {
        return (int)(((unsigned long long)(uint32_t)n * factor) >> shift);
    }
};
inline FastDiv fast_div(int d) {
    int L = 0;
    while (L < 31 && (1ll << L) < d) ++L;
    return {(uint32_t)(((1ull << (31 + L)) + (unsigned)d - 1) / (unsigned)d), 31 + L};
}

// infernt_ragged_batch and the pool geometry as the kernels take them.
struct PagedBatch {
    const int* q_start;
    const int* kv_len;
    const int* table;
    int table_stride, num_seqs, num_rows, max_q_len;
    int num_pages, page_size, nkv;
    FastDiv by_page;
};

// One sequence of a batch: rows [row0, row0 + n_new), length len.
struct PagedSeq {
    int row0, n_new, len;
};

// Sequence s, or no rows (and the error bit) when the device arrays hold
// something out of range: nothing is read or written through such a sequence.
__device__ __forceinline__ PagedSeq paged_seq(const PagedBatch& b, int s, unsigned* err) {
    PagedSeq r;
    r.row0 = b.q_start[s];
    const int end = b.q_start[s + 1];
    r.len = b.kv_len[s];
    r.n_new = end - r.row0;
    const bool ok = r.row0 >= 0 && end >= r.row0 && end <= b.num_rows && r.n_new <= b.max_q_len && r.len >= 0 &&
                    r.len <= kMaxPositions && r.len <= (long long)b.table_stride * b.page_size;
    if (!ok) {
        if (err) atomicOr(err, kErrBatch);
        r.row0 = r.n_new = r.len = 0;
    }
    return r;
}

// bf16 and fp16 as the tensor cores and the stores take them.
template <typename T>
struct Half16;

template <>
struct Half16<__nv_bfloat16> {
    static constexpr bool kBf16 = true;
    // (a, b) rounded to nearest even, a in the low half
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        uint32_t r;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
        return r;
    }
    static __device__ __forceinline__ float2 unpack(uint32_t v) {
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    }
    static __device__ __forceinline__ __nv_bfloat16 round(float a) { return __float2bfloat16_rn(a); }
    static __device__ __forceinline__ uint32_t add_zero_times(uint32_t v, uint32_t sum) {
        uint32_t r;
        asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(v), "r"(0u), "r"(sum));
        return r;
    }
    // ones in each half that is infinite or NaN: an exponent of ones carries into the sign
    static __device__ __forceinline__ uint32_t not_finite(uint32_t v) {
        return ((((v & 0x7f807f80u) + 0x00800080u) & 0x80008000u) >> 15) * 0xffffu;
    }
};

template <>
struct Half16<__half> {
    static constexpr bool kBf16 = false;
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        uint32_t r;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
        return r;
    }
    static __device__ __forceinline__ float2 unpack(uint32_t v) {
        return make_float2(__half2float(__ushort_as_half((unsigned short)(v & 0xffffu))),
                           __half2float(__ushort_as_half((unsigned short)(v >> 16))));
    }
    static __device__ __forceinline__ __half round(float a) { return __float2half_rn(a); }
    static __device__ __forceinline__ uint32_t add_zero_times(uint32_t v, uint32_t sum) {
        uint32_t r;
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(v), "r"(0u), "r"(sum));
        return r;
    }
    static __device__ __forceinline__ uint32_t not_finite(uint32_t v) {
        return ((((v & 0x7c007c00u) + 0x04000400u) & 0x80008000u) >> 15) * 0xffffu;
    }
};

// Lets kernel use `bytes` of dynamic shared memory: once a kernel and device,
// since the setting stays (set_on has a bit per device).
template <typename K>
inline int allow_smem(K kernel, int bytes, std::atomic<unsigned long long>& set_on) {
    const int d = current_device();
    const unsigned long long bit = d >= 0 && d < 64 ? 1ull << d : 0;
    if (set_on.load(std::memory_order_acquire) & bit) return INFERNT_OK;
    INFERNT_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    set_on.fetch_or(bit, std::memory_order_release);
    return INFERNT_OK;
}

// Argument checks that the operators share (paged_rope.cu).
int check_paged_cache(const char* op, const infernt_paged_cache* c);
int check_ragged_batch(const char* op, const infernt_ragged_batch* b);
// p (or NULL) must be memory that the current device reads in place.
int check_device_pointer(const char* op, const char* what, const void* p);
int check_batch_pointers(const char* op, const infernt_paged_cache* c, const infernt_ragged_batch* b, const void* err);

inline PagedBatch paged_batch(const infernt_paged_cache& c, const infernt_ragged_batch& b) {
    PagedBatch r;
    r.q_start = b.q_start;
    r.kv_len = b.kv_len;
    r.table = b.block_table;
    r.table_stride = b.table_stride;
    r.num_seqs = b.num_seqs;
    r.num_rows = b.num_rows;
    r.max_q_len = b.max_q_len;
    r.num_pages = c.num_pages;
    r.page_size = c.page_size;
    r.nkv = c.num_kv_heads;
    r.by_page = fast_div(c.page_size);
    return r;
}

}  // namespace infernt
