// paged_rope.cuh — what the rotary appends share (paged_rope.cu, paged4.cu):
// the way from a token row to its position and page row, angles, and 16-byte
// loads of a row's values.
#pragma once

#include "paged.cuh"

namespace infernt {

constexpr int kRopeThreads = 128;
constexpr int kMaxPairs = 64;

struct RopeDev {
    double turns[kMaxPairs];  // f_i / 2 pi
    double magnitude64;       // what cosine and sine are multiplied by
    float magnitude;
    int half, interleaved;
};

struct RopeArgs {
    PagedBatch b;
    const void* q;
    const void* k;
    const void* v;
    void* q_out;
    void* kp;
    void* vp;
    long long ldq, ldk, ldv, ldo;
    int nq, D;
    unsigned* err;
};

template <typename S>
__device__ __forceinline__ float source_value(const S* p) {
    return to_f32(*p);
}
template <>
__device__ __forceinline__ float source_value<__half>(const __half* p) {
    return __half2float(*p);
}

// Where row r of the batch goes: its sequence's position, and the page row of
// head 0 (-1: nowhere).  False: the row stays as it is.
__device__ __forceinline__ bool place_row(const RopeArgs& a, int r, int& pos, long long& row) {
    const int s = find_seq(a.b.q_start, a.b.num_seqs, r);
    const PagedSeq seq = paged_seq(a.b, s, a.err);
    const int i = r - seq.row0;
    if (i < 0 || i >= seq.n_new) return false;  // behind the last sequence, or a sequence that is skipped
    pos = seq.len - seq.n_new + i;
    if (pos < 0) return false;
    row = -1;
    if (a.k) {
        const int pi = a.b.by_page(pos), page = a.b.table[(size_t)s * a.b.table_stride + pi];
        if (page >= 0 && page < a.b.num_pages)
            row = (long long)page * a.b.nkv * a.b.page_size + (pos - pi * a.b.page_size);
        else if (a.err && threadIdx.x == 0)
            atomicOr(a.err, kErrPage);
    }
    return true;
}

// Error bits of the sequences: this block's share of them, since one that no row
// leads to (no new tokens, or a start above its end) is met nowhere else.
__device__ __forceinline__ void check_sequences(const RopeArgs& a) {
    if (a.err && threadIdx.x == kRopeThreads - 1)
        for (int s = blockIdx.x; s < a.b.num_seqs; s += gridDim.x) paged_seq(a.b, s, a.err);
}

// Cosine and sine of pair p at position pos, times the magnitude.
__device__ __forceinline__ float2 turn_of(const RopeDev& rope, int p, int pos) {
    const double t = (double)pos * rope.turns[p];
    const float f = (float)(t - rint(t));  // [-1/2, 1/2] turns
    float sn, c;
    sincospif(2.0f * f, &sn, &c);
    return make_float2(c * rope.magnitude, sn * rope.magnitude);
}

// Eight values of a row as loaded, and as FP32.
template <typename S>
struct Eight {
    uint4 w[sizeof(S) / 2];
};
template <typename S>
__device__ __forceinline__ Eight<S> load_eight(const S* p) {
    Eight<S> v;
#pragma unroll
    for (int i = 0; i < (int)sizeof(S) / 2; ++i) v.w[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
    return v;
}
__device__ __forceinline__ void to_floats(const Eight<float>& v, float (&x)[8]) {
    const uint32_t w[8] = {v.w[0].x, v.w[0].y, v.w[0].z, v.w[0].w, v.w[1].x, v.w[1].y, v.w[1].z, v.w[1].w};
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
}
template <typename S>
__device__ __forceinline__ void to_floats(const Eight<S>& v, float (&x)[8]) {
    const uint32_t w[4] = {v.w[0].x, v.w[0].y, v.w[0].z, v.w[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = Half16<S>::unpack(w[i]);
        x[2 * i] = p.x;
        x[2 * i + 1] = p.y;
    }
}
template <typename T>
__device__ __forceinline__ void store_eight(T* p, const float (&x)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(Half16<T>::pack(x[0], x[1]), Half16<T>::pack(x[2], x[3]),
                                              Half16<T>::pack(x[4], x[5]), Half16<T>::pack(x[6], x[7]));
}

// Checks p and fills *out for heads of head_dim (paged_rope.cu).
int rope_frequencies(const char* op, const infernt_rope_params& p, int head_dim, RopeDev* out);
// The checks of a rotary append's arguments but for its cache, and a without
// its batch and pools; *empty: nothing to do.
int rope_append_args(const char* op, void* q_out, int ldo, const void* q, int ldq, int nq, const void* k, int ldk,
                     const void* v, int ldv, int src_dtype, int nkv, int head_dim, int dtype,
                     const infernt_ragged_batch* batch, const infernt_rope_params* rope, const unsigned* err,
                     RopeArgs* a, RopeDev* d, bool* empty);

}  // namespace infernt
