// paged4.cu — K and V rows into pages of 4 bits (with the rotary positions of
// paged_rope.cu), and pages' values out again.  paged4.cuh has the format.
//
// Codes go by which side of a border a value is on, so K turns in 64 bits and
// is rounded once to FP32: what a page holds then depends on nothing but the
// rows and the position, not on the last bit of an FP32 sine, and pages of the
// same prefix are the same bits whoever wrote them.
#include <cmath>
#include <cstdint>

#include "paged4.cuh"
#include "paged_rope.cuh"

namespace infernt {

int check_paged_cache4(const char* op, const infernt_paged_cache4* c) {
    INFERNT_REQUIRE(c && c->scales, "%s: null cache", op);
    const infernt_paged_cache g = geometry4(*c);
    if (int s = check_paged_cache(op, &g)) return s;
    INFERNT_REQUIRE(reinterpret_cast<uintptr_t>(c->scales) % 4 == 0, "%s: misaligned scales", op);
    return INFERNT_OK;
}

namespace {

// The largest and least of some values and 0; NaN where one of them is.
struct Range4 {
    float hi, lo;
};
__device__ __forceinline__ float max_of(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float min_of(float a, float b, float c) {
    float r;
    asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
template <int N>
__device__ __forceinline__ void widen(Range4& r, const float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        r.hi = max_of(r.hi, x[i], x[i + 1]);
        r.lo = min_of(r.lo, x[i], x[i + 1]);
    }
}
// Over groups of `lanes` neighbouring lanes (a power of two), by whole warps.
__device__ __forceinline__ void join(Range4& r, int lanes) {
    for (int o = lanes >> 1; o > 0; o >>= 1) {
        const float hi = __shfl_xor_sync(0xffffffffu, r.hi, o), lo = __shfl_xor_sync(0xffffffffu, r.lo, o);
        r.hi = max_of(r.hi, hi, hi);
        r.lo = min_of(r.lo, lo, lo);
    }
}

// A vector's scale, zero and word.  k is the whole number nearest to x / s, a
// tie's even one, which is the rounding of the correctly rounded quotient too:
// s has four bits, so x - (k + 1/2) s is a whole number of x's last places, and
// one of them is more than half a last place of x / s.
constexpr float kWhole = 12582912.0f;  // 1.5 x 2^23 brings a whole number into the low bits
struct Scale4 {
    float s, z;
    float inverse;  // 1 / s
    bool far;       // a rounding may carry a value past the largest number of T, or the vector is not finite
    uint32_t word;
};
// The low bits: k + those of kWhole.  k by x (1 / s) is off by one at most, near
// ties, which the exact x - k s shows.
__device__ __forceinline__ int nearest(float x, const Scale4& q) {
    const float t = __fmaf_rn(x, q.inverse, kWhole);
    const float r = __fmaf_rn(-__fadd_rn(t, -kWhole), q.s, x);
    const int bits = __float_as_int(t), sign = __float_as_int(r) >> 31;  // 0 or -1
    // past the tie, or at it with an odd k
    const bool off = (__float_as_int(r) & 0x7fffffff) + (bits & 1) > __float_as_int(0.5f * q.s);
    return off ? bits + (sign | 1) : bits;
}
template <typename T>
__device__ __forceinline__ Scale4 scale_of(const Range4& r) {
    Scale4 q;
    const float most = max_of(r.hi, -r.lo, 0.0f);
    const bool fine = most <= kLargest4<T>;  // (false for NaN)
    // halves of both sides: the range of numbers near the largest would be infinite
    const float s = __fdiv_rn(0.5f * r.hi - 0.5f * r.lo, 7.5f);
    q.s = fine ? fmaxf(__uint_as_float((__float_as_uint(s) + 0xfffffu) & ~0xfffffu), kLeastScale4<T>) : 1.0f;
    q.inverse = __frcp_rn(q.s);
    q.far = !(most <= 0.5f * kLargest4<T>);
    q.z = fminf(rintf(__fdiv_rn(-r.lo, q.s)), 15.0f);
    q.word = fine ? (__float_as_uint(q.s) >> 16) | (uint32_t)q.z : kNotFinite4;
    return q;
}
// The codes of N neighbouring values, the first in the lowest bits.
template <typename T, int N>
__device__ __forceinline__ uint32_t codes_of(const float (&x)[N], const Scale4& q) {
    uint32_t c = 0;
    if (!q.far) {
        const int up = (int)q.z - __float_as_int(kWhole);
#pragma unroll
        for (int i = 0; i < N; ++i) c |= (uint32_t)max(min(nearest(x[i], q) + up, 15), 0) << (4 * i);
        return c;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float k = rintf(__fdiv_rn(x[i], q.s));
        // a rounding past the largest number of T goes the other way
        if (fabsf(k * q.s) > kLargest4<T>) k -= copysignf(1.0f, k);
        c |= (uint32_t)fminf(fmaxf(k + q.z, 0.0f), 15.0f) << (4 * i);  // (NaN: 0)
    }
    return c;
}

// As turn_of, in 64 bits.
__device__ __forceinline__ double2 turn_of64(const RopeDev& rope, int p, int pos) {
    const double t = (double)pos * rope.turns[p];
    double sn, c;
    sincospi(2.0 * (t - rint(t)), &sn, &c);
    return make_double2(c * rope.magnitude64, sn * rope.magnitude64);
}
__device__ __forceinline__ void turn64(float& x, float& y, double2 cs) {
    const double a = x, b = y;
    x = (float)(a * cs.x - b * cs.y);
    y = (float)(b * cs.x + a * cs.y);
}

// The blocks and units of paged_rope_wide (paged_rope.cu): a block per token
// row, a thread two blocks of eight values of a head, D / 16 threads a head.
// These find the head's range by shuffles and store a word of codes per block.
// 8192 bf16 rows of 32/8 heads of 128, 176 MB: 42 us, 4.2 TB/s; bound by
// instructions, most of them a K or V value's rounding and packing (Q alone
// takes 33; with divisions in place of nearest 45), with more blocks an SM as
// fast.  320 FP32 rows: 7.5 us.
constexpr int kAhead4 = 3;

template <typename S, typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(kRopeThreads)
    paged4_rope_wide(const RopeArgs a, const __grid_constant__ RopeDev rope, uint16_t* scales) {
    __shared__ float2 cs_s[kMaxPairs];
    __shared__ double2 cs64_s[kMaxPairs];
    const int r = blockIdx.x, tid = threadIdx.x, D = a.D, R = 2 * rope.half, nkv = a.b.nkv;
    const int log_u = D == 64 ? 2 : 3, w = tid & ((1 << log_u) - 1);
    const int heads_q = a.q ? a.nq : 0, heads = heads_q + (a.k ? 2 * nkv : 0);
    const bool turns = w < R / 16;
    // this thread's two blocks of a q or k head, and of a v head
    const int lo = turns ? 8 * w : R + 8 * (w - R / 16), hi = turns ? lo + R / 2 : lo + (D - R) / 2;
    auto source = [&](int h) {
        if (h < heads_q) return static_cast<const S*>(a.q) + r * a.ldq + (long long)h * D;
        h -= heads_q;
        return h < nkv ? static_cast<const S*>(a.k) + r * a.ldk + (long long)h * D
                       : static_cast<const S*>(a.v) + r * a.ldv + (long long)(h - nkv) * D;
    };
    const int h0 = tid >> log_u, step = kRopeThreads >> log_u;
    Eight<S> x[kAhead4], y[kAhead4];
#pragma unroll
    for (int i = 0; i < kAhead4; ++i) {
        const int h = min(h0 + i * step, heads - 1);
        const S* p = source(h);
        const bool is_v = h >= heads_q + nkv;
        x[i] = load_eight(p + (is_v ? 8 * w : lo));
        y[i] = load_eight(p + (is_v ? D / 2 + 8 * w : hi));
    }
    int pos;
    long long row;
    if (!place_row(a, r, pos, row)) {
        check_sequences(a);
        return;
    }
    // Turn e of a thread is that of element e of its first block, or (interleaved) of elements 2 e, 2 e + 1 of the
    // first and then the second; those of neighbouring threads lie next to each other, or they would meet in the banks.
    auto pair = [&](int e) { return 8 * e + w; };
    if (tid < rope.half) {
        const int p = tid, late = INTERLEAVED && p >= rope.half / 2 ? 4 : 0, x = late ? p - rope.half / 2 : p;
        const int at = INTERLEAVED ? 8 * (late + x % 4) + x / 4 : 8 * (p % 8) + p / 8;
        if (a.k) {
            const double2 cs = turn_of64(rope, p, pos);
            cs64_s[at] = cs;
            cs_s[at] = make_float2((float)cs.x, (float)cs.y);
        } else {
            cs_s[at] = turn_of(rope, p, pos);
        }
    }
    __syncthreads();
    // h: the head; of a thread past the last one, that one, and nothing is stored
    auto finish = [&](int h, const Eight<S>& ex, const Eight<S>& ey) {
        const bool live = h < heads;
        h = min(h, heads - 1);
        const bool is_q = h < heads_q, is_v = h >= heads_q + nkv;
        float u[8], v[8];
        to_floats(ex, u);
        to_floats(ey, v);
        if (is_q) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float2 cs = turns ? cs_s[pair(e)] : make_float2(1.0f, 0.0f);
                float& p = !INTERLEAVED ? u[e] : e < 4 ? u[2 * e] : v[2 * e - 8];
                float& q = !INTERLEAVED ? v[e] : e < 4 ? u[2 * e + 1] : v[2 * e - 7];
                const float p0 = p, q0 = q;
                p = p0 * cs.x - q0 * cs.y;
                q = q0 * cs.x + p0 * cs.y;
            }
            if (live) {
                T* dst = static_cast<T*>(a.q_out) + r * a.ldo + (long long)h * D;
                store_eight(dst + lo, u);
                store_eight(dst + hi, v);
            }
        } else if (!is_v && turns) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float& p = !INTERLEAVED ? u[e] : e < 4 ? u[2 * e] : v[2 * e - 8];
                float& q = !INTERLEAVED ? v[e] : e < 4 ? u[2 * e + 1] : v[2 * e - 7];
                turn64(p, q, cs64_s[pair(e)]);
            }
        }
        if (__all_sync(0xffffffffu, is_q)) return;
        Range4 range = {0.0f, 0.0f};
        widen(range, u);
        widen(range, v);
        join(range, 1 << log_u);
        if (is_q || !live || row < 0) return;
        const Scale4 q = scale_of<T>(range);
        const uint32_t cu = codes_of<T, 8>(u, q), cv = codes_of<T, 8>(v, q);
        const int kh = h - heads_q;
        const long long at = row + (long long)(is_v ? kh - nkv : kh) * a.b.page_size;
        uint32_t* dst = static_cast<uint32_t*>(is_v ? a.vp : a.kp) + at * (D / 8);
        dst[is_v ? w : lo / 8] = cu;
        dst[is_v ? D / 16 + w : hi / 8] = cv;
        if (w == 0) scales[2 * at + is_v] = (uint16_t)q.word;
    };
#pragma unroll
    for (int i = 0; i < kAhead4; ++i)
        if (i * step < heads) finish(h0 + i * step, x[i], y[i]);
    for (int i = kAhead4; i * step < heads; ++i) {
        const int h = min(h0 + i * step, heads - 1);
        const S* p = source(h);
        const bool is_v = h >= heads_q + nkv;
        finish(h0 + i * step, load_eight(p + (is_v ? 8 * w : lo)), load_eight(p + (is_v ? D / 2 + 8 * w : hi)));
    }
    check_sequences(a);
}

// Any other rotary_dim, stride or alignment: a block per token row, a warp per
// head, D / 32 neighbouring values a lane.  8192 bf16 rows of 32/8 heads of 128,
// 126 of them turned: 135 us (over 16-bit pages 116); 320 rows 13.  Bound by
// instructions: both lanes of a split-half pair turn it in 64 bits, for the half
// that is theirs, and loads are of 2 to 16 bytes a lane.
template <typename S, typename T, int D>
__global__ void __launch_bounds__(kRopeThreads)
    paged4_rope(const RopeArgs a, const __grid_constant__ RopeDev rope, uint16_t* scales) {
    constexpr int N = D / 32;
    __shared__ double2 cs[kMaxPairs];
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 31, half = rope.half, nkv = a.b.nkv;
    int pos;
    long long row;
    if (!place_row(a, r, pos, row)) {
        check_sequences(a);
        return;
    }
    if (tid < half) cs[tid] = turn_of64(rope, tid, pos);
    __syncthreads();
    const int heads_q = a.q ? a.nq : 0, heads = heads_q + (row >= 0 ? 2 * nkv : 0);
    for (int h = tid >> 5; h < heads; h += kRopeThreads / 32) {
        const bool is_v = h >= heads_q + nkv;
        const S* src = h < heads_q ? static_cast<const S*>(a.q) + r * a.ldq + (long long)h * D
                       : !is_v     ? static_cast<const S*>(a.k) + r * a.ldk + (long long)(h - heads_q) * D
                                   : static_cast<const S*>(a.v) + r * a.ldv + (long long)(h - heads_q - nkv) * D;
        float x[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = N * lane + i;
            x[i] = source_value(src + e);
            if (e < 2 * half && !is_v) {
                const bool second = rope.interleaved ? e & 1 : e >= half;
                const int p = rope.interleaved ? e >> 1 : second ? e - half : e;
                const int o = rope.interleaved ? e ^ 1 : second ? e - half : e + half;
                float y = source_value(src + o);
                if (second) {
                    turn64(y, x[i], cs[p]);
                } else {
                    turn64(x[i], y, cs[p]);
                }
            }
        }
        if (h < heads_q) {
            T* dst = static_cast<T*>(a.q_out) + r * a.ldo + (long long)h * D;
            __syncwarp();  // q_out may be q: every lane has read its partners
#pragma unroll
            for (int i = 0; i < N; ++i) dst[N * lane + i] = Half16<T>::round(x[i]);
            continue;
        }
        Range4 range = {0.0f, 0.0f};
        widen(range, x);
        join(range, 32);
        const Scale4 q = scale_of<T>(range);
        const int kh = h - heads_q;
        const long long at = row + (long long)(is_v ? kh - nkv : kh) * a.b.page_size;
        uint8_t* dst = static_cast<uint8_t*>(is_v ? a.vp : a.kp) + at * (D / 2) + lane * (N / 2);
        const uint32_t c = codes_of<T, N>(x, q);
#pragma unroll
        for (int i = 0; i < N; i += 2) dst[i / 2] = (uint8_t)(c >> (4 * i));
        if (lane == 0) scales[2 * at + is_v] = (uint16_t)q.word;
    }
    check_sequences(a);
}

template <typename S, typename T>
int launch(const RopeArgs& a, const RopeDev& d, uint16_t* scales, cudaStream_t st) {
    // rows of S or T `ld` apart that start where 16 bytes may be loaded
    auto wide = [](const void* p, long long ld, size_t size) { return !p || (aligned16(p) && ld * size % 16 == 0); };
    if (d.half % 8 == 0 && wide(a.q, a.ldq, sizeof(S)) && wide(a.k, a.ldk, sizeof(S)) && wide(a.v, a.ldv, sizeof(S)) &&
        wide(a.q_out, a.ldo, sizeof(T))) {
        if (d.interleaved)
            paged4_rope_wide<S, T, true><<<a.b.num_rows, kRopeThreads, 0, st>>>(a, d, scales);
        else
            paged4_rope_wide<S, T, false><<<a.b.num_rows, kRopeThreads, 0, st>>>(a, d, scales);
    } else if (a.D == 64) {
        paged4_rope<S, T, 64><<<a.b.num_rows, kRopeThreads, 0, st>>>(a, d, scales);
    } else {
        paged4_rope<S, T, 128><<<a.b.num_rows, kRopeThreads, 0, st>>>(a, d, scales);
    }
    INFERNT_CUDA_TRY(cudaGetLastError());
    return INFERNT_OK;
}

template <typename T>
int launch_src(const RopeArgs& a, const RopeDev& d, uint16_t* scales, int src, cudaStream_t st) {
    if (src == INFERNT_DTYPE_F32) return launch<float, T>(a, d, scales, st);
    if (src == INFERNT_DTYPE_BF16) return launch<__nv_bfloat16, T>(a, d, scales, st);
    return launch<__half, T>(a, d, scales, st);
}

// ------------------------------------------------- values out of the pages
// A thread takes words of eight codes, neighbours in a page: 4 bytes in, 16
// out, for K and then for V, four at once.  8288 positions of 8 heads of 128, 43
// MB: 7.9 us, 5.4 TB/s, 1.2 times what HBM takes; the rest is start and end.
constexpr int kUnpackThreads = 256;
constexpr int kUnpackAtOnce = 4;

struct UnpackArgs {
    const uint32_t* k4;
    const uint32_t* v4;
    const uint32_t* scales;
    uint4* k;
    uint4* v;
    const int* src;
    const int* dst;
    int n, page_words;  // pages, and words of one
    int pages_in, pages_out, log_row;  // a row has 2^log_row words
    unsigned* err;
};

template <typename T>
__global__ void __launch_bounds__(kUnpackThreads) paged4_unpack(const UnpackArgs a) {
    const Masks4 mk = make_masks4<T>();
    // y: pages, x: parts of a page
    for (int m = blockIdx.y; m < a.n; m += gridDim.y) {
        const int from = a.src[m], to = a.dst[m];
        if (from < 0 || from >= a.pages_in || to < 0 || to >= a.pages_out) {
            if (a.err && threadIdx.x == 0) atomicOr(a.err, kErrPage);
            continue;
        }
        const long long in = (long long)from * a.page_words, out = (long long)to * a.page_words;
        for (int base = blockIdx.x * kUnpackThreads * kUnpackAtOnce; base < a.page_words;
             base += gridDim.x * kUnpackThreads * kUnpackAtOnce) {
            uint32_t wk[kUnpackAtOnce], wv[kUnpackAtOnce], sc[kUnpackAtOnce];
#pragma unroll
            for (int i = 0; i < kUnpackAtOnce; ++i) {
                const int at = min(base + i * kUnpackThreads + (int)threadIdx.x, a.page_words - 1);
                wk[i] = __ldcs(a.k4 + in + at);
                wv[i] = __ldcs(a.v4 + in + at);
                sc[i] = __ldg(a.scales + ((in + at) >> a.log_row));
            }
#pragma unroll
            for (int i = 0; i < kUnpackAtOnce; ++i) {
                const int at = base + i * kUnpackThreads + (int)threadIdx.x;
                if (at >= a.page_words) break;
                const uint32_t sk = sc[i] & 0xffffu, sv = sc[i] >> 16;
                a.k[out + at] = values4<T>(wk[i], zeros4(sk, mk), scale_pair4<T>(sk), mk);
                a.v[out + at] = values4<T>(wv[i], zeros4(sv, mk), scale_pair4<T>(sv), mk);
            }
        }
    }
}

}  // namespace
}  // namespace infernt

extern "C" int infernt_paged4_rope_append(void* q_out, int ldo, const void* q, int ldq, int nq, const void* k, int ldk,
                                          const void* v, int ldv, int src_dtype, const infernt_paged_cache4* cache,
                                          const infernt_ragged_batch* batch, const infernt_rope_params* rope,
                                          unsigned* err, void* stream) {
    using namespace infernt;
    const char* op = "paged4_rope_append";
    if (int s = check_paged_cache4(op, cache)) return s;
    if (int s = check_ragged_batch(op, batch)) return s;
    RopeArgs a;
    RopeDev d;
    bool empty;
    if (int s = rope_append_args(op, q_out, ldo, q, ldq, nq, k, ldk, v, ldv, src_dtype, cache->num_kv_heads,
                                 cache->head_dim, cache->dtype, batch, rope, err, &a, &d, &empty))
        return s;
    if (empty) return INFERNT_OK;
    const infernt_paged_cache g = geometry4(*cache);
    if (int s = check_batch_pointers(op, &g, batch, err)) return s;
    if (int s = check_device_pointer(op, "the scales", cache->scales)) return s;
    a.b = paged_batch(g, *batch);
    a.kp = cache->k;
    a.vp = cache->v;
    a.err = err;
    uint16_t* scales = reinterpret_cast<uint16_t*>(cache->scales);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return cache->dtype == INFERNT_DTYPE_BF16 ? launch_src<__nv_bfloat16>(a, d, scales, src_dtype, st)
                                              : launch_src<__half>(a, d, scales, src_dtype, st);
}

extern "C" int infernt_paged4_unpack(const infernt_paged_cache4* from, const infernt_paged_cache* to, const int* src,
                                     const int* dst, int n, unsigned* err, void* stream) {
    using namespace infernt;
    const char* op = "paged4_unpack";
    if (int s = check_paged_cache4(op, from)) return s;
    if (int s = check_paged_cache(op, to)) return s;
    INFERNT_REQUIRE(from->num_kv_heads == to->num_kv_heads && from->page_size == to->page_size &&
                        from->head_dim == to->head_dim && from->dtype == to->dtype,
                    "%s: pools of %d x %d x %d (type %d) into %d x %d x %d (type %d)", op, from->num_kv_heads,
                    from->page_size, from->head_dim, from->dtype, to->num_kv_heads, to->page_size, to->head_dim, to->dtype);
    INFERNT_REQUIRE(n >= 0 && (n == 0 || (src && dst)), "%s: %d pages, null list", op, n);
    for (const void* p : {static_cast<const void*>(src), static_cast<const void*>(dst), static_cast<const void*>(err)})
        INFERNT_REQUIRE(reinterpret_cast<uintptr_t>(p) % 4 == 0, "%s: misaligned list or err", op);
    const long long page_words = (long long)from->num_kv_heads * from->page_size * (from->head_dim / 8);
    INFERNT_REQUIRE(page_words < (1ll << 30), "%s: pages of %lld rows", op, page_words / (from->head_dim / 8));
    if (n == 0) return INFERNT_OK;
    if (int s = check_device_pointer(op, "the 4-bit K pool", from->k)) return s;
    if (int s = check_device_pointer(op, "the 4-bit V pool", from->v)) return s;
    if (int s = check_device_pointer(op, "the scales", from->scales)) return s;
    if (int s = check_device_pointer(op, "the K pool", to->k)) return s;
    if (int s = check_device_pointer(op, "the V pool", to->v)) return s;
    if (int s = check_device_pointer(op, "src", src)) return s;
    if (int s = check_device_pointer(op, "dst", dst)) return s;
    if (int s = check_device_pointer(op, "err", err)) return s;
    UnpackArgs a;
    a.k4 = static_cast<const uint32_t*>(from->k);
    a.v4 = static_cast<const uint32_t*>(from->v);
    a.scales = from->scales;
    a.k = static_cast<uint4*>(to->k);
    a.v = static_cast<uint4*>(to->v);
    a.src = src;
    a.dst = dst;
    a.page_words = (int)page_words;
    a.n = n;
    a.pages_in = from->num_pages;
    a.pages_out = to->num_pages;
    a.log_row = from->head_dim == 64 ? 3 : 4;
    a.err = err;
    const int per = kUnpackThreads * kUnpackAtOnce;
    const int x = (int)((page_words + per - 1) / per < 64 ? (page_words + per - 1) / per : 64);
    const dim3 grid(x, n < 65535 ? n : 65535);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (from->dtype == INFERNT_DTYPE_BF16)
        paged4_unpack<__nv_bfloat16><<<grid, kUnpackThreads, 0, st>>>(a);
    else
        paged4_unpack<__half><<<grid, kUnpackThreads, 0, st>>>(a);
    INFERNT_CUDA_TRY(cudaGetLastError());
    return INFERNT_OK;
}
