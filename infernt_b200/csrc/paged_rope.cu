// paged_rope.cu — rotary positions of a ragged batch of new tokens and the
// append of their K and V rows into pages (cuda/rope.cu:13-34 and
// cuda/kv_cache.cu:4-14 are one token of one sequence, split-half, unscaled).
//
//   (x, y) -> m (x cos a - y sin a, y cos a + x sin a),  a = p f_i
//
// for the pairs of the rotated part of each q and k head.  Positions run to
// 10^5 and more, where an FP32 product p f_i is off by 10^-2 radians, so
// f_i / 2 pi is held in 64 bits: p f_i / 2 pi mod 1 is exact to about 2^-36
// at p = 2^17 and enters the FP32 sine and cosine as a fraction of a turn.
#include <cmath>
#include <cstdint>

#include "paged_rope.cuh"

namespace infernt {

int check_paged_cache(const char* op, const infernt_paged_cache* c) {
    INFERNT_REQUIRE(c && c->k && c->v, "%s: null cache", op);
    INFERNT_REQUIRE(c->num_pages >= 1 && c->num_kv_heads >= 1 && c->page_size >= 1,
                    "%s: %d pages of %d positions, %d KV heads", op, c->num_pages, c->page_size, c->num_kv_heads);
    // page rows are counted in 32 bits, bytes in 64
    INFERNT_REQUIRE((long long)c->num_kv_heads * c->page_size < (1ll << 31) &&
                        (long long)c->num_pages * ((long long)c->num_kv_heads * c->page_size) < (1ll << 31),
                    "%s: a pool of 2^31 rows or more", op);
    INFERNT_REQUIRE(c->head_dim == 64 || c->head_dim == 128, "%s: head_dim %d (64 or 128)", op, c->head_dim);
    INFERNT_REQUIRE(c->dtype == INFERNT_DTYPE_BF16 || c->dtype == INFERNT_DTYPE_F16, "%s: cache type %d (bf16 or fp16)",
                    op, c->dtype);
    INFERNT_REQUIRE(aligned16(c->k) && aligned16(c->v), "%s: pools not 16-byte aligned", op);
    return INFERNT_OK;
}

int check_ragged_batch(const char* op, const infernt_ragged_batch* b) {
    INFERNT_REQUIRE(b, "%s: null batch", op);
    INFERNT_REQUIRE(b->num_seqs >= 0 && b->num_seqs <= 65535 && b->num_rows >= 0 && b->num_rows < kMaxPositions &&
                        b->max_q_len >= 0 && b->table_stride >= 0,
                    "%s: %d sequences, %d rows, at most %d new tokens, table rows of %d", op, b->num_seqs, b->num_rows,
                    b->max_q_len, b->table_stride);
    INFERNT_REQUIRE(b->num_seqs == 0 || (b->q_start && b->kv_len && (b->block_table || b->table_stride == 0)),
                    "%s: null batch array", op);
    for (const int* p : {b->q_start, b->kv_len, b->block_table})
        INFERNT_REQUIRE(reinterpret_cast<uintptr_t>(p) % sizeof(int) == 0, "%s: misaligned batch array", op);
    return INFERNT_OK;
}

int check_device_pointer(const char* op, const char* what, const void* p) {
    if (!p) return INFERNT_OK;
    cudaPointerAttributes at;
    INFERNT_CUDA_TRY(cudaPointerGetAttributes(&at, p));
    INFERNT_REQUIRE(at.type == cudaMemoryTypeManaged ||
                        (at.type == cudaMemoryTypeDevice && at.device == current_device()),
                    "%s: %s is not memory of the current device", op, what);
    return INFERNT_OK;
}

int check_batch_pointers(const char* op, const infernt_paged_cache* c, const infernt_ragged_batch* b, const void* err) {
    if (int s = check_device_pointer(op, "the K pool", c->k)) return s;
    if (int s = check_device_pointer(op, "the V pool", c->v)) return s;
    if (int s = check_device_pointer(op, "q_start", b->q_start)) return s;
    if (int s = check_device_pointer(op, "kv_len", b->kv_len)) return s;
    if (int s = check_device_pointer(op, "block_table", b->block_table)) return s;
    return check_device_pointer(op, "err", err);
}

int rope_frequencies(const char* op, const infernt_rope_params& p, int head_dim, RopeDev* out) {
    const int R = p.rotary_dim;
    INFERNT_REQUIRE(R >= 2 && R <= head_dim && R % 2 == 0, "%s: rotary_dim %d of %d", op, R, head_dim);
    INFERNT_REQUIRE(std::isfinite(p.theta) && p.theta > 0, "%s: theta %g", op, p.theta);
    INFERNT_REQUIRE(p.scaling >= INFERNT_ROPE_NONE && p.scaling <= INFERNT_ROPE_YARN, "%s: scaling %d", op,
                    p.scaling);
    INFERNT_REQUIRE(p.scaling == INFERNT_ROPE_NONE || (std::isfinite(p.factor) && p.factor > 0),
                    "%s: factor %g", op, p.factor);
    if (p.scaling == INFERNT_ROPE_LLAMA3 || p.scaling == INFERNT_ROPE_YARN)
        INFERNT_REQUIRE(p.original_max_len >= 1 && std::isfinite(p.low) && std::isfinite(p.high) && p.low > 0 &&
                            p.high > p.low,
                        "%s: original_max_len %d, low %g, high %g", op, p.original_max_len, p.low, p.high);
    INFERNT_REQUIRE(p.scaling != INFERNT_ROPE_YARN || p.theta > 1.0, "%s: YaRN needs theta above 1", op);
    const double two_pi = 6.283185307179586476925;
    double lo = 0, hi = 0;
    out->half = R / 2;
    out->interleaved = p.interleaved != 0;
    out->magnitude64 = 1.0;
    if (p.scaling == INFERNT_ROPE_YARN) {
        // the pair index at which a pair makes t turns over the original context
        auto border = [&](double t) {
            return R * std::log(p.original_max_len / (t * two_pi)) / (2 * std::log(p.theta));
        };
        lo = std::fmax(0.0, std::floor(border(p.high)));
        hi = std::fmin(R - 1.0, std::ceil(border(p.low)));
        // a factor up to 1 stretches nothing, and its logarithm would shrink or flip q and k
        out->magnitude64 = p.factor > 1.0 ? 0.1 * std::log(p.factor) + 1.0 : 1.0;
    }
    // f_i by repeated products: 64 of them are off by 64 x 2^-53; divisions
    // stay out of the loop, which runs at each call
    const double ratio = std::pow(p.theta, -2.0 / R), turns = 1.0 / two_pi;
    const double shrink = p.scaling == INFERNT_ROPE_NONE ? 1.0 : 1.0 / p.factor, llama3 = 1.0 / (p.high - p.low),
                 yarn = 1.0 / std::fmax(hi - lo, 0.001);
    double f = 1.0;
    for (int i = 0; i < R / 2; ++i, f *= ratio) {
        double g = f, keep = 1.0;  // share of f, the rest is f / factor
        if (p.scaling == INFERNT_ROPE_LINEAR) keep = 0.0;
        if (p.scaling == INFERNT_ROPE_LLAMA3)
            keep = (p.original_max_len * f * turns - p.low) * llama3;
        if (p.scaling == INFERNT_ROPE_YARN) keep = 1.0 - (i - lo) * yarn;
        keep = std::fmin(1.0, std::fmax(0.0, keep));
        if (p.scaling != INFERNT_ROPE_NONE) g = f * keep + f * shrink * (1.0 - keep);
        out->turns[i] = g * turns;
    }
    out->magnitude = (float)out->magnitude64;
    return INFERNT_OK;
}

int rope_append_args(const char* op, void* q_out, int ldo, const void* q, int ldq, int nq, const void* k, int ldk,
                     const void* v, int ldv, int src_dtype, int nkv, int head_dim, int dtype,
                     const infernt_ragged_batch* batch, const infernt_rope_params* rope, const unsigned* err,
                     RopeArgs* a, RopeDev* d, bool* empty) {
    INFERNT_REQUIRE(rope, "%s: null rope parameters", op);
    INFERNT_REQUIRE((q != nullptr) == (q_out != nullptr) && (k != nullptr) == (v != nullptr) && (q || k),
                    "%s: q with q_out, k with v", op);
    INFERNT_REQUIRE(src_dtype == INFERNT_DTYPE_F32 || src_dtype == INFERNT_DTYPE_BF16 || src_dtype == INFERNT_DTYPE_F16,
                    "%s: source type %d", op, src_dtype);
    const long long kvd = (long long)nkv * head_dim;
    INFERNT_REQUIRE(!q || (nq >= 1 && ldq >= (long long)nq * head_dim && ldo >= (long long)nq * head_dim),
                    "%s: %d query heads, rows %d and %d apart", op, nq, ldq, ldo);
    INFERNT_REQUIRE(!k || (ldk >= kvd && ldv >= kvd), "%s: k and v rows %d and %d apart for %lld values", op, ldk, ldv,
                    kvd);
    INFERNT_REQUIRE(!q || q != q_out || (src_dtype == dtype && ldq == ldo),
                    "%s: q_out may be q only with its type and row stride", op);
    const unsigned esize = src_dtype == INFERNT_DTYPE_F32 ? 4u : 2u;
    for (const void* p : {q, k, v})
        INFERNT_REQUIRE(reinterpret_cast<uintptr_t>(p) % esize == 0, "%s: misaligned source", op);
    INFERNT_REQUIRE(reinterpret_cast<uintptr_t>(q_out) % 2 == 0 && reinterpret_cast<uintptr_t>(err) % 4 == 0,
                    "%s: misaligned q_out or err", op);
    if (int s = rope_frequencies(op, *rope, head_dim, d)) return s;
    *empty = batch->num_seqs == 0 || batch->num_rows == 0;
    if (*empty) return INFERNT_OK;
    if (int s = check_device_pointer(op, "q", q)) return s;
    if (int s = check_device_pointer(op, "q_out", q_out)) return s;
    if (int s = check_device_pointer(op, "k", k)) return s;
    if (int s = check_device_pointer(op, "v", v)) return s;
    *a = {};
    a->q = q;
    a->k = k;
    a->v = v;
    a->q_out = q_out;
    a->ldq = ldq;
    a->ldk = ldk;
    a->ldv = ldv;
    a->ldo = ldo;
    a->nq = q ? nq : 0;
    a->D = head_dim;
    return INFERNT_OK;
}

namespace {

// A block per token row; for rotary_dim a multiple of 16 and rows that allow
// 16-byte loads.  The unit of work is two blocks of eight values, D / 16 to a
// head: of the rotated part, block w of its first half and of its second
// (which hold whole pairs in either layout), of the rest likewise.  The
// block's threads are a multiple of D / 16, so a thread keeps its w, and with
// it 8 cosines and sines in registers, for all heads.  A thread's first units
// are loaded before the row's position is known, which takes three dependent
// loads.  HBM-bound for chunks (8192 tokens of 32/8 heads of 128, bf16: 37 us,
// 5.5 TB/s; 121 us value by value), latency-bound for single tokens.
constexpr int kAhead = 3;

template <typename S, typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(kRopeThreads)
    paged_rope_wide(const RopeArgs a, const __grid_constant__ RopeDev rope) {
    __shared__ float2 cs_s[kMaxPairs];
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
    Eight<S> x[kAhead], y[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
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
    if (tid < rope.half) cs_s[tid] = turn_of(rope, tid, pos);
    __syncthreads();
    // of pair e of the first block; interleaved, the first block has four pairs, then the second's
    float2 cs[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
        cs[e] = !turns ? make_float2(1.0f, 0.0f)
                       : cs_s[!INTERLEAVED ? 8 * w + e : e < 4 ? 4 * w + e : rope.half / 2 + 4 * w + e - 4];
    auto finish = [&](int h, const Eight<S>& ex, const Eight<S>& ey) {
        float u[8], v[8];
        to_floats(ex, u);
        to_floats(ey, v);
        if (h < heads_q + nkv) {
            if (INTERLEAVED) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float u0 = u[2 * e], u1 = u[2 * e + 1], v0 = v[2 * e], v1 = v[2 * e + 1];
                    u[2 * e] = u0 * cs[e].x - u1 * cs[e].y;
                    u[2 * e + 1] = u1 * cs[e].x + u0 * cs[e].y;
                    v[2 * e] = v0 * cs[4 + e].x - v1 * cs[4 + e].y;
                    v[2 * e + 1] = v1 * cs[4 + e].x + v0 * cs[4 + e].y;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float u0 = u[e], v0 = v[e];
                    u[e] = u0 * cs[e].x - v0 * cs[e].y;
                    v[e] = v0 * cs[e].x + u0 * cs[e].y;
                }
            }
        }
        T* dst;
        int at = lo, to = hi;
        if (h < heads_q) {
            dst = static_cast<T*>(a.q_out) + r * a.ldo + (long long)h * D;
        } else {
            if (row < 0) return;
            const int kh = h - heads_q;
            const bool is_v = kh >= nkv;
            dst = static_cast<T*>(is_v ? a.vp : a.kp) + (row + (long long)(is_v ? kh - nkv : kh) * a.b.page_size) * D;
            if (is_v) {
                at = 8 * w;
                to = D / 2 + 8 * w;
            }
        }
        store_eight(dst + at, u);
        store_eight(dst + to, v);
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
        if (h0 + i * step < heads) finish(h0 + i * step, x[i], y[i]);
    for (int h = h0 + kAhead * step; h < heads; h += step) {
        const S* p = source(h);
        const bool is_v = h >= heads_q + nkv;
        finish(h, load_eight(p + (is_v ? 8 * w : lo)), load_eight(p + (is_v ? D / 2 + 8 * w : hi)));
    }
    check_sequences(a);
}

// Any other rotary_dim, stride or alignment: a block per token row, value by
// value.
template <typename S, typename T>
__global__ void __launch_bounds__(kRopeThreads) paged_rope(const RopeArgs a, const __grid_constant__ RopeDev rope) {
    __shared__ float2 cs[kMaxPairs];
    const int r = blockIdx.x, tid = threadIdx.x, D = a.D, half = rope.half, nkv = a.b.nkv;
    int pos;
    long long row;
    if (!place_row(a, r, pos, row)) {
        check_sequences(a);
        return;
    }
    if (tid < half) cs[tid] = turn_of(rope, tid, pos);
    __syncthreads();
    const int heads = (a.q ? a.nq : 0) + (row >= 0 ? nkv : 0), h0 = a.q ? 0 : a.nq;
    auto src_of = [&](int h) {
        return h < a.nq ? static_cast<const S*>(a.q) + r * a.ldq + (long long)h * D
                        : static_cast<const S*>(a.k) + r * a.ldk + (long long)(h - a.nq) * D;
    };
    auto dst_of = [&](int h) {
        return h < a.nq ? static_cast<T*>(a.q_out) + r * a.ldo + (long long)h * D
                        : static_cast<T*>(a.kp) + (row + (long long)(h - a.nq) * a.b.page_size) * D;
    };
    for (int u = tid; u < heads * half; u += kRopeThreads) {
        const int h = h0 + u / half, p = u % half;
        const int e0 = rope.interleaved ? 2 * p : p, e1 = rope.interleaved ? 2 * p + 1 : p + half;
        const S* src = src_of(h);
        T* dst = dst_of(h);
        const float x = source_value(src + e0), y = source_value(src + e1);
        dst[e0] = Half16<T>::round(x * cs[p].x - y * cs[p].y);
        dst[e1] = Half16<T>::round(y * cs[p].x + x * cs[p].y);
    }
    const int rest = D - 2 * half;
    for (int u = tid; u < heads * rest; u += kRopeThreads) {
        const int h = h0 + u / rest, e = 2 * half + u % rest;
        dst_of(h)[e] = Half16<T>::round(source_value(src_of(h) + e));
    }
    if (row >= 0)
        for (int u = tid; u < nkv * D; u += kRopeThreads) {
            const int h = u / D, e = u % D;
            static_cast<T*>(a.vp)[(row + (long long)h * a.b.page_size) * D + e] =
                Half16<T>::round(source_value(static_cast<const S*>(a.v) + r * a.ldv + u));
        }
    check_sequences(a);
}

template <typename S, typename T>
int launch(const RopeArgs& a, const RopeDev& d, cudaStream_t st) {
    // rows of S or T `ld` apart that start where 16 bytes may be loaded
    auto wide = [](const void* p, long long ld, size_t size) { return !p || (aligned16(p) && ld * size % 16 == 0); };
    if (d.half % 8 == 0 && wide(a.q, a.ldq, sizeof(S)) && wide(a.k, a.ldk, sizeof(S)) && wide(a.v, a.ldv, sizeof(S)) &&
        wide(a.q_out, a.ldo, sizeof(T))) {
        if (d.interleaved)
            paged_rope_wide<S, T, true><<<a.b.num_rows, kRopeThreads, 0, st>>>(a, d);
        else
            paged_rope_wide<S, T, false><<<a.b.num_rows, kRopeThreads, 0, st>>>(a, d);
    } else {
        paged_rope<S, T><<<a.b.num_rows, kRopeThreads, 0, st>>>(a, d);
    }
    INFERNT_CUDA_TRY(cudaGetLastError());
    return INFERNT_OK;
}

template <typename T>
int launch_src(const RopeArgs& a, const RopeDev& d, int src, cudaStream_t st) {
    if (src == INFERNT_DTYPE_F32) return launch<float, T>(a, d, st);
    if (src == INFERNT_DTYPE_BF16) return launch<__nv_bfloat16, T>(a, d, st);
    return launch<__half, T>(a, d, st);
}

}  // namespace
}  // namespace infernt

extern "C" int infernt_paged_rope_append(void* q_out, int ldo, const void* q, int ldq, int nq, const void* k, int ldk,
                                         const void* v, int ldv, int src_dtype, const infernt_paged_cache* cache,
                                         const infernt_ragged_batch* batch, const infernt_rope_params* rope,
                                         unsigned* err, void* stream) {
    using namespace infernt;
    const char* op = "paged_rope_append";
    if (int s = check_paged_cache(op, cache)) return s;
    if (int s = check_ragged_batch(op, batch)) return s;
    RopeArgs a;
    RopeDev d;
    bool empty;
    if (int s = rope_append_args(op, q_out, ldo, q, ldq, nq, k, ldk, v, ldv, src_dtype, cache->num_kv_heads,
                                 cache->head_dim, cache->dtype, batch, rope, err, &a, &d, &empty))
        return s;
    if (empty) return INFERNT_OK;
    if (int s = check_batch_pointers(op, cache, batch, err)) return s;
    a.b = paged_batch(*cache, *batch);
    a.kp = cache->k;
    a.vp = cache->v;
    a.err = err;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return cache->dtype == INFERNT_DTYPE_BF16 ? launch_src<__nv_bfloat16>(a, d, src_dtype, st)
                                              : launch_src<__half>(a, d, src_dtype, st);
}
