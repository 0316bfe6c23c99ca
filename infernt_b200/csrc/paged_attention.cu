// paged_attention.cu — attention of the new tokens of a ragged batch over
// paged KV caches, causal, with an optional sliding window and first tokens
// that stay visible (cuda/attention.cu:9-42 and cuda/softmax.cu:13-48 are one
// token of one sequence over a contiguous cache).
//
// For the token at position pos of a sequence and the query head h,
//   s_p = scale q . K[p],  m = max s_p,  l = sum e^(s_p - m),
//   out = sum e^(s_p - m) V[p] / l,  lse = m + ln l
// over the p that it sees: p <= pos and (p > pos - window or p < sinks).
// One pass over the keys with a running (m, l, out), in base 2.
//
// The query rows of a KV head are its new tokens times its G query heads,
// row = token G + head of the group, so all rows of a tile share the K and V
// rows that the tile reads, whatever G is.
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "paged_attention.cuh"
#include "warp_mma.cuh"

namespace infernt {
namespace {

constexpr int kTileKeys = 64;   // keys of a K / V tile
constexpr int kItemRows = 64;   // query rows of an item: four warps of 16
constexpr int kThreads = 128;
constexpr int kStages = 3;

template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                                         uint32_t b1) {
    mma_bf16_16816(c, a, b0, b1);
}
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Shared memory: the ring of K / V tiles (reused for the merge of the warps'
// results), the pool rows of two tiles, and a flag per query row.
template <int D>
struct Layout {
    static constexpr int kRowBytes = D * 2;
    static constexpr int kTileBytes = kTileKeys * kRowBytes;
    static constexpr int kRing = kStages * 2 * kTileBytes;
    static constexpr int kBytes = kRing + 2 * kTileKeys * 4 + kItemRows;
};

// The tiles [j0, j1) of an item by four warps: RB blocks of 16 rows, each by
// 4 / RB warps that share a tile's keys between them.  Leaves every warp's
// (m, l, out) of its rows in shared memory: slot (key share, row) of
// `m_s`, `l_s` and `o_s`.
template <typename T, int D, int RB>
__device__ __forceinline__ void run_tiles(const AttnArgs& a, const PagedSeq& seq, int s, const Item& it, int j0,
                                          int j1, unsigned char* smem) {
    using L = Layout<D>;
    constexpr int KS = 4 / RB, WK = kTileKeys / KS, NT = WK / 8;  // key shares, keys and n-tiles per warp
    constexpr int CH = L::kRowBytes / 16, KC = D / 16, DB = D / 8;
    constexpr int ROWS_PER_PASS = kThreads / CH, PASSES = kTileKeys / ROWS_PER_PASS;
    int* rows_s = reinterpret_cast<int*>(smem + L::kRing);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tig = lane & 3;
    const int rb = warp % RB, ks = warp / RB;
    const uint32_t ring = smem_addr(smem);
    const unsigned char* kb = static_cast<const unsigned char*>(a.k);
    const unsigned char* vb = static_cast<const unsigned char*>(a.v);

    // pool row of key `tid` of tile j; -1 where no row of the item sees it
    auto row_of = [&](int j) {
        if (tid >= kTileKeys || j >= j1) return -1;
        const int p = tile_key<kTileKeys>(it, j) + tid;
        return item_sees(it, p) ? pool_row(a.b, s, it.kvh, p, a.err) : -1;
    };
    // tile j into stage (j - j0) % kStages; rows that nobody sees become zeros
    auto issue = [&](int j) {
        if (j < j1) {
            const uint32_t st = ring + (uint32_t)((j - j0) % kStages) * 2 * L::kTileBytes;
            const int* rows = rows_s + (j & 1) * kTileKeys;
#pragma unroll
            for (int e = 0; e < PASSES; ++e) {
                const int row = e * ROWS_PER_PASS + tid / CH, ch = tid % CH;
                const int pr = rows[row];
                const size_t off = (size_t)(pr < 0 ? 0 : pr) * L::kRowBytes + ch * 16;
                const uint32_t dst = st + (uint32_t)(row * L::kRowBytes + ((ch ^ (row & 7)) << 4));
                cp_async16(dst, kb + off, pr < 0 ? 0u : 16u);
                cp_async16(dst + L::kTileBytes, vb + off, pr < 0 ? 0u : 16u);
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
        if (tid < kTileKeys) rows_s[((j0 + i) & 1) * kTileKeys + tid] = row_of(j0 + i);
        __syncthreads();
        issue(j0 + i);
    }
    if (tid < kTileKeys) {
        const int r = row_of(j0 + kStages - 1);
        rows_s[((j0 + kStages - 1) & 1) * kTileKeys + tid] = r;  // its slot was read two issues ago
    }

    // query fragments of rows g and g + 8 of the warp's block
    uint32_t qa[KC][4];
    int pos[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = rb * 16 + g + 8 * h, row = it.row0 + r, token = a.by_g(row);
        const bool ok = r < it.rows;
        pos[h] = ok ? row_pos(seq, token) : -1;
        const uint32_t* q = reinterpret_cast<const uint32_t*>(
            static_cast<const uint16_t*>(a.q) + (ok ? (long long)(seq.row0 + token) * a.ldq +
                                                          (long long)(it.kvh * a.G + row - token * a.G) * D + 2 * tig
                                                    : 0));
#pragma unroll
        for (int k = 0; k < KC; ++k) {
            qa[k][h] = ok ? q[8 * k] : 0u;
            qa[k][h + 2] = ok ? q[8 * k + 4] : 0u;
        }
    }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    float acc[DB][4];
#pragma unroll
    for (int b = 0; b < DB; ++b) acc[b][0] = acc[b][1] = acc[b][2] = acc[b][3] = 0.0f;
    const bool busy = rb * 16 < it.rows;

    for (int j = j0; j < j1; ++j) {
        cp_async_wait<kStages - 2>();  // this thread's copies of tile j have landed
        __syncthreads();               // everyone's, the rows of tile j + 2 too; tile j - 1's stage is free
        issue(j + kStages - 1);
        const int next = row_of(j + kStages);
        if (busy) {
            const int k0 = tile_key<kTileKeys>(it, j);
            const uint32_t kt = ring + (uint32_t)((j - j0) % kStages) * 2 * L::kTileBytes, vt = kt + L::kTileBytes;
            float sc[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.0f;
#pragma unroll
            for (int k = 0; k < KC; ++k)
#pragma unroll
                for (int n = 0; n < NT / 2; ++n) {
                    const int x = lane >> 3, row = ks * WK + 8 * (2 * n + (x >> 1)) + (lane & 7), ch = 2 * k + (x & 1);
                    uint32_t b0, b1, b2, b3;
                    ldsm_x4(kt + (uint32_t)(row * L::kRowBytes + ((ch ^ (row & 7)) << 4)), b0, b1, b2, b3);
                    mma_16816<T>(sc[2 * n], qa[k], b0, b1);
                    mma_16816<T>(sc[2 * n + 1], qa[k], b2, b3);
                }
            // a tile that every row sees whole needs no mask
            const bool whole = k0 + kTileKeys - 1 <= it.pos_first &&
                               (a.window == 0 || k0 > it.pos_last - a.window || k0 + kTileKeys <= a.sinks);
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int h = e >> 1, p = k0 + ks * WK + 8 * n + 2 * tig + (e & 1);
                    const bool sees = whole || (p <= pos[h] && (a.window == 0 || p > pos[h] - a.window || p < a.sinks));
                    sc[n][e] = sees ? sc[n][e] * a.scale_log2 : -INFINITY;
                    mx[h] = fmaxf(mx[h], sc[n][e]);
                }
            bool grow = false;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
                grow |= mx[h] > m[h] + kRescale;
            }
            // the reference maximum moves only when probabilities would pass 2^8
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float n = fmaxf(m[h], mx[h]);
                    const float f = m[h] == -INFINITY ? 0.0f : ex2(m[h] - n);
                    m[h] = n;
                    l[h] *= f;
#pragma unroll
                    for (int b = 0; b < DB; ++b) {
                        acc[b][2 * h] *= f;
                        acc[b][2 * h + 1] *= f;
                    }
                }
            }
            const float ref[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sc[n][e] = ex2(sc[n][e] - ref[e >> 1]);
                    l[e >> 1] += sc[n][e];
                }
            // the score fragments of two n-tiles are the A fragment of 16 probabilities
#pragma unroll
            for (int kk = 0; kk < NT / 2; ++kk) {
                const uint32_t pa[4] = {Half16<T>::pack(sc[2 * kk][0], sc[2 * kk][1]),
                                        Half16<T>::pack(sc[2 * kk][2], sc[2 * kk][3]),
                                        Half16<T>::pack(sc[2 * kk + 1][0], sc[2 * kk + 1][1]),
                                        Half16<T>::pack(sc[2 * kk + 1][2], sc[2 * kk + 1][3])};
#pragma unroll
                for (int b = 0; b < DB / 2; ++b) {
                    const int x = lane >> 3, row = ks * WK + 16 * kk + 8 * (x & 1) + (lane & 7), ch = 2 * b + (x >> 1);
                    uint32_t v0, v1, v2, v3;
                    ldsm_x4_trans(vt + (uint32_t)(row * L::kRowBytes + ((ch ^ (row & 7)) << 4)), v0, v1, v2, v3);
                    mma_16816<T>(acc[2 * b], pa, v0, v1);
                    mma_16816<T>(acc[2 * b + 1], pa, v2, v3);
                }
            }
        }
        if (tid < kTileKeys) rows_s[((j + kStages) & 1) * kTileKeys + tid] = next;
    }
    cp_async_wait<0>();
    __syncthreads();  // the ring is free
    float* o_s = reinterpret_cast<float*>(smem);           // [KS][RB 16][D]
    float* m_s = o_s + 4 * 16 * D;                          // [KS][RB 16]
    float* l_s = m_s + 64;
    if (busy) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            const int slot = (ks * RB + rb) * 16 + g + 8 * h;
            if (tig == 0) {
                m_s[slot] = m[h];
                l_s[slot] = l[h];
            }
#pragma unroll
            for (int b = 0; b < DB; ++b)
                *reinterpret_cast<float2*>(o_s + slot * D + 8 * b + 2 * tig) =
                    make_float2(acc[b][2 * h], acc[b][2 * h + 1]);
        }
    }
    __syncthreads();
}

// `shares` sets of (m, l, out) in shared memory.
template <int D>
__device__ __forceinline__ Joined join_shares(const float* o_s, int shares, int r, int d) {
    const float* m_s = o_s + 64 * D;
    const float* l_s = m_s + 64;
    const int stride = 64 / shares;  // rows of one share
    Joined v = {-INFINITY, 0.0f, 0.0f, 0.0f};
    for (int k = 0; k < shares; ++k) v.m = fmaxf(v.m, m_s[k * stride + r]);
    for (int k = 0; k < shares; ++k) {
        const float mk = m_s[k * stride + r], f = mk == -INFINITY ? 0.0f : ex2(mk - v.m);
        const float2 o = *reinterpret_cast<const float2*>(o_s + (k * stride + r) * D + d);
        v.l = fmaf(l_s[k * stride + r], f, v.l);
        v.x = fmaf(o.x, f, v.x);
        v.y = fmaf(o.y, f, v.y);
    }
    return v;
}

template <int M, int D>
__device__ __forceinline__ Joined join_slots(const AttnArgs& a, int first, int last, int r, int d) {
    Joined v = {-INFINITY, 0.0f, 0.0f, 0.0f};
    for (int b = first; b <= last; ++b) v.m = fmaxf(v.m, __ldcg(slot_of<M, D>(a, b, first) + M * D + r));
    for (int b = first; b <= last; ++b) {
        const float* p = slot_of<M, D>(a, b, first);
        const float mk = __ldcg(p + M * D + r), f = mk == -INFINITY ? 0.0f : ex2(mk - v.m);
        const float2 o = __ldcg(reinterpret_cast<const float2*>(p + r * D + d));
        v.l = fmaf(__ldcg(p + M * D + M + r), f, v.l);
        v.x = fmaf(o.x, f, v.x);
        v.y = fmaf(o.y, f, v.y);
    }
    return v;
}

// Columns d and d + 1 of a row's result; true when it is not finite.
template <typename T, int D>
__device__ __forceinline__ bool write_pair(const AttnArgs& a, const PagedSeq& seq, int kvh, int row, int d, Joined v) {
    const int token = a.by_g(row), head = kvh * a.G + row - token * a.G;
    const bool sees = row_pos(seq, token) >= 0;
    const float inv = 1.0f / v.l;
    const float x = sees ? v.x * inv : 0.0f, y = sees ? v.y * inv : 0.0f;
    *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + (long long)(seq.row0 + token) * a.ldo +
                                 (long long)head * D + d) = Half16<T>::pack(x, y);
    if (a.lse && d == 0)
        a.lse[(long long)(seq.row0 + token) * a.nq + head] =
            sees ? (v.m + log2f(v.l)) * kLn2 : -INFINITY;
    return !(fabsf(x) < INFINITY && fabsf(y) < INFINITY);
}

// Counts this CTA's arrival at an item split over `parts` CTAs; true for the
// last one, which then sees the others' slots.
__device__ __forceinline__ bool last_to_arrive(unsigned* ticket, int parts) {
    __shared__ int s_last;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        s_last = atomicAdd(ticket, 1u) + 1u == (unsigned)parts;
        if (s_last) *ticket = 0u;  // ready for the next call
    }
    __syncthreads();
    __threadfence();
    return s_last != 0;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, D == 64 ? 4 : 2) paged_attn(const __grid_constant__ AttnArgs a) {
    using L = Layout<D>;
    constexpr int M = kItemRows;
    extern __shared__ __align__(128) unsigned char smem[];
    const int tid = threadIdx.x;
    float* o_s = reinterpret_cast<float*>(smem);
    unsigned char* flag = smem + L::kRing + 2 * kTileKeys * 4;
    const Place place = find_place<M, kTileKeys, kThreads>(a);
    if (place.s < 0) return;
    walk<M, kTileKeys>(a, place, [&](const PagedSeq& seq, const Item& it, const Part& p) {
        int shares;
        if (it.rows <= 16) {
            run_tiles<T, D, 1>(a, seq, p.s, it, p.j0, p.j1, smem);
            shares = 4;
        } else if (it.rows <= 32) {
            run_tiles<T, D, 2>(a, seq, p.s, it, p.j0, p.j1, smem);
            shares = 2;
        } else {
            run_tiles<T, D, 4>(a, seq, p.s, it, p.j0, p.j1, smem);
            shares = 1;
        }
        const bool split = p.first != p.last;
        if (split) {
            float* slot = slot_of<M, D>(a, blockIdx.x, p.first);
            for (int e = tid; e < it.rows * (D / 2); e += kThreads) {
                const int r = e / (D / 2), d = 2 * (e % (D / 2));
                const Joined v = join_shares<D>(o_s, shares, r, d);
                *reinterpret_cast<float2*>(slot + r * D + d) = make_float2(v.x, v.y);
                if (d == 0) {
                    slot[M * D + r] = v.m;
                    slot[M * D + M + r] = v.l;
                }
            }
        }
        if (!split || last_to_arrive(a.tickets + p.first, p.last - p.first + 1)) {
            if (tid < M) flag[tid] = 0;
            __syncthreads();
            for (int e = tid; e < it.rows * (D / 2); e += kThreads) {
                const int r = e / (D / 2), d = 2 * (e % (D / 2));
                const Joined v =
                    split ? join_slots<M, D>(a, p.first, p.last, r, d) : join_shares<D>(o_s, shares, r, d);
                if (write_pair<T, D>(a, seq, it.kvh, it.row0 + r, d, v)) flag[r] = 1;
            }
            __syncthreads();
            for (int r = tid >> 5; r < it.rows; r += kThreads / 32)
                if (flag[r]) exact_row<T, D>(a, seq, p.s, it.kvh, it.row0 + r);
        }
        __syncthreads();  // shared memory is free for the next item
    });
}

template <typename T, int D>
int launch(const AttnArgs& args, cudaStream_t st) {
    using L = Layout<D>;
    static_assert(4 * 16 * D * 4 + 2 * 64 * 4 <= L::kRing, "the merge must fit the ring");
    static_assert(kSlotsAt + 2 * kMaxCtas * slot_floats<kItemRows, D>() * 4 <= kWorkspaceBytes && kMaxCtas * 4 <= kSlotsAt,
                  "the slots must fit the workspace");
    AttnArgs a = args;
    INFERNT_CUDA_TRY(cudaFuncSetAttribute(paged_attn<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes));
    // as many CTAs as the SMs hold at once
    int ctas = sm_count() * (D == 64 ? 4 : 2);
    if (ctas > kMaxCtas) ctas = kMaxCtas;
    paged_attn<T, D><<<ctas, kThreads, L::kBytes, st>>>(a);
    INFERNT_CUDA_TRY(cudaGetLastError());
    return INFERNT_OK;
}

}  // namespace
}  // namespace infernt

extern "C" size_t infernt_paged_attention_workspace_bytes(void) { return infernt::kWorkspaceBytes; }

extern "C" int infernt_paged_attention(void* out, int ldo, const void* q, int ldq, int nq,
                                       const infernt_paged_cache* cache, const infernt_ragged_batch* batch, int window,
                                       int sinks, float scale, float* lse, void* workspace, unsigned* err,
                                       void* stream) {
    using namespace infernt;
    const char* op = "paged_attention";
    if (int s = check_paged_cache(op, cache)) return s;
    if (int s = check_ragged_batch(op, batch)) return s;
    INFERNT_REQUIRE(q && out && workspace, "%s: null pointer", op);
    const int D = cache->head_dim, nkv = cache->num_kv_heads;
    INFERNT_REQUIRE(nq >= 1 && nq % nkv == 0 && nq / nkv <= 128, "%s: %d query heads, %d KV heads", op, nq, nkv);
    INFERNT_REQUIRE(ldq >= (long long)nq * D && ldo >= (long long)nq * D && ldq % 8 == 0 && ldo % 8 == 0,
                    "%s: rows %d and %d apart for %d heads of %d (multiples of 8)", op, ldq, ldo, nq, D);
    INFERNT_REQUIRE(aligned16(q) && aligned16(out) && aligned16(workspace),
                    "%s: q, out and workspace must be 16-byte aligned", op);
    INFERNT_REQUIRE(window >= 0 && sinks >= 0 && (window > 0 || sinks == 0), "%s: window %d, sinks %d", op, window,
                    sinks);
    INFERNT_REQUIRE(std::isfinite(scale) && scale >= 0.0f, "%s: scale %g", op, scale);
    const int G = nq / nkv;
    INFERNT_REQUIRE((long long)batch->num_rows * G < kMaxPositions, "%s: %d rows of %d heads", op, batch->num_rows, nq);
    // the units of the schedule are counted in 32 bits
    const long long most_kv = std::min<long long>((long long)batch->table_stride * cache->page_size, kMaxPositions);
    const bool chunks = paged_attention_tc_pages(cache->page_size) && (long long)batch->max_q_len * G > kItemRows;
    const long long tile_m = chunks ? kTcItemRows : kItemRows, tile_n = chunks ? kTcTileKeys : kTileKeys;
    INFERNT_REQUIRE(((long long)batch->num_rows * G / tile_m + batch->num_seqs) * nkv < (1ll << 30) / (most_kv / tile_n + 2),
                    "%s: %d rows of %d heads over up to %lld positions (split the call)", op, batch->num_rows, nq,
                    most_kv);
    if (batch->num_seqs == 0 || batch->num_rows == 0) return INFERNT_OK;
    if (int s = check_device_pointer(op, "the cache", cache->k)) return s;
    if (int s = check_device_pointer(op, "q", q)) return s;
    if (int s = check_device_pointer(op, "out", out)) return s;
    AttnArgs a;
    a.b = paged_batch(*cache, *batch);
    a.q = q;
    a.out = out;
    a.k = cache->k;
    a.v = cache->v;
    a.lse = lse;
    a.ldq = ldq;
    a.ldo = ldo;
    a.nq = nq;
    a.G = G;
    a.by_g = fast_div(a.G);
    a.window = window < kMaxPositions ? window : kMaxPositions;
    a.sinks = sinks;
    a.scale = scale != 0.0f ? scale : 1.0f / std::sqrt((float)D);
    a.scale_log2 = a.scale * 1.4426950408889634f;
    a.min_tiles = 4;
    a.tickets = static_cast<unsigned*>(workspace);
    a.slots = reinterpret_cast<float*>(static_cast<char*>(workspace) + kSlotsAt);
    a.err = err;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (chunks) return paged_attention_tc(a, D, cache->dtype, st);
    if (cache->dtype == INFERNT_DTYPE_BF16)
        return D == 64 ? launch<__nv_bfloat16, 64>(a, st) : launch<__nv_bfloat16, 128>(a, st);
    return D == 64 ? launch<__half, 64>(a, st) : launch<__half, 128>(a, st);
}
