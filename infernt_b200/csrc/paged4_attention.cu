// paged4_attention.cu — attention of few new tokens a sequence over pages of
// 4 bits (paged4.cuh has the format, paged_attention.cu the formulas; chunks
// go to the tcgen05 kernel of paged_attention_tc.cu).
//
// The cache is read at a quarter of the bytes, so the work a byte is four
// times that of the kernel for 16-bit pages, which takes as long for a tile as
// HBM does.  Three things make it less:
//   - keys are the M of the MMA, the query rows its N = 8: S^T = K Q^T and
//     O^T = V^T P^T.  The 16 rows of an m16n8k16 are all of use, where query
//     rows as M leave 12 of 16 empty for a group of four heads.
//   - codes go from shared memory to the A operand by a shift, a logic
//     operation and an exact subtraction for two of them: the operand is the
//     whole numbers c - z, the scale s of a key multiplies its scores (K) or
//     its probabilities (V), four values a thread for 16 keys.
//   - the contraction's order is free: a thread takes 32 neighbouring
//     elements of a K row (and the same ones of Q), so a row is a 16-byte load
//     without a shuffle; for V^T it takes D / 8 neighbouring elements of four
//     keys.  P^T comes out of the scores by a transposition of 8 x 8 blocks.
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "paged4.cuh"
#include "paged_attention.cuh"
#include "tc_mma.cuh"
#include "warp_mma.cuh"

namespace infernt {
namespace {

constexpr int kKeys = 128;     // keys of a tile: 16 a warp
constexpr int kWarps = 8;      // that consume
constexpr int kConsumers = 32 * kWarps;
constexpr int kThreads = kConsumers + 32;
constexpr int kMostRows = 64;  // query rows of a KV head from which on the tcgen05 kernel is faster
constexpr int kBulkPage = 16;  // pages from which on a page's rows are one bulk copy

// A weight 2^(s - m) s_V enters the products in 16 bits.  m follows s + log2
// s_V, so weights stay below 2^(kRescale + 1 + kUp) whatever V's scales are;
// fp16 has its normal numbers down to 2^-18 of a row's largest.
template <typename T>
constexpr float kUp = Half16<T>::kBf16 ? 0.0f : 4.0f;
// Scales below it (vectors of zeros have the least) do not lower m further:
// the sum of 2^(s - m) stays in FP32.
constexpr float kLeastLog = -40.0f;

// Shared memory: the ring, per stage K codes, V codes and scale words; then
// what the warps know of an item's rows, a set a warp.
template <int D, int RB>
struct Layout {
    static constexpr int kRows = 8 * RB;
    static constexpr uint32_t kCodes = kKeys * D / 2;
    static constexpr uint32_t kStage = 2 * kCodes + kKeys * 4;
    static constexpr int kPerSm = RB == 1 ? 2 : 1;  // CTAs of an SM
    static constexpr uint32_t kSet = kRows * (D + 2) * 4;
    // Q as the B operands of one n-tile stay in registers; of several, in shared memory
    static constexpr bool kSharedQ = RB > 1;
    static constexpr uint32_t kQ = kSharedQ ? RB * (D / 32) * 512 : 0;
    static constexpr uint32_t kRoom = 227 * 1024 / kPerSm - 3 * 1024;
    static constexpr int kFit = (int)((kRoom - kWarps * kSet - kQ) / kStage);
    static constexpr int kStages = kFit < 8 ? kFit : 8;
    static constexpr uint32_t kScratch = kStages * kStage;
    static constexpr uint32_t kQAt = kScratch + kWarps * kSet;
    static constexpr uint32_t kBytes = kQAt + kQ + 128;
    static_assert(kStages >= 3, "");
};

template <int ST>
struct Ring {
    uint64_t full[ST], empty[ST];
};

__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, uint32_t src_bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
__device__ __forceinline__ uint2 ld_shared2(uint32_t at) {
    uint2 w;
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w.x), "=r"(w.y) : "r"(at) : "memory");
    return w;
}
__device__ __forceinline__ uint32_t ld_shared1(uint32_t at) {
    uint32_t w;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(at) : "memory");
    return w;
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    if (Half16<T>::kBf16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The producer warp.  Of each tile the codes of the pages that some row sees
// (what lies in rows that none sees is a number whatever it is), and the scale
// words, 0 for keys that no row sees or whose page the pool does not have.
template <int D, int RB>
__device__ __forceinline__ void produce(const AttnArgs& a, const Place& place, uint32_t base,
                                        Ring<Layout<D, RB>::kStages>& ring, bool& ok) {
    using L = Layout<D, RB>;
    constexpr int ST = L::kStages, PER = kKeys / 32;
    constexpr uint32_t ROW = D / 2;
    const int lane = threadIdx.x & 31, ps = a.b.page_size;
    const char* kc = static_cast<const char*>(a.k);
    const char* vc = static_cast<const char*>(a.v);
    uint32_t st = 0, turn = 1;  // the first round's stages are free
    walk<L::kRows, kKeys>(a, place, [&](const PagedSeq&, const Item& it, const Part& part) {
        const int* table = a.b.table + (size_t)part.s * a.b.table_stride;
        // pool rows of keys lane, lane + 32, ... of tile j; -1: no row sees the key, or the pool does not have it
        auto look = [&](int j, int (&rows)[PER]) {
            const int k0 = tile_key<kKeys>(it, j);
#pragma unroll
            for (int h = 0; h < PER; ++h) {
                const int p = k0 + lane + 32 * h;
                rows[h] = item_sees(it, p) ? pool_row(a.b, part.s, it.kvh, p, a.err) : -1;
            }
        };
        int rows[PER];
        if (part.j0 < part.j1) look(part.j0, rows);
#pragma unroll 1
        for (int j = part.j0; j < part.j1; ++j) {
            const int k0 = tile_key<kKeys>(it, j);
            const uint32_t kt = base + st * L::kStage, vt = kt + L::kCodes, sct = vt + L::kCodes;
            // the runs of a page, a page a lane at a time
            const int pi0 = a.b.by_page(k0), pages = ps >= kBulkPage ? a.b.by_page(k0 + kKeys - 1) - pi0 + 1 : 0;
            int from = 0, count = 0, at = 0;
            if (lane < pages) {  // (at most 128 / 16 + 1)
                const int pi = pi0 + lane, p0 = max(k0, pi * ps);
                // up to the end of the page, the tile or the last key; (pi + 1) ps may pass 2^31 behind it
                const int p1 = min(min(k0 + kKeys, it.hi), p0 + (ps - (p0 - pi * ps)));
                if (p0 < p1 && (p1 > it.lo || p0 < it.sink_end)) {
                    const int page = table[pi];
                    if (page >= 0 && page < a.b.num_pages) {
                        from = (page * a.b.nkv + it.kvh) * ps + (p0 - pi * ps);
                        count = p1 - p0;
                        at = p0 - k0;
                    }
                }
            }
            const unsigned bytes = __reduce_add_sync(0xffffffffu, (unsigned)count) * 2 * ROW;
            int next[PER];
            if (j + 1 < part.j1) look(j + 1, next);
            tc_wait_bar(&ring.empty[st], turn, ok);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) return;
            if (lane == 0) mbar_arrive_expect_tx(&ring.full[st], bytes);
            __syncwarp();
            if (count > 0) {
                bulk_g2s_plain_at(kt + at * ROW, kc + (size_t)from * ROW, count * ROW, &ring.full[st]);
                bulk_g2s_plain_at(vt + at * ROW, vc + (size_t)from * ROW, count * ROW, &ring.full[st]);
            }
            if (ps < kBulkPage) {
                constexpr int CH = ROW / 16, RPI = 32 / CH;  // chunks of a row, rows at once
#pragma unroll
                for (int h = 0; h < PER; ++h)
#pragma unroll 4
                    for (int i = 0; i < 32 / RPI; ++i) {
                        const int r = i * RPI + lane / CH, ch = lane % CH;
                        const int pr = __shfl_sync(0xffffffffu, rows[h], r);
                        if (pr < 0) continue;
                        const size_t off = (size_t)pr * ROW + ch * 16;
                        cp_async16(kt + (r + 32 * h) * ROW + ch * 16, kc + off, 16u);
                        cp_async16(vt + (r + 32 * h) * ROW + ch * 16, vc + off, 16u);
                    }
            }
#pragma unroll
            for (int h = 0; h < PER; ++h) {
                cp_async4(sct + (lane + 32 * h) * 4, a.scales + max(rows[h], 0), rows[h] >= 0 ? 4u : 0u);
                rows[h] = next[h];
            }
            // this lane's arrival, once its copies have landed
            asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_addr(&ring.full[st])) : "memory");
            if (++st == ST) {
                st = 0;
                turn ^= 1;
            }
        }
    });
    cp_async_wait<0>();
}

// The physical key of row r of a warp's 16: neighbouring rows, and every
// second one, are of both parities, so that neither the 16-byte loads of K
// rows nor the loads of V rows (64 bytes of two keys are 32 banks) meet in a
// bank more often than their size asks for.
__device__ __forceinline__ int key_of(int r) { return r ^ ((r >> 1) & 1); }

// What a warp knows of the item's rows from its keys: of n-tile n the query
// rows 8 n + 2 tig and + 1, of their results the elements g D / 8 ... .
template <int D, int RB>
struct RowState {
    float m[RB][2], l[RB][2];
    float acc[RB][D / 16][4];
};

// The tiles [j0, j1) of an item, 16 keys of each by every warp.
template <typename T, int D, int RB>
__device__ __forceinline__ void consume(const AttnArgs& a, const PagedSeq& seq, const Item& it, const Part& part,
                                        uint32_t base, Ring<Layout<D, RB>::kStages>& ring, uint32_t& st, uint32_t& turn,
                                        RowState<D, RB>& s, bool& ok) {
    using L = Layout<D, RB>;
    constexpr int KC = D / 16, ST = L::kStages, W = D / 32;  // MMA steps of a score; words of a thread's K row
    constexpr uint32_t ROW = D / 2;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tig = lane & 3;
    // Q of row 8 n + g, elements tig D / 4 + 8 w ... as pairs in the order of Codes4
    auto q_of = [&](int n, int w) {
        const int row = it.row0 + min(8 * n + g, it.rows - 1), token = a.by_g(row);
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) +
                                                             (long long)(seq.row0 + token) * a.ldq +
                                                             (it.kvh * a.G + row - token * a.G) * D + tig * (D / 4)) + w);
        // (0, 1) (2, 3) (4, 5) (6, 7) -> (0, 4) (1, 5) (2, 6) (3, 7)
        return make_uint4(__byte_perm(x.x, x.z, 0x5410), __byte_perm(x.x, x.z, 0x7632), __byte_perm(x.y, x.w, 0x5410),
                          __byte_perm(x.y, x.w, 0x7632));
    };
    uint4 qb[L::kSharedQ ? 1 : W];
    const uint32_t q_at = base + L::kQAt + lane * 16;
    if (L::kSharedQ) {
        for (int x = warp; x < RB * W; x += kWarps) st_shared(q_at + x * 512, q_of(x / W, x % W));
        named_sync(1, kConsumers);
    } else {
#pragma unroll
        for (int w = 0; w < W; ++w) qb[L::kSharedQ ? 0 : w] = q_of(0, w);
    }
    int pos[RB][2];
#pragma unroll
    for (int n = 0; n < RB; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = 8 * n + 2 * tig + e;
            pos[n][e] = r < it.rows ? row_pos(seq, a.by_g(it.row0 + r)) : -1;
            s.m[n][e] = -INFINITY;
            s.l[n][e] = 0.0f;
        }
#pragma unroll
        for (int b = 0; b < KC; ++b) s.acc[n][b][0] = s.acc[n][b][1] = s.acc[n][b][2] = s.acc[n][b][3] = 0.0f;
    }
    const uint32_t k_at = (uint32_t)(warp * 16) * ROW;
#pragma unroll 1
    for (int j = part.j0; j < part.j1; ++j) {
        const int k0 = tile_key<kKeys>(it, j) + warp * 16;
        const uint32_t kt = base + st * L::kStage + k_at, vt = kt + L::kCodes;
        const uint32_t sct = base + st * L::kStage + 2 * L::kCodes + warp * 64;
        tc_wait_bar(&ring.full[st], turn, ok);
        // keys of this warp that some row sees
        if (k0 < it.hi && (k0 + 15 >= it.lo || k0 < it.sink_end)) {
            const uint32_t word[2] = {ld_shared1(sct + 4 * key_of(g)), ld_shared1(sct + 4 * key_of(g + 8))};
            float sc[RB][4];
#pragma unroll
            for (int n = 0; n < RB; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.0f;
            {
                uint32_t ka[2][4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t at = kt + key_of(g + 8 * h) * ROW + tig * (D / 8);
                    if (D == 128) {
                        const uint4 x = ld_shared(at);
                        ka[h][0] = x.x;
                        ka[h][1] = x.y;
                        ka[h][2] = x.z;
                        ka[h][3] = x.w;
                    } else {
                        const uint2 x = ld_shared2(at);
                        ka[h][0] = x.x;
                        ka[h][1] = x.y;
                    }
                }
                const uint32_t z0 = Codes4<T>::zeros(word[0] & 15u), z1 = Codes4<T>::zeros(word[1] & 15u);
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    uint32_t x[4], y[4];
                    whole4<T>(ka[0][w], z0, x);
                    whole4<T>(ka[1][w], z1, y);
#pragma unroll
                    for (int n = 0; n < RB; ++n)
                        if (RB == 1 || 8 * n < it.rows) {
                            const uint4 q = L::kSharedQ ? ld_shared(q_at + (n * W + w) * 512) : qb[L::kSharedQ ? 0 : w];
                            mma<T>(sc[n], x[0], y[0], x[1], y[1], q.x, q.y);
                            mma<T>(sc[n], x[2], y[2], x[3], y[3], q.z, q.w);
                        }
                }
            }
            // scores, weights; key h is key_of(g + 8 h)
            const bool whole = seen_whole<16>(a, it, k0);
            float ks[2], vs[2], vl[2];
            bool none[2];  // a V vector of NaN
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                ks[h] = scale4(word[h]) * a.scale_log2;
                const uint32_t v = word[h] >> 16;
                none[h] = (v & 0x7f80u) == 0x7f80u;
                vs[h] = none[h] ? 0.0f : scale4(v);
                vl[h] = fmaxf((float)(int)((v >> 7) & 255u) - 127.0f, kLeastLog) - kUp<T>;
                if (none[h]) vl[h] = -kUp<T>;
            }
            uint32_t pb[RB][2];
            bool grow = false;
            float mx[RB][2];
#pragma unroll
            for (int n = 0; n < RB; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float& x = sc[n][2 * h + e];
                        x *= ks[h];
                        if (!whole && !row_sees(a, pos[n][e], k0 + key_of(g + 8 * h))) x = -INFINITY;
                    }
                    mx[n][e] = fmaxf(sc[n][e] + vl[0], sc[n][2 + e] + vl[1]);
                    grow |= mx[n][e] > s.m[n][e] + kRescale;
                }
            // m moves only when weights would pass 2^(kRescale + kUp)
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int n = 0; n < RB; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1)
                            mx[n][e] = fmaxf(mx[n][e], __shfl_xor_sync(0xffffffffu, mx[n][e], o));
                        const float top = fmaxf(s.m[n][e], mx[n][e]);
                        const float f = s.m[n][e] == -INFINITY ? 0.0f : ex2(s.m[n][e] - top);
                        s.m[n][e] = top;
                        s.l[n][e] *= f;
#pragma unroll
                        for (int b = 0; b < KC; ++b) {
                            s.acc[n][b][e] *= f;
                            s.acc[n][b][2 + e] *= f;
                        }
                    }
            }
            // rows that see a V vector of NaN have no result
            if (__any_sync(0xffffffffu, none[0] || none[1])) {
#pragma unroll
                for (int n = 0; n < RB; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        bool hit = (none[0] && sc[n][e] != -INFINITY) || (none[1] && sc[n][2 + e] != -INFINITY);
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) hit |= __shfl_xor_sync(0xffffffffu, (int)hit, o) != 0;
                        if (hit)
#pragma unroll
                            for (int b = 0; b < KC; ++b) s.acc[n][b][e] = s.acc[n][b][2 + e] = __int_as_float(0x7fffffff);
                    }
            }
#pragma unroll
            for (int n = 0; n < RB; ++n) {
                float w[4];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float ref = s.m[n][e] == -INFINITY ? 0.0f : s.m[n][e];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float p = ex2(sc[n][2 * h + e] - ref);
                        s.l[n][e] += p;
                        w[2 * h + e] = p * vs[h];
                    }
                }
                pb[n][0] = transpose8(Half16<T>::pack(w[0], w[1]));
                pb[n][1] = transpose8(Half16<T>::pack(w[2], w[3]));
            }
            // V^T: elements g D / 8 ... of keys 2 tig, + 1 and 2 tig + 8, + 9
            uint32_t zv[2], va[4][D / 64];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = key_of(2 * tig + (i & 1) + 8 * (i >> 1));
                const uint32_t at = vt + key * ROW + g * (D / 16);
                if (D == 128) {
                    const uint2 x = ld_shared2(at);
                    va[i][0] = x.x;
                    va[i][D / 64 - 1] = x.y;
                } else {
                    va[i][0] = ld_shared1(at);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
                zv[h] = Codes4<T>::zeros((ld_shared1(sct + 4 * key_of(2 * tig + 8 * h)) >> 16) & 15u,
                                         (ld_shared1(sct + 4 * key_of(2 * tig + 1 + 8 * h)) >> 16) & 15u);
#pragma unroll
            for (int q = 0; q < D / 64; ++q)
#pragma unroll
                for (int half = 0; half < 2; ++half) {  // elements 8 q + 4 half ... + 3 of both keys of a pair
                    const uint32_t sel = half ? 0x7632 : 0x5410;
                    uint32_t x[4], y[4];
                    whole4<T>(__byte_perm(va[0][q], va[1][q], sel), zv[0], x);
                    whole4<T>(__byte_perm(va[2][q], va[3][q], sel), zv[1], y);
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int n = 0; n < RB; ++n)
                            if (RB == 1 || 8 * n < it.rows)
                                mma<T>(s.acc[n][4 * q + 2 * half + b], x[2 * b], x[2 * b + 1], y[2 * b], y[2 * b + 1],
                                       pb[n][0], pb[n][1]);
                }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&ring.empty[st]);
        if (++st == ST) {
            st = 0;
            turn ^= 1;
        }
    }
#pragma unroll
    for (int n = 0; n < RB; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) s.l[n][e] += __shfl_xor_sync(0xffffffffu, s.l[n][e], o);
}

// Element 4 i of the stretch g of a row's D in a set: neighbours g for the
// writers' 16-byte stores, neighbours i a stretch's four elements.
template <int D>
__device__ __forceinline__ int set_at(int row, int i, int g) {
    return row * D + i * 32 + g * 4;
}

template <typename T, int D, int RB>
__global__ void __launch_bounds__(kThreads, (Layout<D, RB>::kPerSm)) paged4_attn(const __grid_constant__ AttnArgs a) {
    using L = Layout<D, RB>;
    constexpr int M = L::kRows, ST = L::kStages;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ Ring<ST> ring;
    __shared__ int last_s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tig = lane & 3;
    const uint32_t base = (smem_addr(smem) + 127u) & ~127u;
    float* scratch = reinterpret_cast<float*>(smem + (base - smem_addr(smem)) + L::kScratch);
    if (tid == 0) {
        for (int i = 0; i < ST; ++i) {
            mbar_init(&ring.full[i], 33);
            mbar_init(&ring.empty[i], kWarps);
        }
        mbar_fence_init();
    }
    const Place place = find_place<M, kKeys, kThreads>(a);  // its barriers publish the set-up
    pdl_launch_dependents();  // the tcgen05 kernel may take SMs as they become free
    if (place.s < 0) return;
    bool ok = true;
    if (warp == kWarps) {
        produce<D, RB>(a, place, base, ring, ok);
    } else {
        uint32_t st = 0, turn = 0;
        walk<M, kKeys>(a, place, [&](const PagedSeq& seq, const Item& it, const Part& p) {
            {
                RowState<D, RB> s;
                consume<T, D, RB>(a, seq, it, p, base, ring, st, turn, s, ok);
                float* set = scratch + warp * (L::kSet / 4);
#pragma unroll
                for (int n = 0; n < RB; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int r = 8 * n + 2 * tig + e;
                        if (r >= it.rows) continue;
#pragma unroll
                        for (int i = 0; i < D / 32; ++i)
                            *reinterpret_cast<float4*>(set + set_at<D>(r, i, g)) =
                                make_float4(s.acc[n][2 * i][e], s.acc[n][2 * i][2 + e], s.acc[n][2 * i + 1][e],
                                            s.acc[n][2 * i + 1][2 + e]);
                        if (g == 0) {
                            set[M * D + r] = s.m[n][e];
                            set[M * D + M + r] = s.l[n][e];
                        }
                    }
            }
            named_sync(1, kConsumers);
            // the warps' results, joined in order: four elements of a row a thread
            const bool split = p.first != p.last;
            float* slot = slot_of<M, D>(a, blockIdx.x, p.first);
            for (int x = tid; x < it.rows * (D / 4); x += kConsumers) {
                const int r = x / (D / 4), i = x / 8 % (D / 32), gg = x % 8, d = gg * (D / 8) + 4 * i;
                float m[kWarps], top = -INFINITY, l = 0.0f;
                float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    m[w] = scratch[w * (L::kSet / 4) + M * D + r];
                    top = fmaxf(top, m[w]);
                }
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float* set = scratch + w * (L::kSet / 4);
                    const float f = m[w] == -INFINITY ? 0.0f : ex2(m[w] - top);
                    const float4 v = *reinterpret_cast<const float4*>(set + set_at<D>(r, i, gg));
                    l = fmaf(set[M * D + M + r], f, l);
                    o.x = fmaf(v.x, f, o.x);
                    o.y = fmaf(v.y, f, o.y);
                    o.z = fmaf(v.z, f, o.z);
                    o.w = fmaf(v.w, f, o.w);
                }
                if (split) {
                    *reinterpret_cast<float4*>(slot + r * D + d) = o;
                    if (d == 0) {
                        slot[M * D + r] = top;
                        slot[M * D + M + r] = l;
                    }
                } else {
                    write_pair<T, D>(a, seq, it.kvh, it.row0 + r, d, {top, l, o.x, o.y});
                    write_pair<T, D>(a, seq, it.kvh, it.row0 + r, d + 2, {top, l, o.z, o.w});
                }
            }
            named_sync(1, kConsumers);  // the sets are free
            if (!split) return;
            if (tid == 0) {
                // the others' writes, ordered before by the barrier, become visible with this thread's fence
                __threadfence();
                unsigned* ticket = a.tickets + p.first;
                last_s = atomicAdd(ticket, 1u) + 1u == (unsigned)(p.last - p.first + 1);
                if (last_s) *ticket = 0u;  // ready for the next call
                __threadfence();
            }
            named_sync(1, kConsumers);
            if (last_s) {
                // a warp a row, two columns a lane
                for (int r = warp; r < it.rows; r += kWarps)
#pragma unroll
                    for (int d = 2 * lane; d < D; d += 64)
                        write_pair<T, D>(a, seq, it.kvh, it.row0 + r, d, join_slots<M, D>(a, p.first, p.last, r, d));
            }
            named_sync(1, kConsumers);  // everyone has read last_s
        });
    }
    if (!ok) {
        // a wait ran out: tell the host, and let copies in flight land
        if (a.err) atomicOr(a.err, kErrWaitTimeout);
        const long long t0 = clock64();
        while (clock64() - t0 < 20000000ll) __nanosleep(1000);
    }
}

template <typename T, int D, int RB>
int launch_rows(const AttnArgs& a, cudaStream_t st) {
    using L = Layout<D, RB>;
    static std::atomic<unsigned long long> set_on{0};
    if (int s = allow_smem(paged4_attn<T, D, RB>, (int)L::kBytes, set_on)) return s;
    static_assert(kSlotsAt + 2 * kMaxCtas * slot_floats<L::kRows, D>() * 4 <= kTcWorkspaceAt && kMaxCtas * 4 <= kSlotsAt,
                  "the slots must fit the workspace");
    int ctas = sm_count() * L::kPerSm;  // as many as the SMs hold at once
    if (ctas > kMaxCtas) ctas = kMaxCtas;
    paged4_attn<T, D, RB><<<ctas, kThreads, L::kBytes, st>>>(a);
    INFERNT_CUDA_TRY(cudaGetLastError());
    return INFERNT_OK;
}

// rows: query rows of a KV head that most sequences have
template <typename T, int D>
int launch(const AttnArgs& a, long long rows, cudaStream_t st) {
    if (rows <= 8) return launch_rows<T, D, 1>(a, st);
    if (rows <= 16) return launch_rows<T, D, 2>(a, st);
    return launch_rows<T, D, 4>(a, st);
}

}  // namespace
}  // namespace infernt

extern "C" int infernt_paged4_attention(void* out, int ldo, const void* q, int ldq, int nq,
                                        const infernt_paged_cache4* cache, const infernt_ragged_batch* batch, int window,
                                        int sinks, float scale, float* lse, void* workspace, unsigned* err,
                                        void* stream) {
    using namespace infernt;
    const char* op = "paged4_attention";
    if (int s = check_paged_cache4(op, cache)) return s;
    const infernt_paged_cache geometry = geometry4(*cache);
    AttnArgs a;
    bool empty;
    // tiles of both kernels, for the bound on the call's work: the smaller of each
    if (int s = attention_args(op, out, ldo, q, ldq, nq, &geometry, batch, window, sinks, scale, lse, workspace, err, 8,
                               kTcTileKeys, &a, &empty))
        return s;
    if (empty) return INFERNT_OK;
    if (int s = check_device_pointer(op, "the scales", cache->scales)) return s;
    a.scales = cache->scales;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int D = cache->head_dim;
    // Sequences of up to kMostRows query rows a KV head are bound by their keys,
    // longer ones by their products.  Where the batch's counts do not say that
    // all sequences are as long as the longest, each kernel takes its own.
    const long long most = (long long)batch->max_q_len * a.G;
    const bool chunks = most > kMostRows, both = chunks && batch->num_rows < (long long)batch->num_seqs * batch->max_q_len;
    if (!chunks || both) {
        // rows of an item: those of the longest sequence, or, beside a chunk, what the others have on average
        long long rows = most;
        if (both) {
            a.max_rows = kMostRows;
            rows = std::max(1, (batch->num_rows - batch->max_q_len + batch->num_seqs - 2) / std::max(1, batch->num_seqs - 1));
            rows *= a.G;
        }
        int s;
        if (cache->dtype == INFERNT_DTYPE_BF16)
            s = D == 64 ? launch<__nv_bfloat16, 64>(a, rows, st) : launch<__nv_bfloat16, 128>(a, rows, st);
        else
            s = D == 64 ? launch<__half, 64>(a, rows, st) : launch<__half, 128>(a, rows, st);
        if (s || !chunks) return s;
        a.min_rows = kMostRows;
        a.max_rows = kMaxPositions;
    }
    return paged4_attention_tc(a, D, cache->dtype, both, st);
}
