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
#include <type_traits>

#include "paged_attention.cuh"
#include "tc_mma.cuh"
#include "warp_mma.cuh"

namespace infernt {
namespace {

// This file's kernel takes query rows by the dozen: single tokens, drafts of
// a few, and any chunk whose pages do not make whole boxes.  It is bound by
// the bytes of K and V.  A CTA is a producer warp, which streams the CTA's
// tiles of 64 keys through a ring of shared memory without a pause between
// items, and four warps that consume them on mma.sync; two CTAs share an SM
// and keep 128 KB in flight there.  (Without the producer, each item's start
// waited for its own first tiles and each tile for a barrier of the CTA:
// 64 sequences of 512 to 2048 positions, 32/4 heads of 64, took 38 us.)
constexpr int kTileKeys = 64;   // keys of a K / V tile
constexpr int kItemRows = 64;   // query rows of an item: four warps of 16
constexpr int kConsumers = 128;
constexpr int kThreads = kConsumers + 32;
constexpr uint32_t kBlock = kTileKeys * 128;  // a block of 64 columns: rows of 128 bytes
static_assert(kBlock == 8192, "as chunk_at has it");

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

// Shared memory: the ring (per stage the blocks of K, then those of V; the
// 16-byte chunk c of row r lies at c ^ (r & 7), as a tensor map with 128-byte
// swizzle writes it), then the scratch in which the warps' results meet: up
// to three sets of 8 rows.
template <int D>
struct Layout {
    static constexpr int kBlocks = D / 64;
    static constexpr int kStages = D == 64 ? 6 : 3;
    static constexpr uint32_t kTile = kBlocks * kBlock;
    static constexpr uint32_t kScratch = kStages * 2 * kTile;
    static constexpr uint32_t kBytes = kScratch + 3 * 8 * (D + 2) * 4 + 1024;
};

template <int ST>
struct Ring {
    uint64_t full[ST], empty[ST];
};

// The producer warp: K and V tiles of the CTA's parts, in order.  BOXES: page
// by page through the tensor maps (a page that no row sees, or that the pool
// does not have, becomes zeros); otherwise row by row, hidden rows as zeros.
template <int D, bool BOXES>
__device__ __forceinline__ void produce(const AttnArgs& a, const Place& place, const CUtensorMap& tm_k,
                                        const CUtensorMap& tm_v, uint32_t base, Ring<Layout<D>::kStages>& ring,
                                        bool& ok) {
    using L = Layout<D>;
    constexpr int ST = L::kStages;
    const int lane = threadIdx.x & 31;
    const int ps = a.b.page_size, per_tile = ps < kTileKeys ? kTileKeys / ps : 1;
    const int box_rows = ps < kTileKeys ? ps : kTileKeys;
    uint32_t st = 0, turn = 1;  // the first round's stages are free
    walk<kItemRows, kTileKeys>(a, place, [&](const PagedSeq&, const Item& it, const Part& part) {
#pragma unroll 1
        for (int j = part.j0; j < part.j1; ++j) {
            const int k0 = tile_key<kTileKeys>(it, j);
            const uint32_t kt = base + st * 2 * L::kTile, vt = kt + L::kTile;
            if (BOXES) {
                int page = a.b.num_pages, row = 0;
                if (lane < per_tile) {
                    const int p0 = k0 + lane * box_rows, pi = a.b.by_page(p0);
                    row = p0 - pi * ps;
                    if (p0 < it.hi && (p0 + box_rows > it.lo || p0 < it.sink_end)) {
                        page = a.b.table[(size_t)part.s * a.b.table_stride + pi];
                        if (page < 0 || page >= a.b.num_pages) {
                            if (a.err) atomicOr(a.err, kErrPage);
                            page = a.b.num_pages;
                        }
                    }
                }
                tc_wait_bar(&ring.empty[st], turn, ok);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) return;
                if (lane == 0) mbar_arrive_expect_tx(&ring.full[st], 2 * L::kTile);
                __syncwarp();
                if (lane < per_tile)
#pragma unroll
                    for (int b = 0; b < L::kBlocks; ++b) {
                        tma_load_4d(kt + b * kBlock + lane * box_rows * 128, &tm_k, 64 * b, row, it.kvh, page,
                                    &ring.full[st]);
                        tma_load_4d(vt + b * kBlock + lane * box_rows * 128, &tm_v, 64 * b, row, it.kvh, page,
                                    &ring.full[st]);
                    }
            } else {
                // rows `lane` and `lane + 32` of the tile; -1: zeros
                int rows[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int p = k0 + lane + 32 * h;
                    rows[h] = item_sees(it, p) ? pool_row(a.b, part.s, it.kvh, p, a.err) : -1;
                }
                tc_wait_bar(&ring.empty[st], turn, ok);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) return;
                constexpr int CH = D / 8, RPI = 32 / CH;  // chunks of a row, rows at once
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll 4
                    for (int i = 0; i < 32 / RPI; ++i) {
                        const int r = i * RPI + lane / CH, ch = lane % CH;
                        const int pr = __shfl_sync(0xffffffffu, rows[h], r);
                        const size_t off = (size_t)(pr < 0 ? 0 : pr) * (D * 2) + ch * 16;
                        const uint32_t at = chunk_at(0, r + 32 * h, ch);
                        cp_async16(kt + at, static_cast<const char*>(a.k) + off, pr < 0 ? 0u : 16u);
                        cp_async16(vt + at, static_cast<const char*>(a.v) + off, pr < 0 ? 0u : 16u);
                    }
                // this lane's arrival, once its copies have landed
                asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_addr(&ring.full[st]))
                             : "memory");
            }
            if (++st == ST) {
                st = 0;
                turn ^= 1;
            }
        }
    });
    if (!BOXES) cp_async_wait<0>();
}

// What a warp knows of its 16 rows after a part: lane (g, tig) has rows g and
// g + 8, of each the columns 8 b + 2 tig and + 1.
template <int D>
struct RowState {
    float m[2], l[2];
    float acc[D / 8][4];
};

// The tiles [j0, j1) of an item by four warps: RB blocks of 16 rows, each by
// 4 / RB warps that share a tile's keys between them.  The result is in the
// warps of the first key share (warp < RB).
template <typename T, int D, int RB, bool BOXES>
__device__ __forceinline__ RowState<D> consume(const AttnArgs& a, const PagedSeq& seq, const Item& it, const Part& part,
                                               uint32_t base, float* scratch, Ring<Layout<D>::kStages>& ring,
                                               uint32_t& st, uint32_t& turn, const Current* cur,
                                               volatile int* found_in, bool& ok) {
    using L = Layout<D>;
    constexpr int KS = 4 / RB, WK = kTileKeys / KS, NT = WK / 8;  // key shares, keys and n-tiles of a warp
    constexpr int KC = D / 16, DB = D / 8, ST = L::kStages;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tig = lane & 3;
    const int rb = warp % RB, ks = warp / RB;
    // query fragments of rows g and g + 8 of the warp's block
    uint32_t qa[KC][4];
    int pos[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = rb * 16 + g + 8 * h, row = it.row0 + min(r, it.rows - 1), token = a.by_g(row);
        pos[h] = r < it.rows ? row_pos(seq, token) : -1;
        const uint32_t* q = reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(a.q) +
                                                              (long long)(seq.row0 + token) * a.ldq +
                                                              (it.kvh * a.G + row - token * a.G) * D + 2 * tig);
#pragma unroll
        for (int k = 0; k < KC; ++k) {
            qa[k][h] = __ldg(q + 8 * k);
            qa[k][h + 2] = __ldg(q + 8 * k + 4);
        }
    }
    RowState<D> s;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        s.m[h] = -INFINITY;
        s.l[h] = 0.0f;
    }
#pragma unroll
    for (int b = 0; b < DB; ++b) s.acc[b][0] = s.acc[b][1] = s.acc[b][2] = s.acc[b][3] = 0.0f;
    const bool busy = rb * 16 < it.rows, mixed = it.pos_first != it.pos_last;

#pragma unroll 1
    for (int j = part.j0; j < part.j1; ++j) {
        const int k0 = tile_key<kTileKeys>(it, j);
        const uint32_t kt = base + st * 2 * L::kTile, vt = kt + L::kTile;
        tc_wait_bar(&ring.full[st], turn, ok);
        if (busy) {
            const bool whole = seen_whole<kTileKeys>(a, it, k0);
            if (!whole && (mixed || (BOXES && has_hidden<kTileKeys>(it, k0))))
                clean_rows<T, D, WK>(cur[warp], k0, vt, ks * WK, mixed, found_in);
            float sc[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.0f;
#pragma unroll
            for (int k = 0; k < KC; ++k)
#pragma unroll
                for (int n = 0; n < NT / 2; ++n) {
                    const int x = lane >> 3, row = ks * WK + 8 * (2 * n + (x >> 1)) + (lane & 7);
                    uint32_t b0, b1, b2, b3;
                    ldsm_x4(chunk_at(kt, row, 2 * k + (x & 1)), b0, b1, b2, b3);
                    mma_16816<T>(sc[2 * n], qa[k], b0, b1);
                    mma_16816<T>(sc[2 * n + 1], qa[k], b2, b3);
                }
            // a tile that every row sees whole needs no mask
            if (!whole) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!row_sees(a, pos[e >> 1], k0 + ks * WK + 8 * n + 2 * tig + (e & 1))) sc[n][e] = -INFINITY;
            }
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx[e >> 1] = fmaxf(mx[e >> 1], sc[n][e]);
            bool grow = false;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2)) * a.scale_log2;
                mx[h] -= kShift<T>;
                grow |= mx[h] > s.m[h] + kRescale;
            }
            // the reference moves only when probabilities would pass 2^(kRescale + kShift)
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float n = fmaxf(s.m[h], mx[h]), f = s.m[h] == -INFINITY ? 0.0f : ex2(s.m[h] - n);
                    s.m[h] = n;
                    s.l[h] *= f;
#pragma unroll
                    for (int b = 0; b < DB; ++b) {
                        s.acc[b][2 * h] *= f;
                        s.acc[b][2 * h + 1] *= f;
                    }
                }
            }
            const float ref[2] = {s.m[0] == -INFINITY ? 0.0f : s.m[0], s.m[1] == -INFINITY ? 0.0f : s.m[1]};
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sc[n][e] = ex2(fmaf(sc[n][e], a.scale_log2, -ref[e >> 1]));
                    s.l[e >> 1] += sc[n][e];
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
                    const int x = lane >> 3, row = ks * WK + 16 * kk + 8 * (x & 1) + (lane & 7);
                    uint32_t v0, v1, v2, v3;
                    ldsm_x4_trans(chunk_at(vt, row, 2 * b + (x >> 1)), v0, v1, v2, v3);
                    mma_16816<T>(s.acc[2 * b], pa, v0, v1);
                    mma_16816<T>(s.acc[2 * b + 1], pa, v2, v3);
                }
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
    for (int h = 0; h < 2; ++h) {
        s.l[h] += __shfl_xor_sync(0xffffffffu, s.l[h], 1);
        s.l[h] += __shfl_xor_sync(0xffffffffu, s.l[h], 2);
    }
    // the key shares of a block of rows, joined in order by its first warp
    if (KS > 1) {
        float* m_s = scratch + 3 * 8 * D;
        float* l_s = m_s + 3 * 8;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (8 * h >= it.rows) break;
            const int set = (ks - 1) * RB + rb;
            if (h) named_sync(1, kConsumers);  // the first rows have been read
            if (ks > 0) {
                if (tig == 0) {
                    m_s[set * 8 + g] = s.m[h];
                    l_s[set * 8 + g] = s.l[h];
                }
#pragma unroll
                for (int b = 0; b < DB; ++b)
                    *reinterpret_cast<float2*>(scratch + (set * 8 + g) * D + 8 * b + 2 * tig) =
                        make_float2(s.acc[b][2 * h], s.acc[b][2 * h + 1]);
            }
            named_sync(1, kConsumers);
            if (ks == 0) {
                float M = s.m[h], f[KS];
#pragma unroll
                for (int k = 1; k < KS; ++k) M = fmaxf(M, m_s[((k - 1) * RB + rb) * 8 + g]);
                f[0] = s.m[h] == -INFINITY ? 0.0f : ex2(s.m[h] - M);
                s.m[h] = M;
                s.l[h] *= f[0];
#pragma unroll
                for (int k = 1; k < KS; ++k) {
                    const float mk = m_s[((k - 1) * RB + rb) * 8 + g];
                    f[k] = mk == -INFINITY ? 0.0f : ex2(mk - M);
                    s.l[h] = fmaf(l_s[((k - 1) * RB + rb) * 8 + g], f[k], s.l[h]);
                }
#pragma unroll
                for (int b = 0; b < DB; ++b) {
                    float x = s.acc[b][2 * h] * f[0], y = s.acc[b][2 * h + 1] * f[0];
#pragma unroll
                    for (int k = 1; k < KS; ++k) {
                        const float2 o = *reinterpret_cast<const float2*>(
                            scratch + (((k - 1) * RB + rb) * 8 + g) * D + 8 * b + 2 * tig);
                        x = fmaf(o.x, f[k], x);
                        y = fmaf(o.y, f[k], y);
                    }
                    s.acc[b][2 * h] = x;
                    s.acc[b][2 * h + 1] = y;
                }
            }
        }
    }
    return s;
}

// The values that clean_rows took out of a part's tiles, added to the results
// of the rows r0 + g and r0 + g + 8 that see them: to this lane's columns, as it
// has just written them to the slot, or to out.  (On memory, and with the part
// read from shared memory: on registers in line with the tiles, 32 sequences
// with a window of 4096 took 105 us, not 98.)
template <typename T, int D>
__device__ __noinline__ void restore_rows(const AttnArgs& a, const Current& cur, int row_base, int r0, float* slot) {
    const int lane = threadIdx.x & 31, g = lane >> 2, tig = lane & 3;
    each_not_finite<T, D, kTileKeys>(a, cur, [&](int p, const T* v) {
        for (int r = r0 + g; r < min(cur.it.rows, r0 + 16); r += 8) {
            const int row = cur.it.row0 + r, token = a.by_g(row), head = cur.it.kvh * a.G + row - token * a.G;
            if (!row_sees(a, cur.it.pos_first + token - a.by_g(cur.it.row0), p)) continue;
            T* out = static_cast<T*>(a.out) + (long long)(row_base + token) * a.ldo + (long long)head * D;
            for (int d = 2 * tig; d < D; d += 8) {
                const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(v + d));
                const float2 x = Half16<T>::unpack(w & Half16<T>::not_finite(w));
                if (slot) {
                    float2* at = reinterpret_cast<float2*>(slot + r * D + d);
                    *at = make_float2(at->x + x.x, at->y + x.y);
                } else {
                    uint32_t* at = reinterpret_cast<uint32_t*>(out + d);
                    const float2 o = Half16<T>::unpack(*at);
                    *at = Half16<T>::pack(o.x + x.x, o.y + x.y);
                }
            }
        }
    });
}

template <typename T, int D, bool BOXES>
__global__ void __launch_bounds__(kThreads, 2)
    paged_attn(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap tm_k,
               const __grid_constant__ CUtensorMap tm_v) {
    using L = Layout<D>;
    constexpr int M = kItemRows, ST = L::kStages;
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ Ring<ST> ring;
    __shared__ int last_s, early_s, found_s;  // found_s: the last part in which clean_rows found something
    __shared__ Current cur_s[kConsumers / 32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tig = lane & 3;
    const uint32_t base = (smem_addr(smem) + 1023u) & ~1023u;
    float* scratch = reinterpret_cast<float*>(smem + (base - smem_addr(smem)) + L::kScratch);
    if (tid == 0) {
        for (int i = 0; i < ST; ++i) {
            mbar_init(&ring.full[i], BOXES ? 1 : 32);
            mbar_init(&ring.empty[i], kConsumers / 32);
        }
        mbar_fence_init();
        found_s = 0;
        for (Current& c : cur_s) c.no = 0;
    }
    const Place place = find_place<M, kTileKeys, kThreads>(a);  // its barriers publish the set-up
    pdl_launch_dependents();  // the tcgen05 kernel may take SMs as they become free
    if (place.s < 0) return;
    bool ok = true;
    if (warp == kConsumers / 32) {
        produce<D, BOXES>(a, place, tm_k, tm_v, base, ring, ok);
    } else {
        uint32_t st = 0, turn = 0;
        walk<M, kTileKeys>(a, place, [&](const PagedSeq& seq, const Item& it, const Part& p) {
            set_current(cur_s[warp], it, p);
            // the part, its rows' results and what becomes of them, for RB blocks of rows
            auto run = [&](auto blocks) {
                constexpr int RB = decltype(blocks)::value;
                const RowState<D> s = consume<T, D, RB, BOXES>(a, seq, it, p, base, scratch, ring, st, turn, cur_s,
                                                                   &found_s, ok);
                const bool split = p.first != p.last;
                unsigned taken = 0;
                if (split && tid == 0) taken = tickets_taken(a, p);
                if (warp < RB) {
                    float* slot = slot_of<M, D>(a, blockIdx.x, p.first);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int r = warp * 16 + g + 8 * h;
                        if (r >= it.rows) continue;
                        if (split) {
#pragma unroll
                            for (int b = 0; b < D / 8; ++b)
                                *reinterpret_cast<float2*>(slot + r * D + 8 * b + 2 * tig) =
                                    make_float2(s.acc[b][2 * h], s.acc[b][2 * h + 1]);
                            if (tig == 0) {
                                slot[M * D + r] = s.m[h];
                                slot[M * D + M + r] = s.l[h];
                            }
                        } else {
#pragma unroll
                            for (int b = 0; b < D / 8; ++b)
                                write_pair<T, D>(a, seq, it.kvh, it.row0 + r, 8 * b + 2 * tig,
                                                 {s.m[h], s.l[h], s.acc[b][2 * h], s.acc[b][2 * h + 1]});
                        }
                    }
                    // by this warp, or by one whose keys have met these rows at the barrier of their join
                    if (__any_sync(0xffffffffu, *static_cast<volatile int*>(&found_s) >= cur_s[warp].no))
                        restore_rows<T, D>(a, cur_s[warp], seq.row0, warp * 16, split ? slot : nullptr);
                }
                if (!split) return;
                // where all others have arrived already, no ticket is needed
                if (tid == 0) {
                    early_s = taken == (unsigned)(p.last - p.first);
                    if (early_s) a.tickets[p.first] = 0u;  // ready for the next call
                }
                named_sync(1, kConsumers);
                const bool early = early_s != 0;
                if (!early && tid == 0) {
                    // the others' writes, ordered before by the barrier, become visible with this thread's fence
                    __threadfence();
                    unsigned* ticket = a.tickets + p.first;
                    last_s = atomicAdd(ticket, 1u) + 1u == (unsigned)(p.last - p.first + 1);
                    if (last_s) *ticket = 0u;  // ready for the next call
                    __threadfence();
                }
                if (!early) {
                    named_sync(1, kConsumers);
                    if (!last_s) return;
                }
                // a warp a row, two columns a lane, two rows at once
                for (int r = warp; r < it.rows; r += 2 * (kConsumers / 32)) {
                    const int r2 = r + kConsumers / 32;
#pragma unroll
                    for (int d = 2 * lane; d < D; d += 64) {
                        const Joined v = join_slots<M, D>(a, p.first, p.last, r, d);
                        const Joined v2 = join_slots<M, D>(a, p.first, p.last, min(r2, it.rows - 1), d);
                        write_pair<T, D>(a, seq, it.kvh, it.row0 + r, d, v);
                        if (r2 < it.rows) write_pair<T, D>(a, seq, it.kvh, it.row0 + r2, d, v2);
                    }
                }
            };
            if (it.rows <= 16)
                run(std::integral_constant<int, 1>());
            else if (it.rows <= 32)
                run(std::integral_constant<int, 2>());
            else
                run(std::integral_constant<int, 4>());
            // the scratch is free, and everyone has read last_s
            named_sync(1, kConsumers);
        });
    }
    if (!ok) {
        // a wait ran out: tell the host, and let copies in flight land
        if (a.err) atomicOr(a.err, kErrWaitTimeout);
        const long long t0 = clock64();
        while (clock64() - t0 < 20000000ll) __nanosleep(1000);
    }
}

template <typename T, int D, bool BOXES>
int launch_boxes(const AttnArgs& args, cudaStream_t st) {
    using L = Layout<D>;
    AttnArgs a = args;
    CUtensorMap mk = {}, mv = {};
    if (BOXES) {
        if (int s = paged_pool_map(&mk, a, a.k, D, Half16<T>::kBf16, kTileKeys)) return s;
        if (int s = paged_pool_map(&mv, a, a.v, D, Half16<T>::kBf16, kTileKeys)) return s;
    }
    static std::atomic<unsigned long long> set_on{0};
    if (int s = allow_smem(paged_attn<T, D, BOXES>, (int)L::kBytes, set_on)) return s;
    static_assert(kSlotsAt + 2 * kMaxCtas * slot_floats<kItemRows, D>() * 4 <= kTcWorkspaceAt &&
                      kMaxCtas * 4 <= kSlotsAt,
                  "the slots must fit the workspace");
    int ctas = sm_count() * 2;  // as many as the SMs hold at once
    if (ctas > kMaxCtas) ctas = kMaxCtas;
    paged_attn<T, D, BOXES><<<ctas, kThreads, L::kBytes, st>>>(a, mk, mv);
    INFERNT_CUDA_TRY(cudaGetLastError());
    return INFERNT_OK;
}

template <typename T, int D>
int launch(const AttnArgs& a, cudaStream_t st) {
    return paged_attention_boxes(a.b.page_size) ? launch_boxes<T, D, true>(a, st) : launch_boxes<T, D, false>(a, st);
}

}  // namespace
}  // namespace infernt

extern "C" size_t infernt_paged_attention_workspace_bytes(void) { return infernt::kWorkspaceBytes; }

namespace infernt {

int attention_args(const char* op, void* out, int ldo, const void* q, int ldq, int nq, const infernt_paged_cache* cache,
                   const infernt_ragged_batch* batch, int window, int sinks, float scale, float* lse, void* workspace,
                   unsigned* err, std::initializer_list<WorkBound> work, AttnArgs* args, bool* empty) {
    if (int s = check_paged_cache(op, cache)) return s;
    if (int s = check_ragged_batch(op, batch)) return s;
    INFERNT_REQUIRE(q && out && workspace, "%s: null pointer", op);
    const int D = cache->head_dim, nkv = cache->num_kv_heads;
    INFERNT_REQUIRE(nq >= 1 && nq % nkv == 0 && nq / nkv <= 128, "%s: %d query heads, %d KV heads", op, nq, nkv);
    INFERNT_REQUIRE(ldq >= (long long)nq * D && ldo >= (long long)nq * D && ldq % 8 == 0 && ldo % 8 == 0,
                    "%s: rows %d and %d apart for %d heads of %d (multiples of 8)", op, ldq, ldo, nq, D);
    INFERNT_REQUIRE(aligned16(q) && aligned16(out) && aligned16(workspace),
                    "%s: q, out and workspace must be 16-byte aligned", op);
    INFERNT_REQUIRE(reinterpret_cast<uintptr_t>(lse) % 4 == 0 && reinterpret_cast<uintptr_t>(err) % 4 == 0,
                    "%s: misaligned lse or err", op);
    INFERNT_REQUIRE(q != out, "%s: out may not be q", op);
    INFERNT_REQUIRE(window >= 0 && sinks >= 0 && (window > 0 || sinks == 0), "%s: window %d, sinks %d", op, window,
                    sinks);
    INFERNT_REQUIRE(std::isfinite(scale) && scale >= 0.0f, "%s: scale %g", op, scale);
    const int G = nq / nkv;
    INFERNT_REQUIRE((long long)batch->num_rows * G < kMaxPositions, "%s: %d rows of %d heads", op, batch->num_rows, nq);
    // the units of the schedule are counted in 32 bits
    const long long most_kv = std::min<long long>((long long)batch->table_stride * cache->page_size, kMaxPositions);
    for (const WorkBound& w : work)
        INFERNT_REQUIRE((w.rows / w.item_rows + batch->num_seqs) * nkv <
                            (1ll << 30) / (most_kv / w.tile_keys + 2 + kItemCost),
                        "%s: %d rows of %d heads over up to %lld positions (split the call)", op, batch->num_rows, nq,
                        most_kv);
    *empty = batch->num_seqs == 0 || batch->num_rows == 0;
    if (*empty) return INFERNT_OK;
    if (int s = check_batch_pointers(op, cache, batch, err)) return s;
    if (int s = check_device_pointer(op, "q", q)) return s;
    if (int s = check_device_pointer(op, "out", out)) return s;
    if (int s = check_device_pointer(op, "lse", lse)) return s;
    if (int s = check_device_pointer(op, "workspace", workspace)) return s;
    AttnArgs& a = *args;
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
    a.min_units = kLeast;
    a.min_rows = 0;
    a.max_rows = kMaxPositions;
    a.tickets = static_cast<unsigned*>(workspace);
    a.slots = reinterpret_cast<float*>(static_cast<char*>(workspace) + kSlotsAt);
    a.err = err;
    a.scales = nullptr;
    return INFERNT_OK;
}

}  // namespace infernt

extern "C" int infernt_paged_attention(void* out, int ldo, const void* q, int ldq, int nq,
                                       const infernt_paged_cache* cache, const infernt_ragged_batch* batch, int window,
                                       int sinks, float scale, float* lse, void* workspace, unsigned* err,
                                       void* stream) {
    using namespace infernt;
    const char* op = "paged_attention";
    if (int s = check_paged_cache(op, cache)) return s;
    if (int s = check_ragged_batch(op, batch)) return s;
    const int D = cache->head_dim, nkv = cache->num_kv_heads, G = nq / nkv;
    const bool chunks = paged_attention_boxes(cache->page_size) && (long long)batch->max_q_len * G > kItemRows;
    const WorkBound work = {(long long)batch->num_rows * G, chunks ? kTcItemRows : kItemRows,
                            chunks ? kTcTileKeys : kTileKeys};
    AttnArgs a;
    bool empty;
    if (int s = attention_args(op, out, ldo, q, ldq, nq, cache, batch, window, sinks, scale, lse, workspace, err,
                               {work}, &a, &empty))
        return s;
    if (empty) return INFERNT_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // Sequences of up to kItemRows query rows are bound by the bytes of their
    // keys, which the mma.sync kernel streams faster; longer ones by their
    // products.  Where the batch's counts do not say that all sequences are
    // as long as the longest, each kernel takes its own.
    const bool both = chunks && batch->num_rows < (long long)batch->num_seqs * batch->max_q_len;
    if (both) a.max_rows = kItemRows;
    if (!chunks || both) {
        int s;
        if (cache->dtype == INFERNT_DTYPE_BF16)
            s = D == 64 ? launch<__nv_bfloat16, 64>(a, st) : launch<__nv_bfloat16, 128>(a, st);
        else
            s = D == 64 ? launch<__half, 64>(a, st) : launch<__half, 128>(a, st);
        if (s || !chunks) return s;
        a.min_rows = kItemRows;
        a.max_rows = kMaxPositions;
    }
    return paged_attention_tc(a, D, cache->dtype, both, st);
}
