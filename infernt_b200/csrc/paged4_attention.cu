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
//   - codes go from shared memory to the A operand by a logic operation and an
//     exact fp16 one for two of them, and a shift for eight: the operand is the
//     whole numbers c - z, the scale s of a key multiplies its scores (K) or
//     its probabilities (V), four values a thread for 16 keys.
//   - the contraction's order is free: a thread takes 32 neighbouring
//     elements of a K row (and the same ones of Q), so a row is a 16-byte load
//     without a shuffle; for V^T it takes D / 8 neighbouring elements of four
//     keys.  P^T comes out of the scores by a transposition of 8 x 8 blocks.
// 16 sequences of 32768 positions, 32/8 heads of 128 (554 MB, 85 us of HBM): 137
// to 145 us, 4.0 TB/s, of which 111 grow with the keys: some 23 instructions a key and
// warp, and the rest is the first loads, unequal ends and the joins.  64
// sequences of 512 to 2048 with 40 query rows of 64: 40 us, where 2 instructions
// of 4 that could be issue a cycle: 12 warps an SM with their waits for products.
// Spilled, in bytes a thread: 24 to 56 where registers are held to let 3 or 4 CTAs
// an SM run (D 128 of 8 rows, D 64 of 16 and 24), 244 at D 128 of 32 rows.
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "paged4.cuh"
#include "paged_attention.cuh"
#include "warp_mma.cuh"

namespace infernt {
namespace {

constexpr int kWarps = 4;
constexpr int kGroups = 2;  // of 16 keys, of a tile, a warp
constexpr int kWarpKeys = 16 * kGroups;
constexpr int kKeys = kWarps * kWarpKeys;  // of a tile
constexpr int kThreads = 32 * kWarps;
// Parts of one tile of 128 keys: a border moves less than with two (the 16-bit
// kernels' tiles are of 64; the drafts of 64 sequences of 512 to 2048 took 41.5 us
// with two, 43 with three, 40 so).
constexpr int kLeast4 = kItemCost + 1;
constexpr int kStages = 3;     // tiles of a warp's ring: one is worked on, two are on their way
// Query rows of a KV head above which the tcgen05 kernel is faster.  64 sequences
// of 512 to 2048 positions, and 4 of 30000 to 32768, take here and there: of 64
// elements, 24 rows 30 and 51 us, 39 and 71; 48 rows 41 and 51, 48 and 70; 64
// rows 51 and 51, 56 and 70; of 128, 32 rows 85 and 102, 95 and 137; 48 rows 113
// and 104, 125 and 138; 64 rows 147 and 105, 157 and 138.
constexpr int most_rows(int dim) { return dim == 64 ? 64 : 48; }

// The products are in fp16 whatever the cache's type is, since codes get there
// with one shift for eight of them (bf16, with seven bits behind its leading
// one, takes three): Q enters times a power of two that brings the largest
// element of the item's rows to 2^14 (what is lost of an element is 2^-38 of
// that one, and so of the item's largest scores),
// and a weight is 2^(s - m) s_V.  m follows s + log2 s_V, so weights fit
// whatever V's scales are: m moves when a key's weights would pass kMostWeight
// and puts a row's largest at 2^kUp to 2^(kUp + 1).  Normal numbers then reach
// down to 2^-18 of it.
constexpr float kUp = 4.0f;
constexpr float kMostWeight = 16384.0f;
// Scales below 2^-92 (the least is 2^-100, of vectors of zeros too) do not lower
// m further, and m moves too where a 2^(s - m) passes 2^97: the sum of 2^30 of
// them stays in FP32.  Weights beside the least scale are 2^-4 to 2^-3 at a row's
// largest, and normal numbers down to 2^-10 of it.  At the other end, beside V
// vectors of scale 2^x, a 2^(s - m) below 2^(x - 130) of the row's largest is 0.
constexpr float kLeastLog = -92.0f, kMostSingle = 1.5845632502852868e29f;
// sum + l 2^d, d <= 0, for sums of weights: the m of two parts are up to 217 apart
// by their V scales alone, and their sums as far the other way.
__device__ __forceinline__ float add_lowered(float sum, float l, float d) {
    return fmaf(l * ex2(fminf(d + 120.0f, 0.0f)), ex2(fmaxf(d, -120.0f)), sum);
}

// Shared memory: a ring of its own for each warp, per stage the codes of its K
// and V rows and their scale words.  When a part is done the ring is empty, and
// what the warp knows of the item's rows (its set) lies over it.
template <int D, int RB>
struct Layout {
    static constexpr int kRows = 8 * RB;
    static constexpr uint32_t kCodes = kWarpKeys * D / 2;
    static constexpr uint32_t kStage = 2 * kCodes + kWarpKeys * 4;
    static constexpr uint32_t kSet = kRows * (D + 2) * 4;
    static constexpr uint32_t kRing = kStages * kStage > kSet ? kStages * kStage : (kSet + 127) / 128 * 128;
    // CTAs of an SM: what its registers hold (128, 168 or 255 a thread)
    static constexpr int kPerSm = RB * D <= 128 ? 4 : RB * D < 256 ? 3 : 2;
    // Q as the B operands of one n-tile stay in registers; of several, in shared memory
    static constexpr bool kSharedQ = RB > 1;
    static constexpr uint32_t kQ = kSharedQ ? RB * (D / 32) * 512 + 32 : 0;  // and the warps' largest
    static constexpr uint32_t kQAt = kWarps * kRing;
    static constexpr uint32_t kBytes = kQAt + kQ + 128;
    static_assert(kPerSm * (kBytes + 2048) <= 228 * 1024, "");
};

__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, uint32_t src_bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
__device__ __forceinline__ void cp_async16_always(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
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
// The largest, NaN where one of them is.
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// What codes become whole numbers with.  A nibble in the low bits of a half
// under the exponent of 2^10 is 1024 + c, one four bits up under that of 2^6
// 64 + c.  The masks come out of a register that the compiler cannot see through: as
// immediates they take two logic operations for each pair, and those are the
// unit that this kernel has least of.
struct Masks {
    uint32_t low, high, low_one, high_one;
};
__device__ __forceinline__ Masks make_masks() {
    Masks k;
    asm volatile("mov.b32 %0, 0x000f000f;" : "=r"(k.low));
    asm volatile("mov.b32 %0, 0x00f000f0;" : "=r"(k.high));
    asm volatile("mov.b32 %0, 0x64006400;" : "=r"(k.low_one));
    asm volatile("mov.b32 %0, 0x54005400;" : "=r"(k.high_one));
    return k;
}
__device__ __forceinline__ uint32_t half2_sub(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// A pair of zeros as what is taken off: 1024 + z and 64 + z.
struct Zeros {
    uint32_t low, high;
};
__device__ __forceinline__ Zeros make_zeros(uint32_t pair, const Masks& k) {
    Zeros z;
    z.low = and_or(pair, k.low, k.low_one);
    z.high = half2_sub(z.low, 0x63806380u);  // 960
    return z;
}
// The pairs of nibbles (j, j + 4) of w as c - z.
__device__ __forceinline__ void whole(uint32_t w, const Zeros& z, const Masks& k, uint32_t (&p)[4]) {
    const uint32_t v = w >> 8;
    p[0] = half2_sub(and_or(w, k.low, k.low_one), z.low);
    p[1] = half2_sub(and_or(w, k.high, k.high_one), z.high);
    p[2] = half2_sub(and_or(v, k.low, k.low_one), z.low);
    p[3] = half2_sub(and_or(v, k.high, k.high_one), z.high);
}

// The copies of a tile's keys of this warp, the pool row of key `lane` in row
// (-1: no row of the item sees it, or the pool does not have its page): codes
// (not of such keys: what lies there are numbers whatever it is, and copies of
// one row for all of them would meet in one place of L2), and scale words, 0
// for such keys.  Every warp fetches for itself, two tiles ahead, so none waits
// for another; the table's entry of a key is loaded three tiles ahead and looked
// at one tile later (looked at at once, it held the warp up).  (16
// sequences of 32768 positions took 141 us with a warp that streamed for the
// others, which spends a fifth of the issue slots on its loops over pages, and
// 141 with three bulk copies a warp and tile.)
template <int D>
__device__ __forceinline__ void fetch(const AttnArgs& a, int row, int lane, uint32_t stage) {
    constexpr uint32_t ROW = D / 2, CODES = kWarpKeys * ROW;
    constexpr int CH = ROW / 16, RPI = 32 / CH;  // 16-byte pieces of a row, rows at once
    const char* kc = static_cast<const char*>(a.k) + 16 * (lane % CH);
    const char* vc = static_cast<const char*>(a.v) + 16 * (lane % CH);
#pragma unroll
    for (int i = 0; i < kWarpKeys / RPI; ++i) {
        const int r = __shfl_sync(0xffffffffu, row, i * RPI + lane / CH);
        const uint32_t at = stage + (i * RPI) * ROW + lane * 16;
        if (r >= 0) {
            cp_async16_always(at, kc + (size_t)r * ROW);
            cp_async16_always(at + CODES, vc + (size_t)r * ROW);
        }
    }
    cp_async4(stage + 2 * CODES + 4 * lane, a.scales + max(row, 0), row >= 0 ? 4u : 0u);
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

// Eight elements of a row of T, times f, as fp16 pairs (0, 4) (1, 5) (2, 6) (3, 7).
template <typename T>
__device__ __forceinline__ uint4 eight_of(uint4 x, float f) {
    float2 v[4] = {Half16<T>::unpack(x.x), Half16<T>::unpack(x.y), Half16<T>::unpack(x.z), Half16<T>::unpack(x.w)};
    return make_uint4(Half16<__half>::pack(v[0].x * f, v[2].x * f), Half16<__half>::pack(v[0].y * f, v[2].y * f),
                      Half16<__half>::pack(v[1].x * f, v[3].x * f), Half16<__half>::pack(v[1].y * f, v[3].y * f));
}

// Q of n-tile n as its B operand will have it: word w has the elements tig D /
// 4 + 8 w ... of row 8 n + g.
template <int D>
__device__ __forceinline__ void load_q(const AttnArgs& a, const PagedSeq& seq, const Item& it, int n, int lane,
                                       uint4 (&q)[D / 32]) {
    const int g = lane >> 2, tig = lane & 3;
    const int row = it.row0 + min(8 * n + g, it.rows - 1), token = a.by_g(row);
    const uint4* at = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) +
                                                     (long long)(seq.row0 + token) * a.ldq +
                                                     (it.kvh * a.G + row - token * a.G) * D + tig * (D / 4));
#pragma unroll
    for (int w = 0; w < D / 32; ++w) q[w] = __ldg(at + w);
}
// The largest finite magnitude of these, over the warp, as the bits of a float.
template <typename T, int W>
__device__ __forceinline__ uint32_t largest_of(const uint4 (&q)[W]) {
    uint32_t top = 0;
#pragma unroll
    for (int w = 0; w < W; ++w)
        for (const uint32_t x : {q[w].x, q[w].y, q[w].z, q[w].w}) {
            const float2 v = Half16<T>::unpack(x);
            const uint32_t b0 = __float_as_uint(v.x) & 0x7fffffffu, b1 = __float_as_uint(v.y) & 0x7fffffffu;
            top = max(top, max(b0 < 0x7f800000u ? b0 : 0u, b1 < 0x7f800000u ? b1 : 0u));
        }
    return __reduce_max_sync(0xffffffffu, top);
}
// The power of two that brings it to 2^14: -113 for the largest numbers of bf16, at
// most 126 (rows below 2^-112), so that it and its inverse are normal numbers.
__device__ __forceinline__ int shift_of(uint32_t top) { return min(14 - ((int)(top >> 23) - 127), 126); }
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((127 + e) << 23); }

// The tiles [j0, j1) of an item, 32 keys of each by every warp.
template <typename T, int D, int RB>
__device__ __forceinline__ void consume(const AttnArgs& a, const PagedSeq& seq, const Item& it, const Part& part, int warp,
                                        int lane, uint32_t base, RowState<D, RB>& s) {
    using L = Layout<D, RB>;
    constexpr int KC = D / 16, W = D / 32;  // MMA steps of a score; words of a thread's K row
    constexpr uint32_t ROW = D / 2;
    const int g = lane >> 2, tig = lane & 3;
    const uint32_t ring = base + warp * L::kRing;
    // where key `lane` of this warp in tile j is; its copies into stage n
    const int* table = a.b.table + (size_t)part.s * a.b.table_stride;
    auto look = [&](int j) {
        const int p = tile_key<kKeys>(it, j) + warp * kWarpKeys + lane;
        return page_of(a.b, table, p, j < part.j1 && item_sees(it, p));
    };
    auto get = [&](PageOf at, uint32_t n) {
        fetch<D>(a, pool_row(a.b, it.kvh, at, a.err), lane, ring + n * L::kStage);
        cp_async_commit();
    };
    PageOf ahead[kStages];
#pragma unroll
    for (int i = 0; i < kStages; ++i) ahead[i] = look(part.j0 + i);
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) get(ahead[i], i);
    PageOf next = ahead[kStages - 1];
    const Masks mk = make_masks();
    uint4 qb[W];
    int shift;
    const uint32_t q_at = base + L::kQAt + lane * 16, top_at = base + L::kQAt + RB * W * 512;
    if (L::kSharedQ) {
        uint32_t top = 0;
        for (int n = warp; n < RB; n += kWarps) {
            load_q<D>(a, seq, it, n, lane, qb);
            top = max(top, largest_of<T, W>(qb));
        }
        if (lane == 0) asm volatile("st.shared.b32 [%0], %1;" ::"r"(top_at + 4 * warp), "r"(top) : "memory");
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = max(top, ld_shared1(top_at + 4 * w));
        shift = shift_of(top);
        for (int n = warp; n < RB; n += kWarps) {
            load_q<D>(a, seq, it, n, lane, qb);
#pragma unroll
            for (int w = 0; w < W; ++w) st_shared(q_at + (n * W + w) * 512, eight_of<T>(qb[w], power_of_two(shift)));
        }
        __syncthreads();
    } else {
        load_q<D>(a, seq, it, 0, lane, qb);
        shift = shift_of(largest_of<T, W>(qb));
#pragma unroll
        for (int w = 0; w < W; ++w) qb[w] = eight_of<T>(qb[w], power_of_two(shift));
    }
    const float back = a.scale_log2 * power_of_two(-shift);
    // rows 8 n + 2 tig + e that have an m (bit 2 n + e), and those that need one
    unsigned set = 0, need = 0;
#pragma unroll
    for (int n = 0; n < RB; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            s.m[n][e] = 0.0f;
            s.l[n][e] = 0.0f;
            if (8 * n + 2 * tig + e < it.rows) need |= 1u << (2 * n + e);
        }
#pragma unroll
        for (int b = 0; b < KC; ++b) s.acc[n][b][0] = s.acc[n][b][1] = s.acc[n][b][2] = s.acc[n][b][3] = 0.0f;
    }
    bool unset = true;
    // tiles of which every row sees all keys of this warp: not among the first ones that stay visible, not before the
    // last row's window, not past the first row
    const int first_key = (it.lo_tile - it.sink_tiles) * kKeys + warp * kWarpKeys;  // of tile 0, behind those
    const int whole_lo = max(it.sink_tiles, a.window > 0 ? (max(it.pos_last - a.window + 1 - first_key, 0) + kKeys - 1) / kKeys : 0);
    const int whole_hi = it.pos_first + 1 - kWarpKeys >= first_key ? (it.pos_first + 1 - kWarpKeys - first_key) / kKeys + 1 : 0;
    const unsigned whole_n = (unsigned)max(whole_hi - whole_lo, 0);
    // K rows g and g + 8 of a group of keys, the V rows of the contraction's order, their scale words
    const int kg = key_of(g), kt0 = key_of(2 * tig), kt1 = key_of(2 * tig + 1);  // (of r + 8: 8 more)
    const uint32_t k_at = kg * ROW + tig * (D / 8);
    const uint32_t v_at0 = (uint32_t)L::kCodes + kt0 * ROW + g * (D / 16), v_at1 = v_at0 + (kt1 - kt0) * ROW;
    const uint32_t s_at = 2 * L::kCodes;
    uint32_t now = 0;  // the stage of tile j
#pragma unroll 1
    for (int j = part.j0; j < part.j1; ++j) {
        get(next, now == 0 ? kStages - 1 : now - 1);
        next = look(j + kStages);
        cp_async_wait<kStages - 1>();
        __syncwarp();
        const uint32_t stage = ring + now * L::kStage;
        const bool whole_tile = (unsigned)(j - whole_lo) < whole_n;
        const int k0 = tile_key<kKeys>(it, j) + warp * kWarpKeys;
        // keys of this warp that some row sees
        if (whole_tile || (k0 < it.hi && (k0 + kWarpKeys > it.lo || k0 < it.sink_end))) {
            // what is lane's of group i is key 16 i + kg + 8 h
            uint32_t word[kGroups][2];
            float sc[kGroups][RB][4];
#pragma unroll
            for (int i = 0; i < kGroups; ++i) {
                uint32_t ka[2][4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    word[i][h] = ld_shared1(stage + s_at + 4 * (16 * i + 8 * h) + 4 * kg);
                    const uint32_t at = stage + k_at + (16 * i + 8 * h) * ROW;
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
                const Zeros z0 = make_zeros(__byte_perm(word[i][0], word[i][0], 0x1010), mk);
                const Zeros z1 = make_zeros(__byte_perm(word[i][1], word[i][1], 0x1010), mk);
#pragma unroll
                for (int n = 0; n < RB; ++n) sc[i][n][0] = sc[i][n][1] = sc[i][n][2] = sc[i][n][3] = 0.0f;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    uint32_t x[4], y[4];
                    whole(ka[0][w], z0, mk, x);
                    whole(ka[1][w], z1, mk, y);
#pragma unroll
                    for (int n = 0; n < RB; ++n) {  // (n-tiles without rows too: asking costs as much)
                        const uint4 q = L::kSharedQ ? ld_shared(q_at + (n * W + w) * 512) : qb[w];
                        mma(sc[i][n], x[0], y[0], x[1], y[1], q.x, q.y);
                        mma(sc[i][n], x[2], y[2], x[3], y[3], q.z, q.w);
                    }
                }
            }
            // a score in base 2 is sc f
            float f[kGroups][2], vs[kGroups][2];
#pragma unroll
            for (int i = 0; i < kGroups; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    f[i][h] = back * scale4(word[i][h]);
                    vs[i][h] = __uint_as_float(word[i][h] & 0xfff00000u);
                }
            if (!whole_tile) {
                bool none[kGroups][2];  // a K vector of NaN: of the rows that see it alone
#pragma unroll
                for (int i = 0; i < kGroups; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        none[i][h] = !(f[i][h] < INFINITY);
                        f[i][h] = none[i][h] ? 1.0f : fmaxf(f[i][h], 1e-37f);  // -infinity times it is -infinity
                    }
#pragma unroll
                for (int n = 0; n < RB; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int r = 8 * n + 2 * tig + e, pos = r < it.rows ? row_pos(seq, a.by_g(it.row0 + r)) : -1;
#pragma unroll
                        for (int i = 0; i < kGroups; ++i)
#pragma unroll
                            for (int h = 0; h < 2; ++h)
                            {
                                float& x = sc[i][n][2 * h + e];
                                if (none[i][h]) x = __int_as_float(0x7fffffff);
                                if (!row_sees(a, pos, k0 + 16 * i + 8 * h + kg)) x = -INFINITY;
                            }
                    }
            }
            // weights under the m of the keys before; where a row's do not fit (and for its first keys), its m
            // moves and they are computed again.  A row's m depends on its own weights alone.
            float p[kGroups][RB][4], w[kGroups][RB][4];
            auto weights = [&]() {
#pragma unroll
                for (int i = 0; i < kGroups; ++i)
#pragma unroll
                    for (int n = 0; n < RB; ++n)
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            p[i][n][x] = ex2(fmaf(sc[i][n][x], f[i][x >> 1], -s.m[n][x & 1]));
                            w[i][n][x] = p[i][n][x] * vs[i][x >> 1];
                        }
            };
            weights();
            float most_p = 0.0f, most_w = 0.0f;
#pragma unroll
            for (int i = 0; i < kGroups; ++i)
#pragma unroll
                for (int n = 0; n < RB; ++n)
#pragma unroll
                    for (int x = 0; x < 4; x += 2) {
                        most_p = max_nan(most_p, p[i][n][x], p[i][n][x + 1]);
                        most_w = max_nan(most_w, w[i][n][x], w[i][n][x + 1]);
                    }
            if (unset || !__all_sync(0xffffffffu, most_w <= kMostWeight && most_p <= kMostSingle)) {
#pragma unroll
                for (int i = 0; i < kGroups; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        // a V vector of NaN: rows that see it have no result
                        const bool none = !(vs[i][h] < INFINITY);
                        if (__any_sync(0xffffffffu, none)) {
#pragma unroll
                            for (int n = 0; n < RB; ++n)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    bool hit = none && sc[i][n][2 * h + e] != -INFINITY;
#pragma unroll
                                    for (int o = 4; o < 32; o <<= 1) hit |= __shfl_xor_sync(0xffffffffu, (int)hit, o) != 0;
                                    if (hit)
#pragma unroll
                                        for (int b = 0; b < KC; ++b)
                                            s.acc[n][b][e] = s.acc[n][b][2 + e] = __int_as_float(0x7fffffff);
                                }
                        }
                        if (none) vs[i][h] = 0.0f;
                    }
#pragma unroll
                for (int n = 0; n < RB; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float top = -INFINITY, high_w = 0.0f, high_p = 0.0f;
#pragma unroll
                        for (int i = 0; i < kGroups; ++i)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const float log = (float)((int)(__float_as_uint(vs[i][h]) >> 23) - 127);
                                top = fmaxf(top, fmaf(sc[i][n][2 * h + e], f[i][h], fmaxf(log, kLeastLog) - kUp));
                                high_w = fmaxf(high_w, w[i][n][2 * h + e]);
                                high_p = fmaxf(high_p, p[i][n][2 * h + e]);
                            }
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) {
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                            high_w = fmaxf(high_w, __shfl_xor_sync(0xffffffffu, high_w, o));
                            high_p = fmaxf(high_p, __shfl_xor_sync(0xffffffffu, high_p, o));
                        }
                        const unsigned bit = 1u << (2 * n + e);
                        if (set & bit ? high_w > kMostWeight || high_p > kMostSingle : top != -INFINITY) {
                            const float down = set & bit ? s.m[n][e] - top : -INFINITY, x = ex2(down);
                            set |= bit;
                            s.m[n][e] = top;
                            s.l[n][e] = add_lowered(0.0f, s.l[n][e], down);
#pragma unroll
                            for (int b = 0; b < KC; ++b) {
                                s.acc[n][b][e] *= x;
                                s.acc[n][b][2 + e] *= x;
                            }
                        }
                    }
                unset = __any_sync(0xffffffffu, need & ~set);
                weights();
            }
#pragma unroll
            for (int i = 0; i < kGroups; ++i) {
                uint32_t pb[RB][2];
#pragma unroll
                for (int n = 0; n < RB; ++n) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) s.l[n][e] += p[i][n][e] + p[i][n][2 + e];
                    pb[n][0] = transpose8(Half16<__half>::pack(w[i][n][0], w[i][n][1]));
                    pb[n][1] = transpose8(Half16<__half>::pack(w[i][n][2], w[i][n][3]));
                }
                // V^T: elements g D / 8 ... of keys 2 tig, + 1 and 2 tig + 8, + 9
                uint32_t va[4][D / 64];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const uint32_t at = stage + (x & 1 ? v_at1 : v_at0) + (16 * i + 8 * (x >> 1)) * ROW;
                    if (D == 128) {
                        const uint2 y = ld_shared2(at);
                        va[x][0] = y.x;
                        va[x][D / 64 - 1] = y.y;
                    } else {
                        va[x][0] = ld_shared1(at);
                    }
                }
                Zeros zv[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t at = stage + s_at + 4 * (16 * i + 8 * h);
                    zv[h] = make_zeros(__byte_perm(ld_shared1(at + 4 * kt0), ld_shared1(at + 4 * kt1), 0x7632), mk);
                }
#pragma unroll
                for (int q = 0; q < D / 64; ++q)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {  // elements 8 q + 4 half ... + 3 of both keys of a pair
                        const uint32_t sel = half ? 0x7632 : 0x5410;
                        uint32_t x[4], y[4];
                        whole(__byte_perm(va[0][q], va[1][q], sel), zv[0], mk, x);
                        whole(__byte_perm(va[2][q], va[3][q], sel), zv[1], mk, y);
#pragma unroll
                        for (int b = 0; b < 2; ++b)
#pragma unroll
                            for (int n = 0; n < RB; ++n)
                                mma(s.acc[n][4 * q + 2 * half + b], x[2 * b], x[2 * b + 1], y[2 * b], y[2 * b + 1],
                                    pb[n][0], pb[n][1]);
                    }
            }
        }
        __syncwarp();  // the stage is read
        now = now + 1 == kStages ? 0 : now + 1;
    }
    cp_async_wait<0>();
#pragma unroll
    for (int n = 0; n < RB; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) s.l[n][e] += __shfl_xor_sync(0xffffffffu, s.l[n][e], o);
#pragma unroll
    for (int x = 0; x < 2 * RB; ++x)
        if (!(set >> x & 1u)) s.m[x / 2][x & 1] = -INFINITY;
}

// Element 4 i of the stretch g of a row's D in a set: neighbours g for the
// writers' 16-byte stores, neighbours i a stretch's four elements.
template <int D>
__device__ __forceinline__ int set_at(int row, int i, int g) {
    return row * D + i * 32 + g * 4;
}

// A split item's result from its CTAs' slots, in order, by the last of them to
// arrive.
template <typename T, int D, int M>
__device__ __forceinline__ void join_item(const AttnArgs& a, const PagedSeq& seq, const Item& it, const Part& p, int tid) {
    // four elements of a row a thread, four CTAs' at once
    for (int x = tid; x < it.rows * (D / 4); x += kThreads) {
        const int r = x / (D / 4), d = 4 * (x % (D / 4));
        float top = -INFINITY, l = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int b = p.first; b <= p.last; b += 4) {
            float mb[4], lb[4], up = top;
            float4 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float* at = slot_of<M, D>(a, min(b + i, p.last), p.first);
                mb[i] = __ldcg(at + M * D + r);
                lb[i] = __ldcg(at + M * D + M + r);
                v[i] = __ldcg(reinterpret_cast<const float4*>(at + r * D + d));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (b + i > p.last) mb[i] = -INFINITY;
                up = fmaxf(up, mb[i]);
            }
            const float down = top == -INFINITY ? top : top - up, f = ex2(down);
            top = up;
            l = add_lowered(0.0f, l, down);
            o = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // (of a row whose scores are NaN, m is -infinity and l NaN)
                const float d = mb[i] == -INFINITY ? mb[i] : mb[i] - top, w = ex2(d);
                l = add_lowered(l, lb[i], d);
                o.x = fmaf(v[i].x, w, o.x);
                o.y = fmaf(v[i].y, w, o.y);
                o.z = fmaf(v[i].z, w, o.z);
                o.w = fmaf(v[i].w, w, o.w);
            }
        }
        write_pair<T, D>(a, seq, it.kvh, it.row0 + r, d, {top, l, o.x, o.y});
        write_pair<T, D>(a, seq, it.kvh, it.row0 + r, d + 2, {top, l, o.z, o.w});
    }
}

template <typename T, int D, int RB>
__global__ void __launch_bounds__(kThreads, (Layout<D, RB>::kPerSm)) paged4_attn(const __grid_constant__ AttnArgs a) {
    using L = Layout<D, RB>;
    constexpr int M = L::kRows;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int last_s;
    // out of a register that the compiler cannot see through: it would read the thread's number again and again
    int tid;
    asm volatile("mov.u32 %0, %%tid.x;" : "=r"(tid));
    const int warp = tid >> 5, lane = tid & 31, g = lane >> 2, tig = lane & 3;
    const uint32_t base = (smem_addr(smem) + 127u) & ~127u;
    const float* sets = reinterpret_cast<const float*>(smem + (base - smem_addr(smem)));
    const Place place = find_place<M, kKeys, kThreads>(a);
    pdl_launch_dependents();  // the tcgen05 kernel may take SMs as they become free
    if (place.s < 0) return;
    walk<M, kKeys, kLeast4>(a, place, [&](const PagedSeq& seq, const Item& it, const Part& p) {
        {
            RowState<D, RB> s;
            consume<T, D, RB>(a, seq, it, p, warp, lane, base, s);
            float* set = const_cast<float*>(sets) + warp * (L::kRing / 4);
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
        __syncthreads();
        // the warps' results, joined in order: four elements of a row a thread
        const bool split = p.first != p.last;
        float* slot = slot_of<M, D>(a, blockIdx.x, p.first);
        for (int x = tid; x < it.rows * (D / 4); x += kThreads) {
            const int r = x / (D / 4), i = x / 8 % (D / 32), gg = x % 8, d = gg * (D / 8) + 4 * i;
            float m[kWarps], top = -INFINITY, l = 0.0f;
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                m[w] = sets[w * (L::kRing / 4) + M * D + r];
                top = fmaxf(top, m[w]);
            }
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float* set = sets + w * (L::kRing / 4);
                const float d = m[w] == -INFINITY ? m[w] : m[w] - top, f = ex2(d);
                const float4 v = *reinterpret_cast<const float4*>(set + set_at<D>(r, i, gg));
                l = add_lowered(l, set[M * D + M + r], d);
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
        __syncthreads();  // the sets are free
        if (!split) return;
        if (tid == 0) {
            // the others' writes, ordered before by the barrier, become visible with this thread's fence
            __threadfence();
            const unsigned sh = 16u * (p.first & 1), n = (unsigned)(p.last - p.first + 1);
            unsigned* ticket = a.tickets + p.first / 2;
            last_s = (atomicAdd(ticket, 1u << sh) >> sh & 0xffffu) + 1u == n;
            if (last_s) atomicSub(ticket, n << sh);  // ready for the next call
            __threadfence();
        }
        __syncthreads();
        if (last_s) join_item<T, D, M>(a, seq, it, p, tid);
        __syncthreads();  // everyone has read last_s
    });
}

// CTAs of a launch at most.  Half a word of the tickets is an item's: it counts
// to the item's CTAs.
constexpr int kMost4Ctas = 1024;

template <typename T, int D, int RB>
int launch_rows(const AttnArgs& a, cudaStream_t st) {
    using L = Layout<D, RB>;
    static std::atomic<unsigned long long> set_on{0};
    if (int s = allow_smem(paged4_attn<T, D, RB>, (int)L::kBytes, set_on)) return s;
    // as many as the SMs hold at once and the workspace has slots for
    constexpr int room = (int)((kTcWorkspaceAt - kSlotsAt) / (2 * slot_floats<L::kRows, D>() * 4));
    static_assert(kMost4Ctas / 2 * 4 <= kSlotsAt, "the tickets must fit the workspace");
    const int ctas = std::min({sm_count() * L::kPerSm, room, kMost4Ctas});
    paged4_attn<T, D, RB><<<ctas, kThreads, L::kBytes, st>>>(a);
    INFERNT_CUDA_TRY(cudaGetLastError());
    return INFERNT_OK;
}

// rows: query rows of a KV head that most sequences have.  They make as few
// items as can be, of up to four n-tiles, and as many n-tiles in each: a
// part's rows cost their softmax whether they are there or not (40 rows as 24 and
// 16 take 40 us in the first of the cases above, as 32 and 8 they took 52 when they
// were 43).  rows may be 0: the kernel then has the sequences' error bits to set.
template <typename T, int D>
int launch(const AttnArgs& a, long long rows, cudaStream_t st) {
    const long long tiles = std::max(1ll, (rows + 7) / 8), items = (tiles + 3) / 4, each = (tiles + items - 1) / items;
    if (each <= 1) return launch_rows<T, D, 1>(a, st);
    if (each == 2) return launch_rows<T, D, 2>(a, st);
    if (each == 3) return launch_rows<T, D, 3>(a, st);
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
    if (int s = check_ragged_batch(op, batch)) return s;
    const infernt_paged_cache geometry = geometry4(*cache);
    const int D = cache->head_dim, G = nq / cache->num_kv_heads;
    // Sequences of up to most_rows query rows a KV head are bound by their keys,
    // longer ones by their products.  Where the batch's counts do not say that
    // all sequences are as long as the longest, each kernel takes its own.
    const long long most = (long long)batch->max_q_len * G, all = (long long)batch->num_rows * G;
    const bool chunks = most > most_rows(D), both = chunks && batch->num_rows < (long long)batch->num_seqs * batch->max_q_len;
    // of the kernels that run; the few-row kernel's sequences have most_rows at most
    const WorkBound long_rows = {all, kTcItemRows, kTcTileKeys},
                    few_rows = {std::min(all, (long long)batch->num_seqs * most_rows(D)), 8, kKeys},
                    first = chunks ? long_rows : few_rows;
    AttnArgs a;
    bool empty;
    if (int s = attention_args(op, out, ldo, q, ldq, nq, &geometry, batch, window, sinks, scale, lse, workspace, err,
                               {first, both ? few_rows : first}, &a, &empty))
        return s;
    if (empty) return INFERNT_OK;
    if (int s = check_device_pointer(op, "the scales", cache->scales)) return s;
    a.scales = cache->scales;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!chunks || both) {
        // rows of an item: those of the longest sequence, or, beside a chunk, what the others have on average
        long long rows = most;
        if (both) {
            a.max_rows = most_rows(D);
            rows = std::max(1, (batch->num_rows - batch->max_q_len + batch->num_seqs - 2) / std::max(1, batch->num_seqs - 1));
            rows *= a.G;
        }
        int s;
        if (cache->dtype == INFERNT_DTYPE_BF16)
            s = D == 64 ? launch<__nv_bfloat16, 64>(a, rows, st) : launch<__nv_bfloat16, 128>(a, rows, st);
        else
            s = D == 64 ? launch<__half, 64>(a, rows, st) : launch<__half, 128>(a, rows, st);
        if (s || !chunks) return s;
        a.min_rows = most_rows(D);
        a.max_rows = kMaxPositions;
    }
    return paged4_attention_tc(a, D, cache->dtype, both, st);
}
