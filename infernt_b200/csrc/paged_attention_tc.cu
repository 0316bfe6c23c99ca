// paged_attention_tc.cu — attention of chunks of new tokens over paged KV
// caches on the 5th-generation tensor cores (paged_attention.cu has the
// formulas and the kernel for single tokens).
//
// An item is 256 query rows (new token, head of the group) of a KV head, two
// row tiles A and B of 128, the M of the MMA; K and V arrive in tiles of 64
// keys.  Per tile i and row tile X:
//   S_X = Q_X K_i^T        A and B operands from shared memory, S in TMEM
//   P_X = 2^(S_X scale - m) one thread per row: S out of TMEM, P back into it
//                          in 16 bits
//   O_X += P_X V_i         A operand from TMEM, V as the pages hold it
// A group of MMAs ends 550 cycles after its last operand is read, so the
// products of a row tile must not wait for one another: each row tile has
// two score buffers of 64 columns, and while its threads work on one, S of
// the next tile goes into the other and P V of the one before is under way.
// (Tiles of 128 keys with one buffer: 4300 cycles a pair of 128 x 128 tiles,
// of which the products take 2048.  An MMA of 64 keys reads Q as often as one
// of 128 and takes 49 cycles instead of 32; two buffers are still the better
// deal.)  At head_dim 128, O and S fill the 512 columns and P lies over the
// half of its scores that has been read, so S of tile i + 2 waits for P V of
// tile i; at 64 it has columns of its own.
//
// Twelve warps: warp 0 loads K and V tiles page by page by TMA (a tensor map
// of the pool [page][KV head][position][dim]; a page that no row sees, or that
// the pool does not have, is a coordinate past its end and becomes zeros),
// warps 1 and 3 issue the MMAs of A and of B, warp 2 takes out of V what must
// not meet a probability of 0 (clean_rows), warps 4-7 and 8-11 hold the rows of
// A and B.  Of the 384 x 168
// registers of a launch the first four warps keep 88 a thread, the others
// take 208.
//
// The probabilities of a tile are computed with the m of the tiles before,
// with no search for their maximum: any m gives the same result, so long as
// the probabilities fit their 16 bits, and a tile whose sum is at most
// kMostSum does.  Where it is not (and for first keys and hidden ones) the
// tile is computed again with its own maximum, and O is rescaled if m moves: by
// more than kRescale, or at all after such a sum, so that the next tiles pass.
// P goes to TMEM eight columns at a time.
//
// 4096 tokens at 12288 positions (32/8 heads of 128, bf16): 555 us in bursts,
// 1238 TFLOP/s (636 us back to back, at the power limit).  What was tried stood
// beside 529 us, in bursts, at its time: 594 with the maximum searched beside
// the probabilities, 559 with P stored as a whole, 548 with the join of split
// items in line with the tiles, 622 with turns at the exponentials between the
// warps of a scheduler; a part of the 2^x on the FMA pipe instead of the special
// function unit changes nothing.  The call at a part's end that puts values back
// (restore_values) costs 15 of the 555 us by the registers around it, not by its
// own time (543 without it, all else the same; 565 in line, 575 with its
// arguments in registers).  The busiest unit is at 77 %, the special function
// unit at 64 %.
#include <cmath>
#include <cstdint>

#include <cudaTypedefs.h>

#include "paged4.cuh"
#include "paged_attention.cuh"
#include "tc_mma.cuh"
#include "warp_mma.cuh"

namespace infernt {

void* tensor_map_encoder();  // bgemm.cu

namespace {

constexpr int kM = kTcItemRows;  // query rows of an item
constexpr int kN = kTcTileKeys;  // keys of a tile
constexpr int kThreadsTc = 384;
// Parts of a split item that are read at once (of pages of 4 bits, whose launch
// has more threads, one: ptxas has no registers for two).
template <bool FOUR>
constexpr int kJoin = FOUR ? 1 : 2;
constexpr int kRowThreads = 256;
constexpr uint32_t kBoxQ = 16384;  // 128 rows of 64 values: a swizzled operand block
constexpr uint32_t kBox = 8192;    // 64 rows: a block of chunk_at

// Shared memory: Q of both row tiles, then the stages of K and of V tiles,
// each of D / 64 blocks.
template <int D>
struct LayoutTc {
    static constexpr uint32_t kBlocks = D / 64;
    static constexpr uint32_t kTileQ = kBlocks * kBoxQ;
    static constexpr uint32_t kTile = kBlocks * kBox;
    static constexpr int kStages = 4;
    static constexpr uint32_t kQ = 0;
    static constexpr uint32_t kK = 2 * kTileQ;
    static constexpr uint32_t kV = kK + kStages * kTile;
    static constexpr uint32_t kBytes = kV + kStages * kTile + 1024;
    // Pages of 4 bits: rings of codes and scale words behind those, one for each half of K's and of V's tiles
    static constexpr uint32_t kCodes = kN / 2 * D / 2, kRaw = kCodes + kN / 2 * 4;
    static constexpr int kRaws = 3;
    static constexpr uint32_t kRawAt = kV + kStages * kTile;
    static constexpr uint32_t kBytes4 = kRawAt + 4 * kRaws * kRaw + 1024;
};

struct Barriers {
    uint64_t full_k[4], empty_k[4], full_v[4], clean_v[4], empty_v[4];
    uint64_t q[2];
    uint64_t s[2][2], p[2][2], o[2][2];  // [row tile][score buffer]
};

// Pairs of FP32 values, each lane rounded as the scalar operation.
using F2 = unsigned long long;
__device__ __forceinline__ F2 f2(float a, float b) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 un2(F2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// 16-byte chunk c of row r of a row tile's Q (and, at the end, its result) at
// `tile` in shared memory.
__device__ __forceinline__ uint32_t row_chunk(uint32_t tile, int r, int c) {
    return tile + (c >> 3) * kBoxQ + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// 32 columns of a result, the chunks from c on of row r.  FOUR: the columns
// come in the order of V's tiles (put4).
template <typename T, bool FOUR>
__device__ __forceinline__ void put_result(uint32_t tile, int r, int c, float (&o)[32], bool sees, float inv) {
    constexpr int at[8] = {0, FOUR ? 2 : 1, FOUR ? 4 : 2, FOUR ? 6 : 3, FOUR ? 1 : 4, FOUR ? 3 : 5, FOUR ? 5 : 6, 7};
#pragma unroll
    for (int e = 0; e < 32; ++e) o[e] = sees ? o[e] * inv : 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float* x = o + 8 * e;
        st_shared(row_chunk(tile, r, c + e),
                  make_uint4(Half16<T>::pack(x[at[0]], x[at[1]]), Half16<T>::pack(x[at[2]], x[at[3]]),
                             Half16<T>::pack(x[at[4]], x[at[5]]), Half16<T>::pack(x[at[6]], x[at[7]])));
    }
}

// The values that clean_rows took out of a part's tiles, added to O of the
// row at pos (a row of tm_o a lane) where the row sees them.
template <typename T, int D>
__device__ __noinline__ void restore_values(const AttnArgs& a, const Current& cur, int pos, uint32_t tm_o) {
    each_not_finite<T, D, kN>(a, cur, [&](int p, const T* v) {
        const bool sees = row_sees(a, pos, p);
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
            float o[32];
            uint32_t w[32];
            tmem_ld32(tm_o + 32 * c, o);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const uint32_t x = __ldg(reinterpret_cast<const uint32_t*>(v + 32 * c) + e);
                const float2 y = Half16<T>::unpack(x & Half16<T>::not_finite(x));
                w[2 * e] = __float_as_uint(sees ? o[2 * e] + y.x : o[2 * e]);
                w[2 * e + 1] = __float_as_uint(sees ? o[2 * e + 1] + y.y : o[2 * e + 1]);
            }
            tmem_st32(tm_o + 32 * c, w);
            tmem_st_wait();
        }
    });
}

// ------------------------------------------------- pages of 4 bits
// The tiles are the same, in 16 bits, but for how they get there: four warps
// more make them out of codes (paged4.cuh), the halves of K's by warps 12 and
// 13, of V's by 14 and 15.  Half a tile's codes and scale words come by
// cp.async, row by row, two tiles ahead of the one that the warp turns into
// values; the table's entries are loaded three ahead.  The values are numbers of
// T, so the products are those over 16-bit pages.  Eight values lie in the order
// in which they come out of a word, (0, 4) (1, 5) (2, 6) (3, 7): the row warps
// put Q into that order too, and take the result out of it.
// The 512 x 128 registers of a launch are 176 a thread of the row warps and 80
// of the others; some 130 bytes a thread are spilled.  4096 tokens at 12288
// positions, 32/8 heads of 128, bf16: 621 to 670 us in bursts, where 16-bit pages
// take 555 to 578 (the row warps have 32 registers less, joins read one part at
// a time).  Before: 1259 us with the first four warps' two
// idle ones in place of four more (a tile is 1600 instructions, one behind the
// other), 1931 as straight code for whole tiles (waiting for instructions),
// 705 with 64 registers, 889 with 48.
constexpr int kThreads4 = 512;
constexpr int kHalf = kN / 2;  // keys of a warp's half

template <int D>
struct Half4 {
    static constexpr int kPieces = D / 32;  // 16-byte pieces of a row's codes
    static constexpr int kRpi = 32 / kPieces, kRounds = kHalf / kRpi;  // rows at once, rounds
};

// The copies of half a tile, key `lane` at `at`: zeros (a scale of 0) for keys
// that no row sees, and for pages that the pool does not have.
template <int D>
__device__ __forceinline__ void fetch4(const AttnArgs& a, const Item& it, const void* pool, PageOf at, uint32_t raw) {
    using X = Half4<D>;
    const int lane = threadIdx.x & 31, own = pool_row(a.b, it.kvh, at, a.err);
    const char* codes = static_cast<const char*>(pool) + 16 * (lane % X::kPieces);
#pragma unroll
    for (int i = 0; i < X::kRounds; ++i) {
        const int row = __shfl_sync(0xffffffffu, own, i * X::kRpi + lane / X::kPieces);
        cp_async16(raw + 16 * lane + i * 512, codes + (size_t)max(row, 0) * (D / 2), row >= 0 ? 16u : 0u);
    }
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(raw + kHalf * (D / 2) + 4 * lane),
                 "l"(a.scales + max(own, 0)), "r"(own >= 0 ? 4u : 0u)
                 : "memory");
}
// The values of half a tile of codes, their scale words `shift` bits up in the
// pair's.  none: vectors of NaN become zeros.
template <typename T, int D>
__device__ __forceinline__ void put4(uint32_t raw, uint32_t tile, int shift, bool none, const Masks4& mk) {
    using X = Half4<D>;
    const int lane = threadIdx.x & 31, piece = lane % X::kPieces, r0 = lane / X::kPieces;
    const uint32_t words = raw + kHalf * (D / 2) + 4 * r0;
    // rows r0 + i kRpi: kRpi is 8 or 16, so the row's place in the swizzle stays
    const uint32_t dst = tile + (uint32_t)(piece >> 1) * kBox + r0 * 128, flip = (uint32_t)((4 * piece) & 7) ^ (r0 & 7);
    uint4 w = ld_shared(raw + 16 * lane);
#pragma unroll
    for (int i = 0; i < X::kRounds; ++i) {
        uint32_t x;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x) : "r"(words + 4 * i * X::kRpi) : "memory");
        const uint4 next = ld_shared(raw + 16 * lane + min(i + 1, X::kRounds - 1) * 512);
        x = (x >> shift) & 0xffffu;
        if (none && (x & 0x7f80u) == 0x7f80u) x = 0u;
        const uint32_t z2 = zeros4(x, mk), s2 = scale_pair4<T>(x);
        // pieces of the second block of columns begin with another word, or they would meet the first's in the banks
        const bool late = piece & 2;
        const uint32_t codes[4] = {late ? w.z : w.x, late ? w.w : w.y, late ? w.x : w.z, late ? w.y : w.w};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            uint32_t p[4];
            pairs4<T>(codes[c], z2, s2, mk, p);
            st_shared(dst + i * X::kRpi * 128 + ((flip ^ c ^ (late ? 2u : 0u)) << 4), make_uint4(p[0], p[1], p[2], p[3]));
        }
        w = next;
    }
    fence_proxy_async_smem();  // before the products read the tile
    __syncwarp();
}

// A warp's halves of all tiles of a CTA's parts.  V vectors of NaN in tiles
// that rows see in part become zeros, and *found_in the part.
template <typename T, int D>
__device__ __forceinline__ void produce4(const AttnArgs& a, const Place& place, uint32_t base, Barriers& bar, Current& cur,
                                         volatile int* found_in, bool is_v, int half, bool& ok) {
    using L = LayoutTc<D>;
    constexpr int ST = L::kStages, RW = L::kRaws;
    const int lane = threadIdx.x & 31, shift = is_v ? 16 : 0;
    const uint32_t raw = base + L::kRawAt + (2 * (int)is_v + half) * (RW * L::kRaw);
    const uint32_t tiles = base + (is_v ? L::kV : L::kK) + half * (kHalf * 128);
    const void* pool = is_v ? a.v : a.k;
    uint64_t* empty = is_v ? bar.empty_v : bar.empty_k;
    uint64_t* full = is_v ? bar.full_v : bar.full_k;
    const Masks4 mk = make_masks4<T>();
    uint32_t n = 0;  // tiles so far, over all parts
    walk<kM, kN>(a, place, [&](const PagedSeq&, const Item& it, const Part& part) {
        set_current(cur, it, part);
        const bool mixed = it.pos_first != it.pos_last;
        const int* table = a.b.table + (size_t)part.s * a.b.table_stride;
        auto look = [&](int j) {
            const int p = tile_key<kN>(it, j) + kHalf * half + lane;
            return page_of(a.b, table, p, j < part.j1 && item_sees(it, p));
        };
        PageOf pages[RW];
        __syncwarp();  // the raw tiles of the part before are read
#pragma unroll
        for (int i = 0; i < RW; ++i) pages[i] = look(part.j0 + i);
#pragma unroll
        for (int i = 0; i < RW - 1; ++i) {
            fetch4<D>(a, it, pool, pages[i], raw + i * L::kRaw);
            cp_async_commit();
        }
        PageOf ahead = pages[RW - 1];
        uint32_t at = 0, next = RW - 1;  // raw tiles: this one's, the one to be fetched
#pragma unroll 1
        for (int j = part.j0; j < part.j1; ++j, ++n) {
            const uint32_t st = n % ST, turn = (n / ST) & 1u;
            fetch4<D>(a, it, pool, ahead, raw + next * L::kRaw);
            cp_async_commit();
            ahead = look(j + RW);
            cp_async_wait<RW - 1>();
            __syncwarp();
            const bool partly = is_v && mixed && !seen_whole<kN>(a, it, tile_key<kN>(it, j));
            if (partly) {
                uint32_t x;
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x) : "r"(raw + at * L::kRaw + L::kCodes + 4 * lane) : "memory");
                if (__any_sync(0xffffffffu, (x >> 16 & 0x7f80u) == 0x7f80u)) {
                    if (lane == 0) *found_in = cur.no;
                    __threadfence_block();
                }
            }
            if (n >= ST) tc_wait_bar(&empty[st], turn ^ 1u, ok);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            put4<T, D>(raw + at * L::kRaw, tiles + st * L::kTile, shift, partly, mk);
            if (lane == 0) {
                mbar_arrive(&full[st]);
                if (is_v) mbar_arrive(&bar.clean_v[st]);
            }
            at = at + 1 == RW ? 0 : at + 1;
            next = next + 1 == RW ? 0 : next + 1;
        }
        cp_async_wait<0>();
    });
}

// As restore_values: rows that see a V vector of NaN have no result.
template <int D>
__device__ __noinline__ void restore_none(const AttnArgs& a, const Current& cur, int pos, uint32_t tm_o) {
    const int lane = threadIdx.x & 31;
    const Item& it = cur.it;
    bool hit = false;
    for (int j = cur.part.j0; j < cur.part.j1; ++j) {
        const int k0 = tile_key<kN>(it, j);
        if (seen_whole<kN>(a, it, k0)) continue;
        for (int h = 0; h < kN; h += 32) {
            const int p = k0 + h + lane, row = item_sees(it, p) ? pool_row(a.b, cur.part.s, it.kvh, p, nullptr) : -1;
            const bool none = row >= 0 && (__ldg(a.scales + row) >> 16 & 0x7f80u) == 0x7f80u;
            for (unsigned left = __ballot_sync(0xffffffffu, none); left; left &= left - 1)
                hit |= row_sees(a, pos, k0 + h + __ffs(left) - 1);
        }
    }
#pragma unroll 1
    for (int c = 0; c < D / 32; ++c) {
        float o[32];
        uint32_t w[32];
        tmem_ld32(tm_o + 32 * c, o);
#pragma unroll
        for (int e = 0; e < 32; ++e) w[e] = hit ? 0x7fffffffu : __float_as_uint(o[e]);
        tmem_st32(tm_o + 32 * c, w);
        tmem_st_wait();
    }
}

// Row ri (r of its row tile) of a split item, joined over its CTAs in order
// into shared memory: kJoin parts of 32 columns are read at once, since each
// read is a trip to L2.  A function of its own, so that its registers are not
// the tiles' (two parts: three spill, 528 -> 609 us in the case above).  Of CTA
// own, m, l and O are still in its registers and TMEM (O when it had tiles).
template <typename T, int D, bool FOUR>
__device__ __noinline__ void join_row(const AttnArgs& a, int first, int last, int ri, uint32_t tile, int r, bool sees,
                                      float* lse, int own, bool some, uint32_t tm_o, float m_own, float l_own) {
    float M = -INFINITY, l = 0.0f;
    for (int b = first; b <= last; b += 4) {
        float mb[4], lb[4], top = M;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float* p = slot_of<kM, D>(a, min(b + i, last), first) + kM * D + ri;
            mb[i] = b + i == own ? m_own : __ldcg(p);
            lb[i] = b + i == own ? l_own : __ldcg(p + kM);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (b + i > last) {
                mb[i] = -INFINITY;
                lb[i] = 0.0f;
            }
            top = fmaxf(top, mb[i]);
        }
        l *= M == -INFINITY ? 0.0f : ex2(M - top);
        M = top;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (FOUR || mb[i] != -INFINITY)  // (FOUR: the lse of a row whose scores are NaN is NaN, split or not)
                l = fmaf(lb[i], mb[i] == -INFINITY ? 0.0f : ex2(mb[i] - M), l);
    }
    if (lse) *lse = sees ? (M + log2f(l)) * kLn2 : -INFINITY;
    const float inv = 1.0f / l;
#pragma unroll 1
    for (int c = 0; c < D / 32; ++c) {
        float o[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = 0.0f;
#pragma unroll 1
        for (int b = first; b <= last; b += kJoin<FOUR>) {
            float mb[kJoin<FOUR>];
            float4 v[kJoin<FOUR>][8];
#pragma unroll
            for (int i = 0; i < kJoin<FOUR>; ++i) {
                if (b + i > last) break;
                if (b + i == own) {
                    mb[i] = m_own;
                    float t[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) t[e] = 0.0f;
                    if (some) tmem_ld32(tm_o + 32 * c, t);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[i][e] = make_float4(t[4 * e], t[4 * e + 1], t[4 * e + 2], t[4 * e + 3]);
                    continue;
                }
                const float* p = slot_of<kM, D>(a, b + i, first);
                mb[i] = __ldcg(p + kM * D + ri);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[i][e] = __ldcg(reinterpret_cast<const float4*>(p) + (8 * c + e) * kM + ri);
            }
#pragma unroll
            for (int i = 0; i < kJoin<FOUR>; ++i) {
                if (b + i > last) break;
                const float f = mb[i] == -INFINITY ? 0.0f : ex2(mb[i] - M);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    o[4 * e] = fmaf(v[i][e].x, f, o[4 * e]);
                    o[4 * e + 1] = fmaf(v[i][e].y, f, o[4 * e + 1]);
                    o[4 * e + 2] = fmaf(v[i][e].z, f, o[4 * e + 2]);
                    o[4 * e + 3] = fmaf(v[i][e].w, f, o[4 * e + 3]);
                }
            }
        }
        put_result<T, FOUR>(tile, r, 4 * c, o, sees, inv);
    }
}

// FOUR: pages of 4 bits
template <typename T, int D, bool FOUR>
__global__ void __launch_bounds__(FOUR ? kThreads4 : kThreadsTc, 1)
    paged_attn_tc(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap tm_k,
                  const __grid_constant__ CUtensorMap tm_v) {
    using L = LayoutTc<D>;
    constexpr int NB = (int)L::kBlocks, ST = L::kStages;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ Barriers bar;
    __shared__ uint32_t tmem_s;
    __shared__ int ok_s;
    __shared__ int last_s, early_s, found_s;  // found_s: the last part in which clean_rows found something
    constexpr int NT = FOUR ? kThreads4 : kThreadsTc;
    __shared__ Current cur_s[NT / 32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
    if (tid == 0) {
        for (int i = 0; i < ST; ++i) {
            mbar_init(&bar.full_k[i], FOUR ? 2 : 1);
            mbar_init(&bar.empty_k[i], 2);
            mbar_init(&bar.full_v[i], FOUR ? 2 : 1);
            mbar_init(&bar.clean_v[i], FOUR ? 2 : 1);
            mbar_init(&bar.empty_v[i], 2);
        }
        for (int x = 0; x < 2; ++x) {
            mbar_init(&bar.q[x], 128);
            for (int b = 0; b < 2; ++b) {
                mbar_init(&bar.s[x][b], 1);
                mbar_init(&bar.p[x][b], 128);
                mbar_init(&bar.o[x][b], 1);
            }
        }
        mbar_fence_init();
        ok_s = 1;
        found_s = 0;
        for (Current& c : cur_s) c.no = 0;
    }
    if (warp == 1) tmem_alloc(&tmem_s, 512);
    const Place place = find_place<kM, kN, NT>(a);  // its barriers publish the set-up
    tc_fence_after();
    __syncthreads();
    // TMEM columns: S of A at 0 and 64, of B at 128 and 192; O of A at 256, of B D further; P
    const uint32_t tmem = tmem_s;
    auto tm_score = [&](int x, int b) { return tmem + 128u * x + 64u * b; };
    auto tm_prob = [&](int x, int b) { return D == 128 ? tm_score(x, b) + 32u : tmem + 384u + 64u * x + 32u * b; };
    auto tm_out = [&](int x) { return tmem + 256u + (uint32_t)D * x; };
    bool ok = true;
    if (FOUR && warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 80;" ::: "memory");
        if (place.s >= 0) produce4<T, D>(a, place, base, bar, cur_s[warp], &found_s, warp >= 14, warp & 1, ok);
    } else if (warp < 4) {
        if (FOUR)
            asm volatile("setmaxnreg.dec.sync.aligned.u32 80;" ::: "memory");
        else
            asm volatile("setmaxnreg.dec.sync.aligned.u32 88;" ::: "memory");
        if (!FOUR && warp == 0 && place.s >= 0) {
            // ---- K and V tiles.  n: tiles so far, over all parts.
            uint32_t n = 0;
            const int ps = a.b.page_size, per_tile = ps < kN ? kN / ps : 1, box_rows = ps < kN ? ps : kN;
            const int run = 32 / per_tile;  // tiles of a look-up
            walk<kM, kN>(a, place, [&](const PagedSeq&, const Item& it, const Part& part) {
                int2 boxes = {};
                for (int j = part.j0, k = run; j < part.j1; ++j, ++n) {
                    const int st = (int)(n % ST);
                    const uint32_t turn = (n / ST) & 1u;
                    if (k == run) {
                        boxes = look_up<kN>(a, it, part, j, per_tile, box_rows);
                        k = 0;
                    }
                    const int page = __shfl_sync(0xffffffffu, boxes.x, k * per_tile + lane),
                              row = __shfl_sync(0xffffffffu, boxes.y, k * per_tile + lane);
                    ++k;
                    if (n >= ST) tc_wait_bar(&bar.empty_k[st], turn ^ 1u, ok);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) return;
                    if (lane == 0) mbar_arrive_expect_tx(&bar.full_k[st], L::kTile);
                    __syncwarp();
                    if (lane < per_tile)
#pragma unroll
                        for (int b = 0; b < NB; ++b)
                            tma_load_4d(base + L::kK + st * L::kTile + b * kBox + lane * box_rows * 128, &tm_k, 64 * b, row,
                                        it.kvh, page, &bar.full_k[st]);
                    if (n >= ST) tc_wait_bar(&bar.empty_v[st], turn ^ 1u, ok);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) return;
                    if (lane == 0) mbar_arrive_expect_tx(&bar.full_v[st], L::kTile);
                    __syncwarp();
                    if (lane < per_tile)
#pragma unroll
                        for (int b = 0; b < NB; ++b)
                            tma_load_4d(base + L::kV + st * L::kTile + b * kBox + lane * box_rows * 128, &tm_v, 64 * b, row,
                                        it.kvh, page, &bar.full_v[st]);
                }
            });
        } else if ((warp == 1 || warp == 3) && place.s >= 0) {
            // ---- the MMAs of row tile x, issued by one lane.  n: key tiles so far, nx: those of
            // this row tile.  Each row tile has a warp of its own, so that neither waits for the
            // other's probabilities.
            const int x = warp >> 1;
            uint32_t n = 0, nx = 0, parts = 0;
            const uint32_t id_s = tc_instr(Half16<T>::kBf16, false, kN), id_o = tc_instr(Half16<T>::kBf16, true, D);
            const uint64_t qd = tc_desc_k(base + L::kQ + x * L::kTileQ);
            const bool leader = tc_elect();
            // S of key tile m into buffer b
            auto scores = [&](uint32_t m, uint32_t b) {
                const uint32_t st = m % ST;
                const uint64_t k = tc_desc_k(base + L::kK + st * L::kTile);
                tc_fence_after();
#pragma unroll
                for (uint32_t kk = 0; kk < D / 16; ++kk) {
                    // 32 bytes a step within a block of 64 columns
                    const uint32_t c = kk >> 2, r = 2 * (kk & 3);
                    tc_mma_ss(tm_score(x, b), qd + c * (kBoxQ >> 4) + r, k + c * (kBox >> 4) + r, id_s, kk);
                }
                tc_commit_to(&bar.s[x][b]);
                tc_commit_to(&bar.empty_k[st]);
            };
            walk<kM, kN>(a, place, [&](const PagedSeq&, const Item& it, const Part& part) {
                const int tiles = part.j1 - part.j0;
                if (leader && tiles > 0 && ok) {
                    if (it.rows <= 128 * x) {
                        // no such rows: the stages go back unread
#pragma unroll 1
                        for (int j = 0; j < tiles; ++j, ++n) {
                            const uint32_t st = n % ST, turn = (n / ST) & 1u;
                            tc_wait_bar(&bar.full_k[st], turn, ok);
                            mbar_arrive(&bar.empty_k[st]);
                            tc_wait_bar(&bar.clean_v[st], turn, ok);
                            mbar_arrive(&bar.empty_v[st]);
                        }
                    } else {
                        tc_wait_bar(&bar.q[x], parts++ & 1u, ok);
                        // round i: P V of tile i - 2 and S of tile i.  At head_dim 128 S goes over
                        // P's columns, after P V; at 64 S, for which rows wait, goes first.
#pragma unroll 1
                        for (int i = 0; i < tiles + 2 && ok; ++i) {
                            const uint32_t b = (nx + i) & 1u, turn = ((nx + i - 2) >> 1) & 1u, m = n + i - 2;
                            if (i >= 2) tc_wait_bar(&bar.p[x][b], turn, ok);
                            if (D == 64 && i < tiles) {
                                tc_wait_bar(&bar.full_k[(n + i) % ST], ((n + i) / ST) & 1u, ok);
                                if (!ok) break;
                                scores(n + i, b);
                            }
                            if (i >= 2) {
                                const uint32_t st = m % ST;
                                const uint64_t v = tc_desc_mn(base + L::kV + st * L::kTile, kBox);
                                tc_wait_bar(&bar.full_v[st], (m / ST) & 1u, ok);
                                tc_wait_bar(&bar.clean_v[st], (m / ST) & 1u, ok);
                                if (!ok) break;
                                tc_fence_after();
#pragma unroll
                                for (uint32_t kk = 0; kk < kN / 16; ++kk)
                                    tc_mma_ts(tm_out(x), tm_prob(x, b) + 8u * kk, v + kk * (2048u >> 4), id_o,
                                              (uint32_t)(i - 2) | kk);
                                tc_commit_to(&bar.o[x][b]);
                                tc_commit_to(&bar.empty_v[st]);
                            }
                            if (D == 128 && i < tiles) {
                                tc_wait_bar(&bar.full_k[(n + i) % ST], ((n + i) / ST) & 1u, ok);
                                if (i >= 2) tc_wait_bar(&bar.o[x][b], turn, ok);
                                if (!ok) break;
                                scores(n + i, b);
                            }
                        }
                        n += tiles;
                        nx += tiles;
                    }
                }
                __syncwarp();
            });
        } else if (!FOUR && warp == 2 && place.s >= 0) {
            // ---- what of V must not meet a probability of 0 becomes zeros
            uint32_t n = 0;
            walk<kM, kN>(a, place, [&](const PagedSeq&, const Item& it, const Part& part) {
                set_current(cur_s[2], it, part);
                const bool mixed = it.pos_first != it.pos_last;
                for (int j = part.j0; j < part.j1; ++j, ++n) {
                    const int k0 = tile_key<kN>(it, j);
                    const uint32_t st = n % ST;
                    tc_wait_bar(&bar.full_v[st], (n / ST) & 1u, ok);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) return;
                    if (!seen_whole<kN>(a, it, k0) && (mixed || has_hidden<kN>(it, k0)))
                        clean_rows<T, D, kN>(cur_s[2], k0, base + L::kV + st * L::kTile, 0, mixed, &found_s);
                    if (lane == 0) mbar_arrive(&bar.clean_v[st]);
                }
            });
        }
    } else {
        if (FOUR)
            asm volatile("setmaxnreg.inc.sync.aligned.u32 176;" ::: "memory");
        else
            asm volatile("setmaxnreg.inc.sync.aligned.u32 208;" ::: "memory");
        if (place.s >= 0) {
            // ---- the rows: thread = TMEM lane r of row tile x
            const int x = (warp - 4) >> 2, quarter = warp & 3, r = 32 * quarter + lane;
            const uint32_t lanes = (uint32_t)(32 * quarter) << 16;
            const uint32_t tm_ox = tm_out(x) + lanes;
            const float sc = a.scale_log2;
            const F2 sc2 = f2(sc, sc);
            constexpr int CH = D / 8, RPI = 32 / CH, LI = 32 / RPI;  // 16-byte chunks of a row, rows at once, rounds
            const int ch = lane % CH;
            const uint32_t own = base + L::kQ + x * L::kTileQ;  // the row tile's Q
            uint32_t n = 0;  // key tiles of this row tile so far
            walk<kM, kN>(a, place, [&](const PagedSeq& seq, const Item& it, const Part& part) {
                set_current(cur_s[warp], it, part);
                // A wait that runs out ends the work on the scores, but not the barriers
                // that the threads of both row tiles meet at.
                const int rows_x = it.rows - 128 * x;  // rows of this tile (of 128)
                const int row = it.row0 + 128 * x + r;
                const bool mine = r < rows_x;
                const int token = mine ? a.by_g(row) : 0, pos = mine ? row_pos(seq, token) : -1;
                float m = -INFINITY, l = 0.0f;  // m in base 2
                bool settled = false;           // every row of the warp has an m
                unsigned taken = 0;
                const bool split = part.first != part.last, some = part.j0 < part.j1 && rows_x > 0;
                if (rows_x > 0 && part.j0 < part.j1) {
                    // Q rows of this warp: D / 8 lanes of 16 bytes a row, eight rounds in flight
                    {
#pragma unroll
                        for (int i0 = 0; i0 < LI; i0 += 8) {
                            uint4 w[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                // past the item's rows its last one again: no branch around a load
                                const int qrow =
                                    it.row0 + 128 * x + min(32 * quarter + (i0 + i) * RPI + lane / CH, rows_x - 1);
                                const int t = a.by_g(qrow);
                                w[i] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) +
                                                                            (long long)(seq.row0 + t) * a.ldq +
                                                                            (it.kvh * a.G + qrow - t * a.G) * D + ch * 8));
                            }
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                if (FOUR)  // (0, 1) (2, 3) (4, 5) (6, 7) -> (0, 4) (1, 5) (2, 6) (3, 7)
                                    w[i] = make_uint4(__byte_perm(w[i].x, w[i].z, 0x5410), __byte_perm(w[i].x, w[i].z, 0x7632),
                                                      __byte_perm(w[i].y, w[i].w, 0x5410), __byte_perm(w[i].y, w[i].w, 0x7632));
                                st_shared(row_chunk(own, 32 * quarter + (i0 + i) * RPI + lane / CH, ch), w[i]);
                            }
                        }
                        fence_proxy_async_smem();
                        mbar_arrive(&bar.q[x]);
                    }
#pragma unroll 1
                    for (int i = 0; i < part.j1 - part.j0; ++i, ++n) {
                        const int k0 = tile_key<kN>(it, part.j0 + i);
                        const uint32_t b = n & 1u;
                        tc_wait_bar(&bar.s[x][b], (n >> 1) & 1u, ok);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        tc_fence_after();
                        float sv[kN];
                        tmem_ld64(tm_score(x, b) + lanes, sv);
                        // keys that every row of the item sees need no mask
                        const bool whole = seen_whole<kN>(a, it, k0);
                        // at head_dim 64 P's columns are free once P V of two tiles ago is done
                        if (D == 64 && i >= 2) {
                            tc_wait_bar(&bar.o[x][b], ((n - 2) >> 1) & 1u, ok);
                            ok = __all_sync(0xffffffffu, ok);
                            if (!ok) break;
                            tc_fence_after();
                        }
                        const uint32_t tm_px = tm_prob(x, b) + lanes;
                        float lsum = 0.0f;
                        bool done = false;
                        if (whole && settled) {
                            // probabilities under the m of the tiles before, unless their sum
                            // says that a score has passed it by far
                            const F2 ref2 = f2(-m, -m);
                            F2 ls[2] = {f2(0.0f, 0.0f), f2(0.0f, 0.0f)};
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                uint32_t w[8];
#pragma unroll
                                for (int e = 8 * c; e < 8 * c + 8; ++e) {
                                    const F2 arg = fma2(f2(sv[2 * e], sv[2 * e + 1]), sc2, ref2);
                                    const float2 v = un2(arg);
                                    const float p0 = ex2(v.x), p1 = ex2(v.y);
                                    ls[e & 1] = add2(ls[e & 1], f2(p0, p1));
                                    w[e & 7] = Half16<T>::pack(p0, p1);
                                }
                                tmem_st8(tm_px + 8 * c, w);
                            }
                            const float2 v = un2(add2(ls[0], ls[1]));
                            lsum = v.x + v.y;
                            done = !__any_sync(0xffffffffu, !(lsum <= kMostSum<T>));
                        }
                        if (!done) {
                            tmem_st_wait();  // the stores that are made again
                            // a row's first keys, hidden keys, and keys whose maximum moves m
                            if (!whole) {
                                const int hi = pos - k0;
                                if (a.window == 0 || k0 > it.pos_last - a.window || k0 + kN <= a.sinks) {
#pragma unroll
                                    for (int e = 0; e < kN; ++e) sv[e] = e <= hi ? sv[e] : -INFINITY;
                                } else {
                                    const int lo = hi - a.window, sink = a.sinks - k0;
#pragma unroll
                                    for (int e = 0; e < kN; ++e) sv[e] = e <= hi && (e > lo || e < sink) ? sv[e] : -INFINITY;
                                }
                            }
                            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                            for (int e = 0; e < kN; e += 4) {
                                mx[0] = fmaxf(mx[0], fmaxf(sv[e], sv[e + 1]));
                                mx[1] = fmaxf(mx[1], fmaxf(sv[e + 2], sv[e + 3]));
                            }
                            const float top = fmaxf(mx[0], mx[1]) * sc - kShift<T>;
                            const bool grow = top > m + (lsum > kMostSum<T> ? 0.0f : kRescale);
                            if (i == 0) {
                                m = top;
                            } else if (__any_sync(0xffffffffu, grow)) {
                                // O must hold the products before it is rescaled
                                tc_wait_bar(&bar.o[x][b ^ 1], ((n - 1) >> 1) & 1u, ok);
                                ok = __all_sync(0xffffffffu, ok);
                                if (!ok) break;
                                tc_fence_after();
                                const float f = !grow ? 1.0f : m == -INFINITY ? 0.0f : ex2(m - top);
#pragma unroll 1
                                for (int c = 0; c < D / 32; ++c) {
                                    float o[32];
                                    uint32_t w[32];
                                    tmem_ld32(tm_ox + 32 * c, o);
#pragma unroll
                                    for (int e = 0; e < 32; ++e) w[e] = __float_as_uint(o[e] * f);
                                    tmem_st32(tm_ox + 32 * c, w);
                                }
                                tmem_st_wait();
                                if (grow) {
                                    l *= f;
                                    m = top;
                                }
                            }
                            settled = !__any_sync(0xffffffffu, m == -INFINITY);
                            const float ref = m == -INFINITY ? 0.0f : m;
                            float ls[2] = {0.0f, 0.0f};
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                uint32_t w[8];
#pragma unroll
                                for (int e = 8 * c; e < 8 * c + 8; ++e) {
                                    const float p0 = ex2(fmaf(sv[2 * e], sc, -ref)), p1 = ex2(fmaf(sv[2 * e + 1], sc, -ref));
                                    ls[0] += p0;
                                    ls[1] += p1;
                                    w[e & 7] = Half16<T>::pack(p0, p1);
                                }
                                tmem_st8(tm_px + 8 * c, w);
                            }
                            lsum = ls[0] + ls[1];
                        }
                        l += lsum;
                        tmem_st_wait();
                        tc_fence_before();
                        mbar_arrive(&bar.p[x][b]);
                    }
                    if (split && tid == 128) taken = tickets_taken(a, part);
                    tc_wait_bar(&bar.o[x][(n - 1) & 1u], ((n - 1) >> 1) & 1u, ok);
                    ok = __all_sync(0xffffffffu, ok);
                    tc_fence_after();
                    // written before V was ready for the products that this thread has waited for
                    if (__any_sync(0xffffffffu, *static_cast<volatile int*>(&found_s) >= cur_s[warp].no)) {
                        if constexpr (FOUR)
                            restore_none<D>(a, cur_s[warp], pos, tm_ox);
                        else
                            restore_values<T, D>(a, cur_s[warp], pos, tm_ox);
                    }
                }
                // ---- the part's result: straight to out, or through the slots
                const int ri = 128 * x + r;
                bool write = true, early = false;
                if (split) {
                    // where all others have arrived, this CTA's part stays where it is
                    if (tid == 128) {
                        early_s = taken == (unsigned)(part.last - part.first);
                        if (early_s) a.tickets[part.first] = 0u;  // ready for the next call
                    }
                    named_sync(1, kRowThreads);
                    early = early_s != 0;
                }
                if (split && !early) {
                    // columns [4 c, 4 c + 4) of row ri at float4 c kM + ri: neighbours in a row of threads
                    float* slot = slot_of<kM, D>(a, blockIdx.x, part.first);
                    if (rows_x > 0) {
#pragma unroll
                        for (int c = 0; c < D / 32; ++c) {
                            float o[32];
                            if (some) tmem_ld32(tm_ox + 32 * c, o);
                            if (mine)
#pragma unroll
                                for (int e = 0; e < 8; ++e)
                                    reinterpret_cast<float4*>(slot)[(8 * c + e) * kM + ri] =
                                        some ? make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3])
                                             : make_float4(0.f, 0.f, 0.f, 0.f);
                        }
                        if (mine) {
                            slot[kM * D + ri] = m;
                            slot[kM * D + kM + ri] = l;
                        }
                    }
                    named_sync(1, kRowThreads);
                    if (tid == 128) {
                        // the others' writes, ordered before by the barrier, become visible with this thread's fence
                        __threadfence();
                        unsigned* ticket = a.tickets + part.first;
                        last_s = atomicAdd(ticket, 1u) + 1u == (unsigned)(part.last - part.first + 1);
                        if (last_s) *ticket = 0u;  // ready for the next call
                        __threadfence();
                    }
                    named_sync(1, kRowThreads);
                    write = last_s != 0;
                }
                if (write && rows_x > 0) {
                    const bool sees = mine && pos >= 0;
                    float* lse = mine && a.lse ? a.lse + (long long)(seq.row0 + token) * a.nq + it.kvh * a.G + row -
                                                     token * a.G
                                               : nullptr;
                    // 32 columns at a time into the row tile's Q, which the products are done with
                    if (split) {
                        join_row<T, D, FOUR>(a, part.first, part.last, ri, own, r, sees, lse, early ? (int)blockIdx.x : -1, some,
                                              tm_ox, m, l);
                    } else {
                        if (lse) *lse = sees ? (m + log2f(l)) * kLn2 : -INFINITY;
                        const float inv = sees ? 1.0f / l : 0.0f;
#pragma unroll
                        for (int c = 0; c < D / 32; ++c) {
                            float o[32];
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = 0.0f;
                            if (some) tmem_ld32(tm_ox + 32 * c, o);
                            put_result<T, FOUR>(own, r, 4 * c, o, sees, inv);
                        }
                    }
                    __syncwarp();
                    // whole rows by D / 8 lanes each
#pragma unroll
                    for (int i = 0; i < LI; ++i) {
                        const int rr = 32 * quarter + i * RPI + lane / CH, orow = it.row0 + 128 * x + rr;
                        if (rr < rows_x) {
                            const int t = a.by_g(orow);
                            uint4 w;
                            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                         : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                                         : "r"(row_chunk(own, rr, ch))
                                         : "memory");
                            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + (long long)(seq.row0 + t) * a.ldo +
                                                      (it.kvh * a.G + orow - t * a.G) * D + ch * 8) = w;
                        }
                    }
                    __syncwarp();
                }
                // O, S and the slots' flag are read before the next part begins
                tc_fence_before();
                if (split) named_sync(1, kRowThreads);
            });
        }
    }
    if (!ok) atomicExch(&ok_s, 0);
    tc_fence_before();
    __syncthreads();
    if (!ok_s) {
        // a wait ran out: tell the host, and let copies in flight land
        if (tid == 0 && a.err) atomicOr(a.err, kErrWaitTimeout);
        const long long t0 = clock64();
        while (clock64() - t0 < 20000000ll) __nanosleep(1000);
    }
    if (warp == 1) {
        tc_fence_after();
        tmem_free(tmem, 512);
    }
    pdl_wait();  // this kernel's end is the call's end
}

template <typename T, int D, bool FOUR>
int launch_tc(const AttnArgs& args, bool after_other, cudaStream_t st) {
    using L = LayoutTc<D>;
    AttnArgs a = args;
    CUtensorMap mk = {}, mv = {};
    if (!FOUR) {
        if (int s = paged_pool_map(&mk, a, a.k, D, Half16<T>::kBf16, kN)) return s;
        if (int s = paged_pool_map(&mv, a, a.v, D, Half16<T>::kBf16, kN)) return s;
    }
    static std::atomic<unsigned long long> set_on{0};
    constexpr uint32_t bytes = FOUR ? L::kBytes4 : L::kBytes;
    if (int s = allow_smem(paged_attn_tc<T, D, FOUR>, (int)bytes, set_on)) return s;
    a.tickets += kTcWorkspaceAt / sizeof(unsigned);
    a.slots += kTcWorkspaceAt / sizeof(float);
    // one CTA an SM, as many as have slots in the workspace
    constexpr int most =
        (int)((kWorkspaceBytes - kTcWorkspaceAt - kSlotsAt) / (2 * slot_floats<kM, D>() * sizeof(float)));
    int ctas = sm_count();
    if (ctas > most) ctas = most;
    if (ctas > kMaxCtas) ctas = kMaxCtas;
    a.min_units = 8;
    // beside the end of the kernel launched just before, when that is the
    // other kernel of this call: neither touches what the other writes
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(FOUR ? kThreads4 : kThreadsTc);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = after_other ? 1 : 0;
    INFERNT_CUDA_TRY(cudaLaunchKernelEx(&cfg, paged_attn_tc<T, D, FOUR>, static_cast<const AttnArgs>(a),
                                        static_cast<const CUtensorMap>(mk), static_cast<const CUtensorMap>(mv)));
    return INFERNT_OK;
}

}  // namespace

// 64-key tiles are whole boxes: a tile is 64 / page_size pages, or a page is
// a whole number of tiles.
bool paged_attention_boxes(int page_size) {
    return page_size % 64 == 0 || (page_size >= 8 && 64 % page_size == 0);
}

int paged_pool_map(CUtensorMap* map, const AttnArgs& a, const void* pool, int D, bool bf16, int tile_keys) {
    auto fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(tensor_map_encoder());
    INFERNT_REQUIRE(fn, "paged_attention: cuTensorMapEncodeTiled is not available");
    const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)a.b.page_size, (cuuint64_t)a.b.nkv,
                                (cuuint64_t)a.b.num_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)D * 2, (cuuint64_t)a.b.page_size * D * 2,
                                   (cuuint64_t)a.b.nkv * a.b.page_size * D * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)(a.b.page_size < tile_keys ? a.b.page_size : tile_keys), 1, 1};
    const cuuint32_t one[4] = {1, 1, 1, 1};
    const CUresult r =
        fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(pool),
           dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    INFERNT_REQUIRE(r == CUDA_SUCCESS, "paged_attention: tensor map encoding failed (%d)", (int)r);
    return INFERNT_OK;
}

namespace {

template <bool FOUR>
int launch_kind(const AttnArgs& a, int head_dim, int dtype, bool after_other, cudaStream_t st) {
    if (dtype == INFERNT_DTYPE_BF16)
        return head_dim == 64 ? launch_tc<__nv_bfloat16, 64, FOUR>(a, after_other, st)
                              : launch_tc<__nv_bfloat16, 128, FOUR>(a, after_other, st);
    return head_dim == 64 ? launch_tc<__half, 64, FOUR>(a, after_other, st)
                          : launch_tc<__half, 128, FOUR>(a, after_other, st);
}

}  // namespace

int paged_attention_tc(const AttnArgs& a, int head_dim, int dtype, bool after_other, cudaStream_t st) {
    return launch_kind<false>(a, head_dim, dtype, after_other, st);
}
int paged4_attention_tc(const AttnArgs& a, int head_dim, int dtype, bool after_other, cudaStream_t st) {
    return launch_kind<true>(a, head_dim, dtype, after_other, st);
}

}  // namespace infernt
