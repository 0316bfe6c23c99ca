// paged_attention.cuh — what the two attention kernels over paged caches
// share: the query rows and keys of an item, the even split of the work over
// the CTAs, the partial results of split items, and values that are not finite.
#pragma once

#include <cuda.h>

#include "paged.cuh"

namespace infernt {

// Probabilities are rounded to V's type, since a matrix instruction takes both
// operands in one: half a step each, independent of one another, next to the
// half step of the result (bf16: 2.0e-3 to 2.3e-3 of the outputs in all, where
// FP32 probabilities leave 1.7e-3).  A split into three terms, as the decode
// attention over contiguous caches has it, would be three products P V where
// chunks are bound by the one.  The denominator sums them in FP32, unrounded.
//
// A row's probabilities are 2^(s - m), s in base 2; m is the largest score met
// less kShift, and moves when a score passes that one by kRescale.  The
// tcgen05 kernel takes a tile's probabilities under an older m as long as
// their sum is at most kMostSum.  Their common factor 2^kShift leaves out and
// lse as they are and puts the probabilities where their 16 bits hold them:
// bf16 as none above 1, so that sums of V's largest values stay finite; fp16
// where a weight of 2^-18 of the row's largest is still a normal number and
// what is lost of a smaller one is 2^-29 of the largest.  (At a shift of 0
// that was 2^-25, and 2^15 such keys were two half-steps of the result.  A
// higher shift lowers the sums that pass, and rows whose first tile shows them
// few keys compute more of the next ones twice: two chunks of 2039 tokens with
// a window of 1000, fp16, take 97 us at a shift of 5 and 2^15, 90 here.)
constexpr float kRescale = 8.0f;
template <typename T>
constexpr float kShift = Half16<T>::kBf16 ? -13.0f : 4.0f;
template <typename T>
constexpr float kMostSum = Half16<T>::kBf16 ? 1.0f : 65504.0f;

// Workspace: for each of the two kernels (a call may run both, the second
// while the first ends) the tickets of split items, then two slots of partial
// results for each CTA.
constexpr size_t kWorkspaceBytes = 64u << 20;
constexpr int kMaxCtas = 320;
constexpr size_t kSlotsAt = 2048;
constexpr size_t kTcWorkspaceAt = 24u << 20;

struct AttnArgs {
    PagedBatch b;
    const void* q;
    void* out;
    const void* k;
    const void* v;
    float* lse;
    long long ldq, ldo;
    int nq, G, window, sinks;
    FastDiv by_g;
    float scale, scale_log2;
    int min_rows, max_rows;  // a sequence of min_rows query rows or fewer, or more than max_rows, is another kernel's
    int min_units;           // least units of a CTA
    unsigned* tickets;       // [CTAs], zero between calls
    float* slots;
    unsigned* err;
};

// Whether tiles of 64 keys of such pages can be loaded as boxes of a tensor
// map, and that map of a pool: [page][KV head][position][dim], boxes of 64
// columns by the rows of a tile or of a page, 128-byte swizzle.
bool paged_attention_boxes(int page_size);
int paged_pool_map(CUtensorMap* map, const AttnArgs& a, const void* pool, int D, bool bf16, int tile_keys);

// The tcgen05 kernel (paged_attention_tc.cu): its items and tiles.
// after_other: the kernel launched just before on st is paged_attn.
constexpr int kTcItemRows = 256;
constexpr int kTcTileKeys = 64;
int paged_attention_tc(const AttnArgs& a, int head_dim, int dtype, bool after_other, cudaStream_t st);

// Rows [row0, row0 + rows) of the query rows of (sequence, KV head), and the
// keys that they see: [0, sink_end) and [lo, hi), as tiles of N keys.
struct Item {
    int kvh, row0, rows;
    int sink_end, lo, hi;  // hi: one past the last row's position (0 when it sees nothing)
    int lo_tile, sink_tiles, tiles;
    int pos_first, pos_last;
};

__device__ __forceinline__ int row_pos(const PagedSeq& s, int token) { return s.len - s.n_new + token; }

template <int M, int N>
__device__ __forceinline__ Item make_item(const AttnArgs& a, const PagedSeq& s, int kvh, int row0) {
    Item it;
    it.kvh = kvh;
    it.row0 = row0;
    it.rows = min(M, s.n_new * a.G - row0);
    it.pos_first = row_pos(s, a.by_g(row0));
    it.pos_last = row_pos(s, a.by_g(row0 + it.rows - 1));
    it.hi = max(0, it.pos_last + 1);
    it.lo = a.window > 0 ? max(0, it.pos_first - a.window + 1) : 0;
    it.sink_end = min(a.sinks, it.lo);
    it.lo_tile = it.lo / N;
    it.sink_tiles = min((it.sink_end + N - 1) / N, it.lo_tile);
    it.tiles = it.hi > 0 ? it.sink_tiles + (it.hi - 1) / N - it.lo_tile + 1 : 0;
    return it;
}

template <int N>
__device__ __forceinline__ int tile_key(const Item& it, int j) {
    return (j < it.sink_tiles ? j : it.lo_tile + (j - it.sink_tiles)) * N;
}

// ------------------------------------------------------------- schedule
// The work of a call is a line of units: for each sequence, each KV head,
// each item of M query rows, one unit per tile of N keys and kItemCost more
// for its start and end.  CTA b takes the units from b c to (b + 1) c, so the
// CTAs finish together whatever the lengths.  A border less than kLeast units
// from an end of an item moves to that end; an item with a border still
// inside is split: its CTAs leave partial results (two slots a CTA are
// enough: one for an item that began before it, one for an item that goes on
// after it), and the last of them to arrive joins them in CTA order.
// Lengths are device data; each CTA finds its own place by a scan over the
// sequences.
//
// In a split item border k c is inside when u0 + kLeast <= k c <= u1 -
// kLeast; the CTAs from the first such k, less one, to the last such k share
// it.  An item that is not split belongs to the CTA of the last border that
// is not past its first kLeast units.
constexpr int kItemCost = 3;
constexpr int kLeast = kItemCost + 2;

// Query rows of a KV head that are this kernel's.
__device__ __forceinline__ int rows_of(const AttnArgs& a, const PagedSeq& s) {
    const int rows = s.n_new * a.G;
    return rows > a.min_rows && rows <= a.max_rows ? rows : 0;
}

template <int M, int N>
__device__ __forceinline__ int item_units(const AttnArgs& a, const PagedSeq& s, int row0) {
    return row0 < rows_of(a, s) ? make_item<M, N>(a, s, 0, row0).tiles + kItemCost : 0;
}

// Units of one KV head of s, by a whole warp.
template <int M, int N>
__device__ __forceinline__ int head_units(const AttnArgs& a, const PagedSeq& s) {
    const int lane = threadIdx.x & 31;
    int n = 0;
    for (int row0 = lane * M; row0 < rows_of(a, s); row0 += 32 * M) n += item_units<M, N>(a, s, row0);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    return n;
}

__device__ __forceinline__ int warp_scan(int v) {  // inclusive
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += y;
    }
    return v;
}

// Row of the item that holds unit `rem` of a KV head; rem becomes the item's
// first unit.  By a whole warp.
template <int M, int N>
__device__ __forceinline__ int find_item(const AttnArgs& a, const PagedSeq& s, int& rem) {
    const int lane = threadIdx.x & 31;
    int before = 0;
    for (int row0 = 0;; row0 += 32 * M) {
        const int mine = item_units<M, N>(a, s, row0 + lane * M), sum = warp_scan(mine);
        const unsigned past = __ballot_sync(0xffffffffu, rem < before + sum);
        const int all = __shfl_sync(0xffffffffu, sum, 31);
        if (past || all == 0) {
            const int k = past ? __ffs(past) - 1 : 0;
            rem = before + __shfl_sync(0xffffffffu, sum - mine, k);
            return row0 + k * M;
        }
        before += all;
    }
}

// Units are counted in 32 bits, up to kMostUnits: the host refuses a call whose
// bound on them is larger.  Sequences that overlap (a q_start that descends
// somewhere, so that several hold the same rows) can have more; such a batch is
// not computed.
constexpr unsigned kMostUnits = 1u << 30;
__device__ __forceinline__ int add_units(int a, int b) { return (int)min((unsigned)a + (unsigned)b, kMostUnits); }

struct Place {
    int c;       // units of a CTA
    int before;  // units before sequence s
    int total;
    int s;       // the sequence that holds unit c x blockIdx.x; -1: nothing for this CTA
    PagedSeq seq;
    int per_head;  // units of one of its KV heads
};

// By all NT threads of the block.
template <int M, int N, int NT>
__device__ __forceinline__ Place find_place(const AttnArgs& a) {
    __shared__ int sums_s[NT / 32];
    __shared__ Place place_s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = a.b.num_seqs;
    // units of a KV head of sequence s (every thread its own); long ones by the whole warp
    auto units = [&](int s, PagedSeq& q) {
        q = {0, 0, 0};
        if (s < n) q = paged_seq(a.b, s, blockIdx.x == 0 ? a.err : nullptr);
        const bool many = rows_of(a, q) > 2 * M;
        int u = many ? 0 : item_units<M, N>(a, q, 0) + item_units<M, N>(a, q, M);
        for (unsigned left = __ballot_sync(0xffffffffu, many); left; left &= left - 1) {
            const int k = __ffs(left) - 1;
            const PagedSeq w = {__shfl_sync(0xffffffffu, q.row0, k), __shfl_sync(0xffffffffu, q.n_new, k),
                                __shfl_sync(0xffffffffu, q.len, k)};
            const int x = head_units<M, N>(a, w);
            if (lane == k) u = x;
        }
        return u;
    };
    // the sum of the values before this thread's, and of all of them
    auto scan = [&](int v, int& all) {
        int x = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x = add_units(x, y);
        }
        __syncthreads();
        if (lane == 31) sums_s[warp] = x;
        __syncthreads();
        int pre = x - v;  // (of no use once a sum is kMostUnits)
        all = 0;
#pragma unroll
        for (int w = 0; w < NT / 32; ++w) {
            if (w < warp) pre = add_units(pre, sums_s[w]);
            all = add_units(all, sums_s[w]);
        }
        return pre;
    };
    Place p = {0, 0, 0, -1, {0, 0, 0}, 0};
    if (tid == 0) place_s.s = -1;
    int before = 0;
    for (int base = 0; base < n; base += NT) {
        int all;
        p.per_head = units(base + tid, p.seq);
        before = add_units(p.total, scan(p.per_head * a.b.nkv, all));
        p.total = add_units(p.total, all);
    }
    if (p.total >= (int)kMostUnits) {
        if (tid == 0 && blockIdx.x == 0 && a.err) atomicOr(a.err, kErrBatch);
        p.total = 0;
    }
    p.c = max(a.min_units, (int)(((unsigned)p.total + gridDim.x - 1) / gridDim.x));
    const int at = p.c * (int)blockIdx.x;
    int sum = 0;
    if (at < p.total)
        for (int base = 0; base < n; base += NT) {
            if (n > NT) {  // a second pass; up to NT sequences are still in registers
                int all;
                p.per_head = units(base + tid, p.seq);
                before = sum + scan(p.per_head * a.b.nkv, all);
                sum += all;
            }
            if (before <= at && at - before < p.per_head * a.b.nkv) {
                p.before = before;
                p.s = base + tid;
                place_s = p;
            }
        }
    __syncthreads();
    return place_s;
}

// Part [j0, j1) of an item's tiles; first and last: the CTAs that share it.
struct Part {
    int s, j0, j1, first, last;
};

// f(sequence, item, part) for the parts of this CTA, by whole warps.
template <int M, int N, typename F>
__device__ __forceinline__ void walk(const AttnArgs& a, const Place& p, F f) {
    const int me = blockIdx.x, begin = p.c * me, end = min(p.c, p.total - begin) + begin;
    int at = begin, before = p.before, per_head = p.per_head;
    PagedSeq seq = p.seq;
    for (int s = p.s;;) {
        if (per_head > 0) {
            int kvh = (at - before) / per_head;
            int u0 = before + kvh * per_head, rem = at - u0;
            int row0 = find_item<M, N>(a, seq, rem);
            u0 += rem;
            while (kvh < a.b.nkv) {
                const Item it = make_item<M, N>(a, seq, kvh, row0);
                const int u1 = u0 + it.tiles + kItemCost;
                const bool more = begin > u0 && begin - u0 >= kLeast;  // it began in an earlier CTA
                if (end <= u0 || (end < u1 && end - u0 < kLeast && end < p.total)) return;
                if (!(begin > u0 && begin - u0 >= kLeast && u1 - begin < kLeast)) {
                    const bool cut = end < u1 && u1 - end >= kLeast;  // it goes on in a later one
                    Part part;
                    part.s = s;
                    part.j0 = more ? begin - u0 - kItemCost : 0;
                    part.j1 = cut ? end - u0 - kItemCost : it.tiles;
                    part.first = more ? (u0 + kLeast + p.c - 1) / p.c - 1 : me;
                    part.last = cut ? (u1 - kLeast) / p.c : me;
                    f(seq, it, part);
                }
                if (end < u1) return;
                u0 = u1;
                row0 += M;
                if (row0 >= seq.n_new * a.G) {
                    row0 = 0;
                    ++kvh;
                }
            }
            at = before += per_head * a.b.nkv;
        }
        if (at >= end || ++s >= a.b.num_seqs) return;
        seq = paged_seq(a.b, s, nullptr);
        per_head = head_units<M, N>(a, seq);
    }
}

// Tickets taken for a split item so far; what their CTAs wrote is visible to a
// thread that has met this one at a barrier.
__device__ __forceinline__ unsigned tickets_taken(const AttnArgs& a, const Part& part) {
    unsigned n;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(n) : "l"(a.tickets + part.first) : "memory");
    return n;
}

// Whether some row of the item sees key p.
__device__ __forceinline__ bool item_sees(const Item& it, int p) {
    return p < it.hi && (p >= it.lo || p < it.sink_end);
}

// Pages of the boxes of tiles j, j + 1, ... of a part, a box a lane (per_tile
// of them, a power of two, to a tile), so that a trip to the table serves up to
// 32 tiles: the box's page (a page past the pool when no row sees the box, or
// the pool does not have it), and its first row there.  (For the tcgen05
// kernel: 15 decodes and a chunk of 509 tokens on pages of 16, 97 us with a trip
// a tile, 95 so.  The other kernel's tiles take long enough to hide theirs.)
template <int N>
__device__ __forceinline__ int2 look_up(const AttnArgs& a, const Item& it, const Part& part, int j, int per_tile,
                                        int box_rows) {
    const int lane = threadIdx.x & 31, tile = j + lane / per_tile;
    int2 at = make_int2(a.b.num_pages, 0);
    if (tile < part.j1) {
        const int p0 = tile_key<N>(it, tile) + lane % per_tile * box_rows, pi = a.b.by_page(p0);
        at.y = p0 - pi * a.b.page_size;
        if (p0 < it.hi && (p0 + box_rows > it.lo || p0 < it.sink_end)) {
            at.x = a.b.table[(size_t)part.s * a.b.table_stride + pi];
            if (at.x < 0 || at.x >= a.b.num_pages) {
                if (a.err) atomicOr(a.err, kErrPage);
                at.x = a.b.num_pages;
            }
        }
    }
    return at;
}

// Pool row of position p of sequence s for KV head kvh, or -1 (a page that
// the pool does not have).
__device__ __forceinline__ int pool_row(const PagedBatch& b, int s, int kvh, int p, unsigned* err) {
    const int pi = b.by_page(p), page = b.table[(size_t)s * b.table_stride + pi];
    if (page < 0 || page >= b.num_pages) {
        if (err) atomicOr(err, kErrPage);
        return -1;
    }
    return (page * b.nkv + kvh) * b.page_size + (p - pi * b.page_size);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ------------------------------------------------- values that are not finite
// A tile multiplies the value of a key that a row does not see by a
// probability of 0, which is NaN where the value is infinite or NaN.  So V
// rows that no row of the item sees become zeros in shared memory, and where
// some rows see a key that others do not, so do its values that are not
// finite.  Those are then added to the sums of the rows that see them
// (restore_*): w V is V for any w > 0.  That is work for the few tiles at the
// ends of an item's keys alone, whatever V holds and however long the cache,
// so no wait of these kernels depends on it.  In tiles that every row sees
// whole the products give what the formula does.

__device__ __forceinline__ bool row_sees(const AttnArgs& a, int pos, int p) {
    return p <= pos && (a.window == 0 || p > pos - a.window || p < a.sinks);
}

// Whether every row of the item sees all N keys of the tile at k0.  Where not,
// and the item has several positions, some rows may see a key that others do
// not.
template <int N>
__device__ __forceinline__ bool seen_whole(const AttnArgs& a, const Item& it, int k0) {
    return k0 + N - 1 <= it.pos_first && (a.window == 0 || k0 > it.pos_last - a.window || k0 + N <= a.sinks);
}

// Whether the tile at k0 has keys that no row of the item sees.
template <int N>
__device__ __forceinline__ bool has_hidden(const Item& it, int k0) {
    return k0 + N > it.hi || (k0 < it.lo && k0 + N > it.sink_end);
}

// Address of 16-byte chunk ch of row `row` of a tile of 64 rows in shared
// memory: blocks of 64 columns, rows of 128 bytes, as a tensor map with
// 128-byte swizzle writes them.
__device__ __forceinline__ uint32_t chunk_at(uint32_t tile, int row, int ch) {
    return tile + (uint32_t)(ch >> 3) * 8192u + (uint32_t)(row * 128 + (((ch & 7) ^ (row & 7)) << 4));
}
__device__ __forceinline__ uint4 ld_shared(uint32_t at) {
    uint4 w;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                 : "r"(at)
                 : "memory");
    return w;
}
__device__ __forceinline__ void st_shared(uint32_t at, uint4 w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w)
                 : "memory");
}

// Ones where eight values are not finite.
template <typename T>
__device__ __forceinline__ uint4 not_finite(uint4 w) {
    return make_uint4(Half16<T>::not_finite(w.x), Half16<T>::not_finite(w.y), Half16<T>::not_finite(w.z),
                      Half16<T>::not_finite(w.w));
}
__device__ __forceinline__ bool any_bit(uint4 w) { return (w.x | w.y | w.z | w.w) != 0u; }

// A warp's part, in shared memory for what runs rarely: the loops over the
// tiles then need not keep all of it in registers.
struct Current {
    Item it;
    Part part;
    int no;  // counts the parts
};
__device__ __forceinline__ void set_current(Current& cur, const Item& it, const Part& part) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) {
        cur.it = it;
        cur.part = part;
        ++cur.no;
    }
    __syncwarp();
}

// The rows [r0, r0 + ROWS) of the V tile of keys k0 ... by a warp: zeros in
// rows that no row of the item sees and, where `some`, for values that are not
// finite.  When there were any, *found_in is the part before they go, so that a
// warp that cleans the same rows and meets them gone finds it there.
template <typename T, int D, int ROWS>
__device__ __noinline__ void clean_rows(const Current& cur, int k0, uint32_t tile, int r0, bool some,
                                        volatile int* found_in) {
    constexpr int kAtOnce = ROWS < 32 ? ROWS : 32, kPerLane = D / 8 * kAtOnce / 32;  // rows; chunks of a lane's row
    static_assert(kPerLane % 4 == 0, "");
    const int lane = threadIdx.x & 31, c0 = lane / kAtOnce * kPerLane;
    const Item it = cur.it;
    // 0 v is 0, or NaN where v is not finite: one step for two values
    uint32_t sum[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int h = 0; h < ROWS; h += kAtOnce) {
        const int r = r0 + h + lane % kAtOnce;
        if (!item_sees(it, k0 + r)) {
#pragma unroll
            for (int c = 0; c < kPerLane; ++c) st_shared(chunk_at(tile, r, c0 + c), make_uint4(0u, 0u, 0u, 0u));
        } else if (some) {
#pragma unroll
            for (int c = 0; c < kPerLane; c += 4) {
                uint4 w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = ld_shared(chunk_at(tile, r, c0 + c + i));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sum[0] = Half16<T>::add_zero_times(w[i].x, sum[0]);
                    sum[1] = Half16<T>::add_zero_times(w[i].y, sum[1]);
                    sum[2] = Half16<T>::add_zero_times(w[i].z, sum[2]);
                    sum[3] = Half16<T>::add_zero_times(w[i].w, sum[3]);
                }
            }
        }
    }
    if (__any_sync(0xffffffffu, any_bit(not_finite<T>(make_uint4(sum[0], sum[1], sum[2], sum[3]))))) {
        if (lane == 0) *found_in = cur.no;
        __threadfence_block();
        __syncwarp();
        for (int i = lane; i < ROWS * (D / 8); i += 32) {
            const uint32_t at = chunk_at(tile, r0 + i % ROWS, i / ROWS);
            const uint4 w = ld_shared(at), x = not_finite<T>(w);
            if (any_bit(x)) st_shared(at, make_uint4(w.x & ~x.x, w.y & ~x.y, w.z & ~x.z, w.w & ~x.w));
        }
    }
    fence_proxy_async_smem();  // before the products read the tile, and before it is loaded again
    __syncwarp();
}

// f(key, its V row in the pool) for the keys of a part's tiles that some rows
// may see and others not, and that have values that are not finite, by a whole
// warp.
template <typename T, int D, int N, typename F>
__device__ __forceinline__ void each_not_finite(const AttnArgs& a, const Current& cur, F f) {
    const int lane = threadIdx.x & 31;
    const Item& it = cur.it;
    for (int j = cur.part.j0; j < cur.part.j1; ++j) {
        const int k0 = tile_key<N>(it, j);
        if (seen_whole<N>(a, it, k0)) continue;
        for (int h = 0; h < N; h += 32) {
            const int p = k0 + h + lane, row = item_sees(it, p) ? pool_row(a.b, cur.part.s, it.kvh, p, nullptr) : -1;
            bool bad = false;
            if (row >= 0) {
                const uint4* v = reinterpret_cast<const uint4*>(static_cast<const T*>(a.v) + (long long)row * D);
#pragma unroll 4
                for (int c = 0; c < D / 8; ++c) bad |= any_bit(not_finite<T>(__ldg(v + c)));
            }
            for (unsigned left = __ballot_sync(0xffffffffu, bad); left; left &= left - 1) {
                const int k = __ffs(left) - 1;
                f(k0 + h + k, static_cast<const T*>(a.v) + (long long)__shfl_sync(0xffffffffu, row, k) * D);
            }
        }
    }
}

// Joined values of row r, columns d and d + 1, of an item's partial results.
struct Joined {
    float m, l, x, y;
};

// A slot: out, M rows of D, then m [M] and l [M] of an item's rows.
template <int M, int D>
constexpr size_t slot_floats() {
    return (size_t)M * (D + 2);
}

// The slot of CTA b for an item whose first CTA is `first`.
template <int M, int D>
__device__ __forceinline__ float* slot_of(const AttnArgs& a, int b, int first) {
    return a.slots + (size_t)(2 * b + (b == first)) * slot_floats<M, D>();
}

constexpr float kLn2 = 0.6931471805599453f;

}  // namespace infernt
