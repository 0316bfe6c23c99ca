// paged_attention.cuh — what the two attention kernels over paged caches
// share: the query rows and keys of an item, the even split of the work over
// the CTAs, the partial results of split items, and the term-by-term row.
#pragma once

#include "paged.cuh"

namespace infernt {

constexpr float kRescale = 8.0f;  // log2 of the largest unnormalised probability

// Workspace: the tickets of split items, then two slots of partial results
// for each CTA.
constexpr size_t kWorkspaceBytes = 64u << 20;
constexpr int kMaxCtas = 640;
constexpr size_t kSlotsAt = 4096;

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
    int min_tiles;      // least tiles of a CTA
    unsigned* tickets;  // [CTAs], zero between calls
    float* slots;
    unsigned* err;
};

// The tcgen05 kernel (paged_attention_tc.cu); pages as paged_attention_tc_pages says.
int paged_attention_tc(const AttnArgs& a, int head_dim, int dtype, cudaStream_t st);
bool paged_attention_tc_pages(int page_size);

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
// each item of M query rows, one unit per tile of N keys (one where a row
// sees nothing: its zeros have to be written).  CTA b takes the units [b c,
// (b + 1) c), so every CTA reads the same number of tiles whatever the
// lengths, and an item that crosses a border is split: its CTAs leave partial
// results (two slots a CTA are enough: one for an item that began before it,
// one for an item that goes on after it), and the last of them to arrive
// joins them in CTA order.  Lengths are device data; each CTA finds its own
// place by a scan over the sequences.
template <int M, int N>
__device__ __forceinline__ int item_units(const AttnArgs& a, const PagedSeq& s, int row0) {
    return row0 < s.n_new * a.G ? max(1, make_item<M, N>(a, s, 0, row0).tiles) : 0;
}

// Units of one KV head of s, by a whole warp.
template <int M, int N>
__device__ __forceinline__ int head_units(const AttnArgs& a, const PagedSeq& s) {
    const int lane = threadIdx.x & 31;
    int n = 0;
    for (int row0 = lane * M; row0 < s.n_new * a.G; row0 += 32 * M) n += item_units<M, N>(a, s, row0);
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

struct Place {
    long long c;       // units of a CTA
    long long before;  // units before sequence seq
    long long total;
    int seq;           // the sequence that holds unit c x blockIdx.x; -1: nothing for this CTA
};

// By all NT threads of the block.
template <int M, int N, int NT>
__device__ __forceinline__ Place find_place(const AttnArgs& a) {
    __shared__ long long sums_s[NT / 32];
    __shared__ long long before_s;
    __shared__ int seq_s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = a.b.num_seqs;
    // units of sequence s (every thread its own); long ones by the whole warp
    auto units = [&](int s) {
        PagedSeq q = {0, 0, 0};
        if (s < n) q = paged_seq(a.b, s, blockIdx.x == 0 ? a.err : nullptr);
        const bool many = q.n_new * a.G > 2 * M;
        int u = many ? 0 : item_units<M, N>(a, q, 0) + item_units<M, N>(a, q, M);
        for (unsigned left = __ballot_sync(0xffffffffu, many); left; left &= left - 1) {
            const int k = __ffs(left) - 1;
            const PagedSeq w = {__shfl_sync(0xffffffffu, q.row0, k), __shfl_sync(0xffffffffu, q.n_new, k),
                                __shfl_sync(0xffffffffu, q.len, k)};
            const int x = head_units<M, N>(a, w);
            if (lane == k) u = x;
        }
        return (long long)u * a.b.nkv;
    };
    // the sum of the values before this thread's, and of all of them
    auto scan = [&](long long v, long long& all) {
        long long x = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 31) sums_s[warp] = x;
        __syncthreads();
        long long pre = x - v;
        all = 0;
#pragma unroll
        for (int w = 0; w < NT / 32; ++w) {
            if (w < warp) pre += sums_s[w];
            all += sums_s[w];
        }
        return pre;
    };
    if (tid == 0) seq_s = -1;
    Place p;
    long long mine = 0, before = 0;
    p.total = 0;
    for (int base = 0; base < n; base += NT) {
        long long all;
        mine = units(base + tid);
        before = p.total + scan(mine, all);
        p.total += all;
    }
    p.c = max((long long)a.min_tiles, (p.total + gridDim.x - 1) / gridDim.x);
    const long long at = p.c * blockIdx.x;
    long long sum = 0;
    for (int base = 0; base < n; base += NT) {
        if (n > NT) {  // a second pass; up to NT sequences are still in registers
            long long all;
            mine = units(base + tid);
            before = sum + scan(mine, all);
            sum += all;
        }
        if (before <= at && at < before + mine) {
            seq_s = base + tid;
            before_s = before;
        }
    }
    __syncthreads();
    p.seq = seq_s;
    p.before = before_s;
    return p;
}

// Part [j0, j1) of an item's tiles; first and last: the CTAs that the item
// begins and ends in.
struct Part {
    int s, j0, j1;
    long long first, last;
};

// f(sequence, item, part) for the parts of this CTA, by whole warps.
template <int M, int N, typename F>
__device__ __forceinline__ void walk(const AttnArgs& a, const Place& p, F f) {
    long long at = p.c * blockIdx.x, before = p.before;
    const long long end = min(at + p.c, p.total);
    for (int s = p.seq; at < end && s < a.b.num_seqs; ++s) {
        const PagedSeq seq = paged_seq(a.b, s, nullptr);
        const int per_head = head_units<M, N>(a, seq);
        if (per_head == 0) continue;
        int kvh = (int)((at - before) / per_head);
        long long u0 = before + (long long)kvh * per_head;
        int rem = (int)(at - u0);
        int row0 = find_item<M, N>(a, seq, rem);
        u0 += rem;
        while (kvh < a.b.nkv && at < end) {
            const Item it = make_item<M, N>(a, seq, kvh, row0);
            const int units = max(1, it.tiles);
            Part part;
            part.s = s;
            part.j0 = (int)(at - u0);
            part.j1 = min(it.tiles, (int)min((long long)units, end - u0));
            part.first = u0 / p.c;
            part.last = (u0 + units - 1) / p.c;
            f(seq, it, part);
            at = u0 += units;
            row0 += M;
            if (row0 >= seq.n_new * a.G) {
                row0 = 0;
                ++kvh;
            }
        }
        before += (long long)per_head * a.b.nkv;
    }
}

// Whether some row of the item sees key p.
__device__ __forceinline__ bool item_sees(const Item& it, int p) {
    return p < it.hi && (p >= it.lo || p < it.sink_end);
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

// One row by one warp, term by term: what a row is computed with when its
// result is not finite.  The tiles above multiply a hidden position's value
// by a probability of 0, which is NaN where the value is infinite or NaN;
// here only what the row sees is touched, so what a row does see that is not
// finite still shows in its result as in the formula.
template <typename T, int D>
__device__ void exact_row(const AttnArgs& a, const PagedSeq& seq, int s, int kvh, int row) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31, token = a.by_g(row), head = kvh * a.G + row - token * a.G;
    const int pos = row_pos(seq, token);
    const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0, sink_end = min(a.sinks, lo);
    const T* q = static_cast<const T*>(a.q) + (long long)(seq.row0 + token) * a.ldq + (long long)head * D + lane * E;
    float qv[E], acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        qv[e] = Half16<T>::value(q[e]);
        acc[e] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (int p = 0; p <= pos; ++p) {
        if (p == sink_end) p = lo;  // lo <= pos
        const int r = pool_row(a.b, s, kvh, p, a.err);
        const T* k = static_cast<const T*>(a.k) + (long long)r * D + lane * E;
        const T* v = static_cast<const T*>(a.v) + (long long)r * D + lane * E;
        float dot = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) dot = fmaf(qv[e], r >= 0 ? Half16<T>::value(k[e]) : 0.0f, dot);
        const float sc = warp_sum(dot) * a.scale, m_new = fmaxf(m, sc);
        const float f = m == -INFINITY ? 0.0f : expf(m - m_new), w = expf(sc - m_new);
        l = l * f + w;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = acc[e] * f + w * (r >= 0 ? Half16<T>::value(v[e]) : 0.0f);
        m = m_new;
    }
    T* o = static_cast<T*>(a.out) + (long long)(seq.row0 + token) * a.ldo + (long long)head * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = Half16<T>::round(acc[e] / l);
    if (a.lse && lane == 0) a.lse[(long long)(seq.row0 + token) * a.nq + head] = m + logf(l);
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
__device__ __forceinline__ float* slot_of(const AttnArgs& a, long long b, long long first) {
    return a.slots + (size_t)(2 * b + (b == first)) * slot_floats<M, D>();
}

constexpr float kLn2 = 0.6931471805599453f;

}  // namespace infernt
