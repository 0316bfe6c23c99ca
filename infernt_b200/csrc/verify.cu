// verify.cu — drafted tokens against the target's distributions: which drafts
// of each sequence stand, and the token after them, drawn from given random
// numbers (src/engine.cpp:78-104 draws one token from softmax(logits / T) on
// the host, by the same walk along the cumulative sum).
//
//   p = e^((l - max l) / T) / Z;  a draft d stands while u q(d) < p(d);
//   at the first that does not, the token is the lowest i with
//   sum_{k <= i} w_k > u' sum_k w_k,  w = max(p - q, 0).
//
// Two launches: the statistics of every row (its logits are read once, HBM),
// then a cluster of CTAs a sequence, which finds the row where the sequence
// stops and draws.  A border of the cumulative sum is as near as 10^-6 to
// u' sum w where there are 10^5 tokens, so what the draw is made of (Z, the
// weights, their sums) is in 64 bits; acceptance is one comparison a row, and
// its Z a sum in FP32.
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "paged.cuh"

namespace infernt {
namespace {

constexpr int kStatThreads = 256;
constexpr int kStatTile = 8192;   // elements of a row that a CTA holds in registers
constexpr int kMostParts = 32;    // CTAs of a row
constexpr float kLog2e = 1.4426950408889634f;

// What a CTA knows of its part of a row: e is the sum of 2^((l - m) c).
struct RowPart {
    float m, e;
    int best;   // of a greedy sequence the lowest index of m; -1: no number
    int flags;  // kBad: a NaN or an element out of range
};
constexpr int kBad = 1;

struct VerifyArgs {
    const void* target;
    const float* draft;
    long long ld, draft_ld;
    const int* tokens;
    const int* q_start;
    const float* temperature;
    const float* u;
    const int* kv_len;
    int* kept;
    int* out;
    int* accepted;
    RowPart* parts;  // [num_rows][kMostParts]
    int num_seqs, num_rows, V, n_parts, part;  // part: elements of one
    int cluster;                               // CTAs that draw for a sequence
    unsigned* err;
};

__device__ __forceinline__ float element(const float* p) { return __ldg(p); }
__device__ __forceinline__ float element(const __nv_bfloat16* p) { return __bfloat162float(__ldg(p)); }
__device__ __forceinline__ float element(const __half* p) { return __half2float(__ldg(p)); }

__device__ __forceinline__ bool is_greedy(float t) { return !(t > 0.0f); }
// log2(e) / T; an infinite T would make 0 of -infinity, one near 0 infinity of 0
__device__ __forceinline__ float sharpness(float t) { return fminf(fmaxf(kLog2e / t, 1e-30f), 1e30f); }
__device__ __forceinline__ double sharpness64(float t) {
    return fmin(fmax(1.4426950408889634074 / (double)t, 1e-30), 1e30);
}

// What a probability may not be.
__device__ __forceinline__ bool is_none(float x) { return !(x < INFINITY) || x < 0.0f; }

// 16 bytes of a row as FP32
__device__ __forceinline__ void sixteen(const float* p, float (&x)[4]) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(p));
    x[0] = v.x;
    x[1] = v.y;
    x[2] = v.z;
    x[3] = v.w;
}
template <typename L>
__device__ __forceinline__ void sixteen(const L* p, float (&x)[8]) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 y = Half16<L>::unpack(w[i]);
        x[2 * i] = y.x;
        x[2 * i + 1] = y.y;
    }
}

// The warp's largest by argmax_better, and its index (-1: none).
__device__ __forceinline__ void best_of_warp(float& m, int& at) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, m, o);
        const int oi = __shfl_xor_sync(0xffffffffu, at, o);
        if (oi >= 0 && (at < 0 || argmax_better(om, oi, m, at))) {
            m = om;
            at = oi;
        }
    }
}

// Block (row, part).  A thread's elements come in 16-byte loads, all of them
// before the first is used, and before the row's sequence is known, which takes
// two or three dependent loads; rows that do not start on 16 bytes start their
// first vector before the row, and the elements outside it are not loaded.
// HBM-bound where rows are many and long: 320 of 128256 in FP32, 164 MB, 33 us,
// 4.9 TB/s; of 32000 in bf16 400 take 16 us, each CTA's own start, loads and sums.
template <typename L, bool PROBS>
__global__ void __launch_bounds__(kStatThreads) verify_rows(const VerifyArgs a) {
    constexpr int N = 16 / (int)sizeof(L), VECS = kStatTile / N / kStatThreads;
    __shared__ float m_s[kStatThreads / 32], e_s[kStatThreads / 32];
    __shared__ int at_s[kStatThreads / 32], bad_s;
    pdl_launch_dependents();
    const int r = blockIdx.x, part = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const L* row = static_cast<const L*>(a.target) + (long long)r * a.ld;
    const int off = (int)(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(L));
    float x[VECS][N], t = 1.0f;
    bool bad = false;
    auto load = [&](int base) {
#pragma unroll
        for (int i = 0; i < VECS; ++i) {
            const int k = base + (i * kStatThreads + tid) * N;
            if (k >= 0 && k + N <= a.V) {
                sixteen(row + k, x[i]);
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) x[i][j] = k + j >= 0 && k + j < a.V ? element(row + k + j) : -INFINITY;
            }
        }
    };
    // only what is drafted, and the row where the sequence stops, are asked of probabilities (but for the greedy)
    if (!PROBS) load(part * a.part - off);
    if (a.temperature) t = a.temperature[find_seq(a.q_start, a.num_seqs, r)];
    const bool greedy = is_greedy(t);
    if (PROBS) {
        if (!greedy) return;
        load(part * a.part - off);
    }
    const float c = greedy ? 0.0f : sharpness(t);
    if (tid == 0) bad_s = 0;
    float m = -INFINITY, e = 0.0f;
    int at = -1;
    for (int tile = 0; tile < a.part; tile += kStatTile) {
        const int base = part * a.part + tile - off;
        if (tile) load(base);
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < VECS; ++i)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                top = fmaxf(top, x[i][j]);
                // what lies outside the row is -infinity, which in it a logit may be and a probability not
                const int k = base + (i * kStatThreads + tid) * N + j;
                bad |= PROBS ? is_none(x[i][j]) && k >= 0 && k < a.V : !(x[i][j] < INFINITY);
            }
        const float ref = fmaxf(m, top);
        if (!greedy && ref > -INFINITY) {
            float sum[2] = {0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < VECS; ++i)
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    float y;
                    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"((x[i][j] - ref) * c));
                    sum[j & 1] += y;
                }
            e = e * (m == -INFINITY ? 0.0f : exp2f((m - ref) * c)) + sum[0] + sum[1];
        }
        if (greedy && top > m) {  // the lowest index of it
#pragma unroll
            for (int i = VECS - 1; i >= 0; --i)
#pragma unroll
                for (int j = N - 1; j >= 0; --j)
                    if (x[i][j] == top) at = base + (i * kStatThreads + tid) * N + j;
        }
        m = ref;
    }
    // the warps' and then the CTA's
    float wm = m;
    best_of_warp(wm, at);
    if (!greedy) wm = warp_max(m);
    e = warp_sum(m == -INFINITY ? 0.0f : e * exp2f((m - wm) * c));
    bad = __any_sync(0xffffffffu, bad);
    __syncthreads();
    if (lane == 0) {
        if (bad) bad_s = 1;
        m_s[warp] = wm;
        e_s[warp] = e;
        at_s[warp] = at;
    }
    __syncthreads();
    if (warp != 0) return;
    m = lane < kStatThreads / 32 ? m_s[lane] : -INFINITY;
    at = lane < kStatThreads / 32 ? at_s[lane] : -1;
    e = lane < kStatThreads / 32 ? e_s[lane] : 0.0f;
    wm = m;
    best_of_warp(wm, at);
    if (!greedy) wm = warp_max(m);
    e = warp_sum(m == -INFINITY ? 0.0f : e * exp2f((m - wm) * c));
    if (lane == 0) a.parts[(size_t)r * kMostParts + part] = {wm, e, at, bad_s ? kBad : 0};
}

// ------------------------------------------------------------------- draw
constexpr int kDrawThreads = 256;
constexpr int kDrawWarps = kDrawThreads / 32;
constexpr int kDrawPerSm = 3;
constexpr int kMostCluster = 8;

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ double peer_double(const double* p, uint32_t rank) {
    uint32_t at;
    double v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// 2^x for x up to 0, from -1000 on (below it as at -1000, -infinity too), to
// about 2e-15: x = (32 n + j) / 32 + g, |g| <= 1 / 64, so 2^x = 2^n 2^(j / 32)
// 2^g, the last by its Taylor series to the fifth power (the sixth is below (ln 2
// / 64)^6 / 720 = 2e-15), the middle one of the 32 roots (in shared memory; from
// lane to lane by shuffles a call took 3 us more).  The constants are in constant
// memory, where the operations take them from without a move.
struct Exp2Constants {
    double big, back;  // 1.5 x 2^52 rounds 32 x to a whole number in its low bits
    double c[6];       // (ln 2)^k / k!
};
__constant__ Exp2Constants kExp2 = {6755399441055744.0,
                                    -1.0 / 32.0,
                                    {1.0, 0.69314718055994530942, 0.24022650695910071233, 0.05550410866482157995,
                                     0.00961812910762847716, 0.00133335581464284434}};
__device__ __forceinline__ double exp2_64(double x, const double* roots) {
    // of negative numbers the high words ascend with the magnitude (-1000: 0xc08f4000); those of others are lower
    x = __hiloint2double((int)min((unsigned)__double2hiint(x), 0xc08f4000u), __double2loint(x));
    const double t = fma(x, 32.0, kExp2.big);
    const int k = __double2loint(t);
    const double g = fma(t - kExp2.big, kExp2.back, x);
    double p = fma(g, kExp2.c[5], kExp2.c[4]);
    p = fma(p, g, kExp2.c[3]);
    p = fma(p, g, kExp2.c[2]);
    p = fma(p, g, kExp2.c[1]);
    p = fma(p, g, kExp2.c[0]);
    const double y = p * roots[k & 31];
    return __hiloint2double(__double2hiint(y) + (k >> 5) * (1 << 20), __double2loint(y));
}

// What becomes of a sequence.
struct Stop {
    int row;    // where it stops
    int token;  // the next token: >= 0 known, kDraw, kLargest
    int minus;  // what is subtracted: 1 the draft's distribution, 2 the drafted token alone
    float m;    // the largest logit of that row
    unsigned err;
};
constexpr int kDraw = -1, kLargest = -2;  // to be drawn; the row's largest number, to be looked for

// A row's statistics, by a whole warp.
template <bool PROBS>
__device__ __forceinline__ RowPart row_stats(const VerifyArgs& a, int r, float c, bool greedy) {
    const int lane = threadIdx.x & 31;
    RowPart p = {-INFINITY, 0.0f, -1, 0};
    if (lane < a.n_parts) p = a.parts[(size_t)r * kMostParts + lane];
    const float m = p.m;
    best_of_warp(p.m, p.best);
    if (!greedy) p.m = warp_max(m);
    p.e = warp_sum(m == -INFINITY ? 0.0f : p.e * exp2f((m - p.m) * c));
    p.flags = __any_sync(0xffffffffu, p.flags & kBad) || !(p.m > (PROBS ? 0.0f : -INFINITY)) ? kBad : 0;
    return p;
}

// Element e of row r that is a probability, or less than 0.
template <typename L>
__device__ __forceinline__ float probability(const VerifyArgs& a, int r, int e) {
    const float p = element(static_cast<const L*>(a.target) + (long long)r * a.ld + e);
    return is_none(p) ? -1.0f : p;
}
__device__ __forceinline__ float in_unit(float u) { return u >= 0.0f ? fminf(u, 0.99999994f) : 0.0f; }

// A row's largest number at its lowest index into *out (0 if it has none), by
// one CTA.  For rows that are no distribution.
template <typename L>
__device__ __noinline__ void put_largest(const L* row, int V, int* out) {
    __shared__ float m_s[kDrawWarps];
    __shared__ int at_s[kDrawWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    float m = -INFINITY;
    int at = -1;
    for (int i = tid; i < V; i += kDrawThreads) {
        const float x = element(row + i);
        if (x > -INFINITY && (at < 0 || argmax_better(x, i, m, at))) {
            m = x;
            at = i;
        }
    }
    best_of_warp(m, at);
    if (lane == 0) {
        m_s[warp] = m;
        at_s[warp] = at;
    }
    __syncthreads();
    if (warp != 0) return;
    m = lane < kDrawWarps ? m_s[lane] : -INFINITY;
    at = lane < kDrawWarps ? at_s[lane] : -1;
    best_of_warp(m, at);
    if (lane == 0) *out = at < 0 ? 0 : at;
}

// A cluster of CTAs a sequence, a slice of the vocabulary each, and in it a
// stretch for each warp, in kSubs pieces.  In every CTA the warps judge the
// sequence's rows; then
//   Z = sum e_i over the cluster, where a distribution is taken off (else w is
//   as good as w Z: a pass less, 100 sequences of 32000 tokens 33 -> 29 us);
//   W = sum w_i over the cluster;
//   the CTA, in it the warp, and of its stretch the piece whose part of the sum
//   has u W in it: that piece is walked along, a group of elements at a time.
// The weights are computed again in each pass (the logits are in L2): some 25
// operations in 64 bits an element, each waiting for the one before, so a lane
// has eight elements on the way.  64 sequences that stop, 128256 tokens from HBM: 43
// us (of 14 that the operations take where none waits); three CTAs an SM with
// 80 registers a thread, four with 64 took 7 us more.  Of probabilities no other
// rows are read (66 MB with the drafts', 10 us of HBM): the call takes 30.5 us in
// a graph, the draw's loads, sums and barriers in turn.
constexpr int kSubs = 16;
constexpr int kEach = 8;  // elements that a lane has at once
constexpr int kGroup = 32 * kEach;

template <typename L, bool PROBS>
__global__ void __launch_bounds__(kDrawThreads, kDrawPerSm) verify_draw(const __grid_constant__ VerifyArgs a) {
    __shared__ double roots[32], sum_s[3][kDrawWarps], shared_s[3];  // shared_s: what the other CTAs read
    __shared__ double sub_s[kDrawWarps][kSubs][32];       // the lanes' sums of the warps' pieces
    __shared__ int first_s;
    __shared__ Stop stop_s[kDrawWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, s = blockIdx.x / a.cluster;
    const uint32_t rank = cluster_rank();
    if (tid < 32) roots[tid] = exp2((double)tid / 32.0);
    if (tid == 0) first_s = 0x7fffffff;
    const int row0 = a.q_start[s], end = a.q_start[s + 1], n = end - row0;
    const bool sane = row0 >= 0 && n >= 0 && end <= a.num_rows;
    const float t = a.temperature ? a.temperature[s] : 1.0f;
    const bool greedy = is_greedy(t), stats = !PROBS || greedy;
    const float c = greedy ? 0.0f : sharpness(t);
    const double c64 = greedy ? 0.0 : sharpness64(t);
    __syncthreads();
    // ---- the first row whose draft does not stand (a warp a row, in turn); what does not hang on verify_rows first
    bool waited = false;
    if (sane)
        for (int i = warp; i < n; i += kDrawWarps) {
            const int r = row0 + i;
            if (waited && __any_sync(0xffffffffu, r > *static_cast<volatile int*>(&first_s))) break;
            const int d = i + 1 < n ? a.tokens[r + 1] : -1;
            const bool drafted = d >= 0 && d < a.V;
            float l = 0.0f, q = 1.0f, u = 0.0f;
            if (drafted && !greedy) {
                l = PROBS ? probability<L>(a, r, d) : element(static_cast<const L*>(a.target) + (long long)r * a.ld + d);
                if (a.draft) q = a.draft[(long long)r * a.draft_ld + d];
                u = in_unit(a.u[r]);
            }
            if (!waited) pdl_wait();  // verify_rows
            waited = true;
            RowPart p = {0.0f, 1.0f, 0, 0};
            if (stats) p = row_stats<PROBS>(a, r, c, greedy);
            Stop st = {r, kDraw, 0, p.m, i + 1 < n && !drafted ? (unsigned)kErrToken : 0u};
            bool stands = false;
            if (greedy) {
                stands = drafted && d == p.best && !(p.flags & kBad);
                st.token = p.best < 0 ? 0 : p.best;
                if (p.flags & kBad) st.err |= kErrValue;
            } else if (p.flags & kBad) {
                st.token = kLargest;
                st.err |= kErrValue;
            } else if (drafted) {
                const double x = ((double)l - (double)p.m) * c64;
                const double pd = PROBS ? (double)l : x > -1000.0 ? exp2_64(x, roots) / (double)p.e : 0.0;
                stands = (double)u * (double)q < pd;
                st.minus = a.draft ? 1 : 2;
            }
            if (!stands) {
                if (lane == 0) {
                    stop_s[warp] = st;
                    atomicMin(&first_s, r);
                }
                __syncwarp();
                break;
            }
        }
    if (!waited) pdl_wait();  // of every thread, so that this kernel's end is the call's end
    __syncthreads();
    if (!sane || n == 0) {  // the whole cluster
        if (rank == 0 && tid == 0) {
            if (!sane && a.err) atomicOr(a.err, kErrBatch);
            if (sane) {
                a.accepted[s] = 0;
                if (a.kept) a.kept[s] = a.kv_len[s];
            }
        }
        return;
    }
    const int stop = first_s;
    const Stop st = stop_s[(stop - row0) % kDrawWarps];
    if (rank == 0) {
        const int good = stop - row0;
        for (int i = tid; i < n; i += kDrawThreads)
            if (i != good) a.out[row0 + i] = i < good ? a.tokens[row0 + i + 1] : -1;
        if (tid == 0) {
            a.accepted[s] = good;
            if (a.kept) a.kept[s] = a.kv_len[s] - (n - 1 - good);
            if (st.token >= 0) a.out[stop] = st.token;
            if (a.err && st.err) atomicOr(a.err, st.err);
        }
        if (st.token == kLargest)
            put_largest<L>(static_cast<const L*>(a.target) + (long long)stop * a.ld, a.V, a.out + stop);
    }
    if (st.token != kDraw) return;  // the whole cluster
    // ---- the draw.  This warp's stretch: groups [g0, g1) of kGroup elements, `sub` of them a piece.
    const L* row = static_cast<const L*>(a.target) + (long long)stop * a.ld;
    const float* draft = a.draft ? a.draft + (long long)stop * a.draft_ld : nullptr;
    const int groups = (a.V + kGroup - 1) / kGroup, per = (groups + a.cluster * kDrawWarps - 1) / (a.cluster * kDrawWarps);
    const int sub = (per + kSubs - 1) / kSubs;
    const int g0 = min(groups, ((int)rank * kDrawWarps + warp) * per), g1 = min(groups, g0 + per);
    const int d = st.minus == 2 ? a.tokens[stop + 1] : -1;
    // x = c l - c m in one operation, off by what the rounding of c m is: the same for all of a row, so no matter, as
    // long as it is small.  From c = 2^35 / |m| on the next FP32 number below m has a weight of 2^-2048 or less, which
    // is 0 here, so a larger c (temperatures from |m| 2^-35 down) changes nothing, and c m stays below 2^35.
    const double c_draw = fmin(c64, 34359738368.0 / fabs((double)st.m)), cm = -c_draw * (double)st.m;
    // weights up to 2^-990 are 0: those of tokens that are not allowed, among others
    constexpr double kLeastWeight = PROBS ? 0.0 : 9.555938177272168e-299;
    bool bad = false;
    double z = 1.0;
    constexpr float kOutside = PROBS ? 0.0f : -INFINITY;  // has no weight
    auto weight = [&](float l) {                          // e, or p
        if (!PROBS) return exp2_64(fma((double)l, c_draw, cm), roots);
        bad |= is_none(l);
        return (double)l;
    };
    // the weight that is drawn from; minus as in Stop
    auto left = [&](auto minus, int i, float l, float q) {
        double w = weight(l);
        if (decltype(minus)::value == 1) w = fma(w, z, -(double)(fabsf(q) < INFINITY ? q : 3.0e38f));
        return w > kLeastWeight && !(decltype(minus)::value == 2 && i == d) ? w : 0.0;
    };
    // a group, kEach elements a lane; the last one's may lie behind the row
    auto get = [&](const auto* from, int g, float none, float (&x)[kEach]) {
        const auto* at = from + (long long)g * kGroup + lane;
        if (g * kGroup + kGroup <= a.V) {
#pragma unroll
            for (int j = 0; j < kEach; ++j) x[j] = element(at + 32 * j);
        } else {
#pragma unroll
            for (int j = 0; j < kEach; ++j) x[j] = g * kGroup + 32 * j + lane < a.V ? element(at + 32 * j) : none;
        }
    };
    // the sum over the CTA's warps into its shared_s[slot], then over the cluster, both in order; the CTAs' sums in of
    using Sums = double[kMostCluster];
    auto over_cluster = [&](double v, int slot, Sums& of) {
        v = warp_sum64(v);
        if (lane == 0) sum_s[slot][warp] = v;
        __syncthreads();
        if (tid == 0) {
            double x = 0.0;
            for (int w = 0; w < kDrawWarps; ++w) x += sum_s[slot][w];
            shared_s[slot] = x;
        }
        cluster_sync();
        // all on their way before the first is added
#pragma unroll
        for (int k = 0; k < kMostCluster; ++k) of[k] = k < a.cluster ? peer_double(&shared_s[slot], k) : 0.0;
        double x = of[0];
#pragma unroll
        for (int k = 1; k < kMostCluster; ++k) x += of[k];
        return x;
    };
    if (!PROBS && st.minus == 1) {
        double v = 0.0;
        for (int g = g0; g < g1; ++g) {
            float l[kEach];
            get(row, g, kOutside, l);
#pragma unroll
            for (int j = 0; j < kEach; j += 2) v += weight(l[j]) + weight(l[j + 1]);
        }
        Sums of;
        z = 1.0 / over_cluster(v, 0, of);
    }
    // this warp's pieces; their sum
    auto pieces = [&](auto minus) {
        double mine = 0.0;
        for (int g = g0, k = 0; k < kSubs; ++k) {
            double piece = 0.0;
            for (const int stop_g = min(g1, g + sub); g < stop_g; ++g) {
                float l[kEach], q[kEach];
                get(row, g, kOutside, l);
                if (decltype(minus)::value == 1) get(draft, g, 0.0f, q);
                const int i = g * kGroup + lane;
#pragma unroll
                for (int j = 0; j < kEach; j += 2)
                    piece += left(minus, i + 32 * j, l[j], q[j]) + left(minus, i + 32 * j + 32, l[j + 1], q[j + 1]);
            }
            sub_s[warp][k][lane] = piece;
            mine += piece;
        }
        return mine;
    };
    using std::integral_constant;
    int minus = st.minus;
    Sums sums;
    double total = over_cluster(minus == 1   ? pieces(integral_constant<int, 1>())
                                : minus == 2 ? pieces(integral_constant<int, 2>())
                                             : pieces(integral_constant<int, 0>()),
                                1, sums);
    if (minus && !(total > 0.0)) {  // nothing is left: from p itself
        minus = 0;
        cluster_sync();  // shared_s is read
        total = over_cluster(pieces(integral_constant<int, 0>()), 1, sums);
    }
    if (PROBS) {
        // a probability that is none, anywhere in the row
        Sums of;
        if (over_cluster(bad ? 1.0 : 0.0, 2, of) > 0.0 || !(total > 0.0)) {
            if (rank == 0) {
                put_largest<L>(row, a.V, a.out + stop);
                if (tid == 0 && a.err) atomicOr(a.err, kErrValue);
            }
            cluster_sync();  // no CTA leaves while others read its sums
            return;
        }
    }
    // ---- of n parts, the one that has the goal in it (by the rounding of the sums alone, none: the last that has any)
    const double goal = (double)in_unit(a.u[end - 1]) * total;
    double before = 0.0;
    auto find = [&](const auto& part, auto parts) {
        int owner = -1, some = 0;
        double at = before, at_some = before, sum = before;
#pragma unroll
        for (int k = 0; k < decltype(parts)::value; ++k) {
            const double x = part(k);
            if (x > 0.0) {
                some = k;
                at_some = sum;
            }
            if (owner < 0 && sum + x > goal) {
                owner = k;
                at = sum;
            }
            sum += x;
        }
        before = owner < 0 ? at_some : at;
        return owner < 0 ? some : owner;
    };
    if (find([&](int k) { return sums[k]; }, integral_constant<int, kMostCluster>()) == (int)rank &&
        find([&](int w) { return sum_s[1][w]; }, integral_constant<int, kDrawWarps>()) == warp) {
        double x = 0.0;  // of piece `lane`
        if (lane < kSubs)
#pragma unroll 8
            for (int k = 0; k < 32; ++k) x += sub_s[warp][lane][(k + lane) % 32];
        const int piece =
            find([&](int k) { return __shfl_sync(0xffffffffu, x, k); }, integral_constant<int, kSubs>());
        const int first = g0 + piece * sub, last = min(g1, first + sub);
        int found = -1, some = min(first * kGroup, a.V - 1);
        for (int g = first; g < last && found < 0; ++g) {
            // kEach rows of 32 elements: the sums along every one of them at once
            float l[kEach], q[kEach] = {};
            get(row, g, kOutside, l);
            if (minus == 1) get(draft, g, 0.0f, q);
            double w[kEach], upto[kEach];
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const int i = g * kGroup + 32 * j + lane;
                w[j] = minus == 1 ? left(integral_constant<int, 1>(), i, l[j], q[j]) : left(integral_constant<int, 0>(), i, l[j], 0.0f);
                if (minus == 2 && i == d) w[j] = 0.0;
                upto[j] = w[j];
            }
#pragma unroll
            for (int o = 1; o < 32; o <<= 1)
#pragma unroll
                for (int j = 0; j < kEach; ++j) {
                    const double y = __shfl_up_sync(0xffffffffu, upto[j], o);
                    if (lane >= o) upto[j] += y;
                }
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const int i0 = g * kGroup + 32 * j;
                const unsigned past = __ballot_sync(0xffffffffu, w[j] > 0.0 && before + upto[j] > goal);
                const unsigned any = __ballot_sync(0xffffffffu, w[j] > 0.0);
                if (past && found < 0) found = i0 + __ffs(past) - 1;
                if (any) some = i0 + 31 - __clz(any);
                before += __shfl_sync(0xffffffffu, upto[j], 31);
            }
        }
        if (lane == 0) a.out[stop] = found >= 0 ? found : some;
    }
    cluster_sync();  // no CTA leaves while others read its sums
}

template <typename L, bool PROBS>
int launch(const VerifyArgs& a, cudaStream_t st) {
    if (a.num_rows > 0) {
        verify_rows<L, PROBS><<<dim3(a.num_rows, a.n_parts), kStatThreads, 0, st>>>(a);
        INFERNT_CUDA_TRY(cudaGetLastError());
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.num_seqs * a.cluster);
    cfg.blockDim = dim3(kDrawThreads);
    cfg.stream = st;
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeClusterDimension;
    attrs[0].val.clusterDim.x = a.cluster;
    attrs[0].val.clusterDim.y = attrs[0].val.clusterDim.z = 1;
    attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attrs;
    cfg.numAttrs = a.num_rows > 0 ? 2 : 1;  // without rows there is no kernel of this call to wait for
    INFERNT_CUDA_TRY(cudaLaunchKernelEx(&cfg, verify_draw<L, PROBS>, static_cast<const VerifyArgs>(a)));
    return INFERNT_OK;
}

}  // namespace
}  // namespace infernt

extern "C" size_t infernt_verify_drafts_workspace_bytes(int num_rows, int num_seqs) {
    (void)num_seqs;
    return num_rows < 1 ? 16 : (size_t)num_rows * infernt::kMostParts * sizeof(infernt::RowPart);
}

extern "C" int infernt_verify_drafts(int* out_tokens, int* accepted, const void* target, long long ld, int target_dtype,
                                     int probabilities, const float* draft_probs, long long draft_ld, const int* tokens,
                                     const int* q_start, int num_seqs, int num_rows, int vocab_size,
                                     const float* temperature, const float* u, const int* kv_len, int* kept,
                                     void* workspace, unsigned* err, void* stream) {
    using namespace infernt;
    const char* op = "verify_drafts";
    INFERNT_REQUIRE(num_seqs >= 0 && num_seqs <= 65535 && num_rows >= 0 && num_rows < kMaxPositions && vocab_size >= 1 &&
                        vocab_size < kMaxPositions,
                    "%s: %d sequences, %d rows of %d", op, num_seqs, num_rows, vocab_size);
    INFERNT_REQUIRE(target_dtype == INFERNT_DTYPE_F32 || target_dtype == INFERNT_DTYPE_BF16 ||
                        target_dtype == INFERNT_DTYPE_F16,
                    "%s: target type %d", op, target_dtype);
    INFERNT_REQUIRE((kv_len != nullptr) == (kept != nullptr), "%s: kv_len with kept", op);
    if (num_seqs == 0) return INFERNT_OK;
    INFERNT_REQUIRE(accepted && q_start, "%s: null pointer", op);
    INFERNT_REQUIRE(num_rows == 0 || (out_tokens && target && tokens && u && workspace), "%s: null pointer", op);
    INFERNT_REQUIRE(ld >= vocab_size && (!draft_probs || draft_ld >= vocab_size), "%s: rows %lld and %lld apart for %d", op,
                    ld, draft_ld, vocab_size);
    INFERNT_REQUIRE(reinterpret_cast<uintptr_t>(target) % (target_dtype == INFERNT_DTYPE_F32 ? 4 : 2) == 0 &&
                        aligned16(workspace),
                    "%s: misaligned target or workspace", op);
    const struct {
        const char* what;
        const void* p;
    } arrays[] = {{"out_tokens", out_tokens}, {"accepted", accepted},       {"draft_probs", draft_probs},
                  {"tokens", tokens},         {"q_start", q_start},         {"temperature", temperature},
                  {"u", u},                   {"kv_len", kv_len},           {"kept", kept},
                  {"err", err},               {"the workspace", workspace}, {"target", target}};
    for (int i = 0; i < 10; ++i)
        INFERNT_REQUIRE(reinterpret_cast<uintptr_t>(arrays[i].p) % 4 == 0, "%s: misaligned %s", op, arrays[i].what);
    const size_t rows4 = 4 * (size_t)num_rows, seqs4 = 4 * (size_t)num_seqs, last = num_rows > 0 ? num_rows - 1 : 0;
    const size_t size = target_dtype == INFERNT_DTYPE_F32 ? 4 : 2, some = num_rows > 0;
    const Span spans[] = {{"out_tokens", out_tokens, rows4, true},
                          {"accepted", accepted, seqs4, true},
                          {"kept", kept, seqs4, true},
                          {"the workspace", workspace, infernt_verify_drafts_workspace_bytes(num_rows, num_seqs) * some, true},
                          {"err", err, 4, true},
                          {"kv_len", kv_len == kept ? nullptr : kv_len, seqs4, false},
                          {"tokens", tokens, rows4, false},
                          {"q_start", q_start, seqs4 + 4, false},
                          {"temperature", temperature, seqs4, false},
                          {"u", u, rows4, false},
                          {"target", target, (last * ld + vocab_size) * size * some, false},
                          {"draft_probs", draft_probs, (last * draft_ld + vocab_size) * 4 * some, false}};
    if (int s = check_apart(op, spans)) return s;
    for (const auto& x : arrays)
        if (int s = check_device_pointer(op, x.what, x.p)) return s;
    VerifyArgs a;
    a.target = target;
    a.draft = draft_probs;
    a.ld = ld;
    a.draft_ld = draft_ld;
    a.tokens = tokens;
    a.q_start = q_start;
    a.temperature = temperature;
    a.u = u;
    a.kv_len = kv_len;
    a.kept = kept;
    a.out = out_tokens;
    a.accepted = accepted;
    a.parts = static_cast<RowPart*>(workspace);
    a.num_seqs = num_seqs;
    a.num_rows = num_rows;
    a.V = vocab_size;
    a.err = err;
    // parts of whole tiles; a row's first vector may start up to 7 elements before it
    const long long tiles = ((long long)vocab_size + 7 + kStatTile - 1) / kStatTile;
    a.part = (int)((tiles + kMostParts - 1) / kMostParts) * kStatTile;
    a.n_parts = (int)(((long long)vocab_size + 7 + a.part - 1) / a.part);
    // as many CTAs a sequence as are sure to run at once: a cluster that has to wait for room waits for another's end
    a.cluster = std::max(1, std::min(kMostCluster, kDrawPerSm * sm_count() / num_seqs));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool p = probabilities != 0;
    if (target_dtype == INFERNT_DTYPE_F32) return p ? launch<float, true>(a, st) : launch<float, false>(a, st);
    if (target_dtype == INFERNT_DTYPE_BF16)
        return p ? launch<__nv_bfloat16, true>(a, st) : launch<__nv_bfloat16, false>(a, st);
    return p ? launch<__half, true>(a, st) : launch<__half, false>(a, st);
}
