// page_tables.cu — block tables, lengths and slots of a step's batch from the
// lengths on the device: which pages each sequence takes and gives back, where
// its new tokens are.
//
// With need_s = ceil((len_s + new_s) / page_size), more_s = need_s - held_s:
//   s waits when more_s > 0 and sum_{t <= s} max(more_t, 0) > free pages, or
//   when new_s > 0 and sum_{t <= s} new_t > max_rows;
//   q_start, the places of taken pages in the ring and those of pages given
//   back are sums over the sequences before s that do not wait.
// Nothing depends on the order of threads: the sums are scans, and the pages
// taken (from the front of the ring) and given back (to its end) are disjoint.
#include <cstdint>

#include "paged.cuh"

namespace infernt {
namespace {

constexpr int kPlanThreads = 1024;
// Up to so many row places the one CTA writes the rows itself; a second launch
// would take longer.
constexpr int kRowsInPlace = 4096;

struct PlanArgs {
    int* table;
    int* held;
    int* ring;
    int* state;
    const int* len;
    const int* new_len;
    int* q_start;
    int* kv_len;
    int* positions;
    int* slots;
    int num_seqs, num_pages, page_size, stride, max_rows;
    bool rows_here;
    FastDiv by_page;
    unsigned* err;
};

// Sums that stay at kMost once they are there: such a sum is past every limit
// that it is held to, and of numbers that no caller can mean.
constexpr unsigned kMost = 0x7fffffffu;
__device__ __forceinline__ unsigned add(unsigned a, unsigned b) { return min(a + b, kMost); }

// Sums of N values over the threads before this one, and of all; by all
// threads of the block.
template <int N>
__device__ __forceinline__ void block_scan(unsigned (&v)[N], unsigned (&all)[N], unsigned (*sums)[32]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned x[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        x[n] = v[n];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, x[n], o);
            if (lane >= o) x[n] = add(x[n], y);
        }
        if (lane == 31) sums[n][warp] = x[n];
        x[n] = __shfl_up_sync(0xffffffffu, x[n], 1);
        if (lane == 0) x[n] = 0;
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
        unsigned w = sums[n][lane];  // of warp `lane`
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w = add(w, y);
        }
        all[n] = __shfl_sync(0xffffffffu, w, 31);
        const unsigned before = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
        v[n] = warp ? add(x[n], before) : x[n];
    }
}

// a + b modulo the ring's size, a below it.  b is more than once around it only
// when held is not what the sequences were given.
__device__ __forceinline__ int wrap(unsigned a, unsigned b, int size) {
    if (b >= (unsigned)size) b %= (unsigned)size;
    const unsigned x = a + b;
    return (int)(x < (unsigned)size ? x : x - (unsigned)size);
}

// 1024 sequences: what the places among their rows, pages taken and pages given
// back are found by.
struct Chunk {
    int len[kPlanThreads], held[kPlanThreads], need[kPlanThreads];
    unsigned row[kPlanThreads], take[kPlanThreads], give[kPlanThreads];  // sums before each
};
// The last sequence of the chunk whose sum before is at most x (one with sums
// above it then begins at it).
__device__ __forceinline__ int owner(const unsigned* before, unsigned x) {
    int at = 0;
#pragma unroll
    for (int step = kPlanThreads / 2; step > 0; step /= 2)
        if (before[at + step] <= x) at += step;
    return at;
}

// One CTA: the scans need every sequence, and up to 1024 of them are one round
// of loads.  Rows and pages are then dealt evenly to the threads, whoever's they
// are.  A page that a sequence takes is read from the ring wherever it is
// needed, so nothing waits for a store.  Latency-bound: loads, two scans, a
// search of ten steps, the ring's and the table's loads, stores.  The step of 256
// sequences takes 5 us (7 from a cold cache), 100 prompts 13 and 5 for their
// rows.  (A thread or a warp a sequence took 20 and 85.)
__global__ void __launch_bounds__(kPlanThreads) paged_plan(const PlanArgs a) {
    pdl_launch_dependents();  // paged_plan_rows waits for this kernel's end
    __shared__ unsigned sums[3][32];
    __shared__ Chunk ch;
    const int tid = threadIdx.x;
    const int head = a.state[0], count = a.state[1];
    const bool sane = head >= 0 && head < a.num_pages && count >= 0 && count <= a.num_pages;
    const unsigned tail = sane ? (unsigned)wrap(head, count, a.num_pages) : 0u;
    unsigned rows_wanted = 0, pages_wanted = 0, rows = 0, taken = 0, given = 0;
    unsigned err = sane ? 0u : kErrBatch;
    for (int base = 0; base < a.num_seqs; base += kPlanThreads) {
        const int s = base + tid;
        int len = 0, n = 0, held = 0, need = 0;
        bool fine = false;
        if (s < a.num_seqs) {
            len = a.len[s];
            n = a.new_len[s];
            held = a.held[s];
            const long long end = (long long)len + n;
            fine = len >= 0 && n >= 0 && end <= kMaxPositions && end <= (long long)a.stride * a.page_size && held >= 0 &&
                   held <= a.stride;
            if (!fine) err |= kErrBatch;
            fine = fine && sane;
            if (fine) need = a.by_page((int)end + a.page_size - 1);
        }
        const unsigned own_rows = fine ? n : 0, own_pages = fine ? max(need - held, 0) : 0;
        unsigned want[2] = {own_rows, own_pages}, all[2];
        block_scan<2>(want, all, sums);
        const bool waits = (own_pages > 0 && add(pages_wanted, add(want[1], own_pages)) > (unsigned)count) ||
                           (own_rows > 0 && add(rows_wanted, add(want[0], own_rows)) > (unsigned)a.max_rows);
        rows_wanted = add(rows_wanted, all[0]);
        pages_wanted = add(pages_wanted, all[1]);
        if (waits) err |= kErrNoRoom;
        if (!fine || waits) {
            n = 0;
            need = held;
        }
        unsigned sum[3] = {(unsigned)n, (unsigned)max(need - held, 0), (unsigned)max(held - need, 0)}, tot[3];
        __syncthreads();  // sums is read
        block_scan<3>(sum, tot, sums);
        ch.len[tid] = len;
        ch.held[tid] = held;
        ch.need[tid] = need;
        ch.row[tid] = sum[0];
        ch.take[tid] = sum[1];
        ch.give[tid] = sum[2];
        if (s < a.num_seqs) {
            a.q_start[s + 1] = (int)(rows + sum[0]) + n;
            a.kv_len[s] = len + n;
            if (need != held) a.held[s] = need;
        }
        __syncthreads();
        // page x of those that the chunk takes: the i-th of sequence o, behind those that it holds
        for (unsigned x = tid; x < tot[1]; x += kPlanThreads) {
            const int o = owner(ch.take, x), i = ch.held[o] + (int)(x - ch.take[o]);
            a.table[(size_t)(base + o) * a.stride + i] = a.ring[wrap(head, taken + x, a.num_pages)];
        }
        // of those that it gives back, behind those that it keeps (a page that was never given: no place for it)
#pragma unroll 4
        for (unsigned x = tid; x < tot[2]; x += kPlanThreads) {
            const int o = owner(ch.give, x), i = ch.need[o] + (int)(x - ch.give[o]);
            int* at = a.table + (size_t)(base + o) * a.stride + i;
            a.ring[wrap(tail, add(given, x), a.num_pages)] = *at;
            *at = -1;
        }
        if (a.rows_here)
            for (unsigned x = tid; x < tot[0]; x += kPlanThreads) {
                const int o = owner(ch.row, x), pos = ch.len[o] + (int)(x - ch.row[o]);
                const int r = (int)(rows + x);
                if (a.positions) a.positions[r] = pos;
                if (a.slots) {
                    const int pi = a.by_page(pos), held_o = ch.held[o];
                    const int page = pi < held_o ? a.table[(size_t)(base + o) * a.stride + pi]
                                                 : a.ring[wrap(head, taken + ch.take[o] + (pi - held_o), a.num_pages)];
                    a.slots[r] = page * a.page_size + (pos - pi * a.page_size);
                }
            }
        rows += tot[0];
        taken += tot[1];
        given = add(given, tot[2]);
        __syncthreads();  // sums and ch are read
    }
    if (tid == 0) {
        a.q_start[0] = 0;
        if (sane) {
            a.state[0] = wrap(head, taken, a.num_pages);
            a.state[1] = (int)add((unsigned)count - taken, given);
        }
    }
    if (a.err && err) atomicOr(a.err, err);
}

// Row r's position and slot; the page is in its table entry.
__device__ __forceinline__ void put_row(const PlanArgs& a, int s, int pos, int r) {
    if (a.positions) a.positions[r] = pos;
    if (a.slots) {
        const int pi = a.by_page(pos);
        a.slots[r] = a.table[(size_t)s * a.stride + pi] * a.page_size + (pos - pi * a.page_size);
    }
}

// The rows' positions and slots, by all SMs: a thread a row; a warp whose rows
// are one sequence's looks for it once.
constexpr int kRowThreads4 = 256;

__global__ void __launch_bounds__(kRowThreads4) paged_plan_rows(const PlanArgs a) {
    pdl_wait();  // paged_plan's arrays
    const int total = a.q_start[a.num_seqs], lane = threadIdx.x & 31;
    for (int w0 = blockIdx.x * kRowThreads4 + (threadIdx.x & ~31); w0 < total; w0 += gridDim.x * kRowThreads4) {
        int s = find_seq(a.q_start, a.num_seqs, w0);
        const int r = w0 + lane;
        if (r < total && a.q_start[s + 1] <= r) {  // a later sequence's
            int hi = a.num_seqs;
            while (hi - s > 1) {
                const int mid = (s + hi) / 2;
                if (a.q_start[mid] <= r)
                    s = mid;
                else
                    hi = mid;
            }
        }
        __syncwarp();
        if (r < total) put_row(a, s, a.kv_len[s] - (a.q_start[s + 1] - r), r);
    }
}

}  // namespace
}  // namespace infernt

extern "C" int infernt_paged_batch_plan(const infernt_page_tables* t, const int* len, const int* new_len, int* q_start,
                                        int* kv_len, int* positions, int* slots, int max_rows, unsigned* err,
                                        void* stream) {
    using namespace infernt;
    const char* op = "paged_batch_plan";
    INFERNT_REQUIRE(t && t->free_pages && t->state && q_start, "%s: null pointer", op);
    INFERNT_REQUIRE(t->num_seqs >= 0 && t->num_seqs <= 65535 && t->num_pages >= 1 && t->page_size >= 1 &&
                        t->table_stride >= 0 && max_rows >= 0 && max_rows < kMaxPositions,
                    "%s: %d sequences, %d pages of %d positions, table rows of %d, %d rows", op, t->num_seqs,
                    t->num_pages, t->page_size, t->table_stride, max_rows);
    INFERNT_REQUIRE((long long)t->num_pages * t->page_size < (1ll << 31) && t->page_size < kMaxPositions,
                    "%s: a pool of 2^31 slots or more", op);
    INFERNT_REQUIRE(t->num_seqs == 0 || (len && new_len && kv_len && t->held && (t->block_table || t->table_stride == 0)),
                    "%s: null pointer", op);
    const struct {
        const char* what;
        const void* p;
    } arrays[] = {{"block_table", t->block_table}, {"held", t->held},           {"free_pages", t->free_pages},
                  {"state", t->state},             {"len", len},                {"new_len", new_len},
                  {"q_start", q_start},            {"kv_len", kv_len},          {"positions", positions},
                  {"slots", slots},                {"err", err}};
    for (const auto& x : arrays)
        INFERNT_REQUIRE(reinterpret_cast<uintptr_t>(x.p) % 4 == 0, "%s: misaligned %s", op, x.what);
    const size_t seqs4 = 4 * (size_t)t->num_seqs, rows4 = 4 * (size_t)max_rows;
    const Span spans[] = {{"block_table", t->block_table, seqs4 * t->table_stride, true},
                          {"held", t->held, seqs4, true},
                          {"free_pages", t->free_pages, 4 * (size_t)t->num_pages, true},
                          {"state", t->state, 16, true},
                          {"q_start", q_start, seqs4 + 4, true},
                          {"kv_len", kv_len, seqs4, true},
                          {"positions", positions, rows4, true},
                          {"slots", slots, rows4, true},
                          {"err", err, 4, true},
                          {"len", len == kv_len ? nullptr : len, seqs4, false},
                          {"new_len", new_len, seqs4, false}};
    if (int s = check_apart(op, spans)) return s;
    for (const auto& x : arrays)
        if (int s = check_device_pointer(op, x.what, x.p)) return s;
    PlanArgs a;
    a.table = t->block_table;
    a.held = t->held;
    a.ring = t->free_pages;
    a.state = t->state;
    a.len = len;
    a.new_len = new_len;
    a.q_start = q_start;
    a.kv_len = kv_len;
    a.positions = positions;
    a.slots = slots;
    a.num_seqs = t->num_seqs;
    a.num_pages = t->num_pages;
    a.page_size = t->page_size;
    a.stride = t->table_stride;
    a.max_rows = max_rows;
    a.by_page = fast_div(t->page_size);
    a.err = err;
    const bool rows = (positions || slots) && max_rows > 0 && t->num_seqs > 0;
    a.rows_here = rows && max_rows <= kRowsInPlace;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    paged_plan<<<1, kPlanThreads, 0, st>>>(a);
    INFERNT_CUDA_TRY(cudaGetLastError());
    if (!rows || a.rows_here) return INFERNT_OK;
    cudaLaunchConfig_t cfg = {};
    const int blocks = (max_rows + kRowThreads4 - 1) / kRowThreads4, most = sm_count() * 8;
    cfg.gridDim = dim3(blocks < most ? blocks : most);
    cfg.blockDim = dim3(kRowThreads4);
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    INFERNT_CUDA_TRY(cudaLaunchKernelEx(&cfg, paged_plan_rows, static_cast<const PlanArgs>(a)));
    return INFERNT_OK;
}
