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

// Sums of N values over the threads before this one, and of all; by all
// threads of the block.
template <int N>
__device__ __forceinline__ void block_scan(long long (&v)[N], long long (&all)[N], long long (*sums)[32]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long x[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        x[n] = v[n];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x[n], o);
            if (lane >= o) x[n] += y;
        }
    }
    __syncthreads();
    if (lane == 31)
#pragma unroll
        for (int n = 0; n < N; ++n) sums[n][warp] = x[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
        long long w = sums[n][lane];  // of warp `lane`
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += y;
        }
        all[n] = __shfl_sync(0xffffffffu, w, 31);
        const long long before = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
        v[n] = x[n] - v[n] + (warp ? before : 0);
    }
}

// n >= 0 modulo the ring's size; more than once around it only when held is
// not what the sequences were given.
__device__ __forceinline__ int wrap(long long n, int size) {
    if (n < size) return (int)n;
    n -= size;
    return (int)(n < size ? n : n % size);
}

// What a sequence's pages and rows come to.
struct Move {
    int s, held, need;    // pages before and after
    long long take, give; // places in the ring: the first page taken, the first given back
    int len, n, row0;     // positions kept, new tokens, the first row
};

// Pages [i0, i0 + step, ...) of a move.
__device__ __forceinline__ void move_pages(const PlanArgs& a, const Move& m, int i0, int step) {
    int* row = a.table + (size_t)m.s * a.stride;
#pragma unroll 4
    for (int i = m.held + i0; i < m.need; i += step) row[i] = a.ring[wrap(m.take + (i - m.held), a.num_pages)];
#pragma unroll 4
    for (int i = m.need + i0; i < m.held; i += step) {
        a.ring[wrap(m.give + (i - m.need), a.num_pages)] = row[i];
        row[i] = -1;
    }
}

// Row r's position and slot; the page is in its table entry.
__device__ __forceinline__ void put_row(const PlanArgs& a, int s, int pos, int r) {
    if (a.positions) a.positions[r] = pos;
    if (a.slots) {
        const int pi = a.by_page(pos);
        a.slots[r] = a.table[(size_t)s * a.stride + pi] * a.page_size + (pos - pi * a.page_size);
    }
}
__device__ __forceinline__ void move_rows(const PlanArgs& a, const Move& m, int i0, int step) {
    for (int i = i0; i < m.n; i += step) put_row(a, m.s, m.len + i, m.row0 + i);
}

// One CTA: the scans need every sequence, and up to 1024 of them are one round
// of loads.  A sequence's pages and rows are its thread's; where they are more
// than kOwn, its warp's.  Latency-bound: loads, two scans, the ring's loads,
// stores.
constexpr int kOwn = 4;

__global__ void __launch_bounds__(kPlanThreads) paged_plan(const PlanArgs a) {
    __shared__ long long sums[3][32];
    pdl_launch_dependents();  // paged_plan_rows waits for this kernel's end
    const int tid = threadIdx.x, lane = tid & 31;
    const int head = a.state[0], count = a.state[1];
    const bool sane = head >= 0 && head < a.num_pages && count >= 0 && count <= a.num_pages;
    long long rows_wanted = 0, pages_wanted = 0, rows = 0, taken = 0, given = 0;
    unsigned err = sane ? 0u : kErrBatch;
    for (int base = 0; base < a.num_seqs; base += kPlanThreads) {
        const int s = base + tid;
        Move m = {s, 0, 0, 0, 0, 0, 0, 0};
        bool fine = false;
        if (s < a.num_seqs) {
            m.len = a.len[s];
            m.n = a.new_len[s];
            m.held = a.held[s];
            const long long end = (long long)m.len + m.n;
            fine = m.len >= 0 && m.n >= 0 && end <= kMaxPositions && end <= (long long)a.stride * a.page_size &&
                   m.held >= 0 && m.held <= a.stride;
            if (!fine) err |= kErrBatch;
            fine = fine && sane;
            if (fine) m.need = a.by_page((int)end + a.page_size - 1);
        }
        long long want[2] = {fine ? m.n : 0, fine && m.need > m.held ? m.need - m.held : 0}, all[2];
        const long long own[2] = {want[0], want[1]};
        block_scan<2>(want, all, sums);
        const bool waits = (own[1] > 0 && pages_wanted + want[1] + own[1] > count) ||
                           (own[0] > 0 && rows_wanted + want[0] + own[0] > a.max_rows);
        rows_wanted += all[0];
        pages_wanted += all[1];
        if (waits) err |= kErrNoRoom;
        if (!fine || waits) {
            m.n = 0;
            m.need = m.held;
        }
        long long sum[3] = {m.n, m.need > m.held ? m.need - m.held : 0, m.held > m.need ? m.held - m.need : 0}, tot[3];
        __syncthreads();  // sums is read
        block_scan<3>(sum, tot, sums);
        m.row0 = (int)(rows + sum[0]);
        m.take = head + taken + sum[1];
        m.give = (long long)head + count + given + sum[2];
        rows += tot[0];
        taken += tot[1];
        given += tot[2];
        if (s < a.num_seqs) {
            a.q_start[s + 1] = m.row0 + m.n;
            a.kv_len[s] = m.len + m.n;
            if (m.need != m.held) a.held[s] = m.need;
        }
        // pages, then rows: by their thread, or all 32 lanes on one sequence after the other
        const int pages = abs(m.need - m.held), here = a.rows_here ? m.n : 0;
        const bool many = pages > kOwn || here > kOwn;
        if (!many) {
            move_pages(a, m, 0, 1);
            if (here) move_rows(a, m, 0, 1);
        }
        for (unsigned left = __ballot_sync(0xffffffffu, many); left; left &= left - 1) {
            const int k = __ffs(left) - 1;
            Move o;
            o.s = __shfl_sync(0xffffffffu, m.s, k);
            o.held = __shfl_sync(0xffffffffu, m.held, k);
            o.need = __shfl_sync(0xffffffffu, m.need, k);
            o.take = __shfl_sync(0xffffffffu, m.take, k);
            o.give = __shfl_sync(0xffffffffu, m.give, k);
            o.len = __shfl_sync(0xffffffffu, m.len, k);
            o.n = __shfl_sync(0xffffffffu, m.n, k);
            o.row0 = __shfl_sync(0xffffffffu, m.row0, k);
            move_pages(a, o, lane, 32);
            __syncwarp();  // the table's new entries are seen by all lanes
            if (a.rows_here) move_rows(a, o, lane, 32);
        }
        __syncthreads();  // sums is read
    }
    if (tid == 0) {
        a.q_start[0] = 0;
        if (sane) {
            a.state[0] = (int)((head + taken) % a.num_pages);
            a.state[1] = (int)min((long long)count - taken + given, (long long)0x7fffffff);
        }
    }
    if (a.err && err) atomicOr(a.err, err);
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
    INFERNT_REQUIRE(kv_len != new_len || t->num_seqs == 0, "%s: kv_len may not be new_len", op);
    const struct {
        const char* what;
        const void* p;
    } arrays[] = {{"block_table", t->block_table}, {"held", t->held},           {"free_pages", t->free_pages},
                  {"state", t->state},             {"len", len},                {"new_len", new_len},
                  {"q_start", q_start},            {"kv_len", kv_len},          {"positions", positions},
                  {"slots", slots},                {"err", err}};
    for (const auto& x : arrays)
        INFERNT_REQUIRE(reinterpret_cast<uintptr_t>(x.p) % 4 == 0, "%s: misaligned %s", op, x.what);
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
