// page_pool.cpp — which sequence holds which pages of a paged cache: pages
// counted by their holders, shared by forks, copied before a write to a
// shared one, compacted to the front of the pool.  Host logic only; the
// copies that it reports are run by infernt_pages_copy.  The reference keeps
// one contiguous cache of one sequence (include/kv_cache.h:7-15).
#include <new>
#include <vector>

#include "../../../include/infernt_capi.h"
#include "../internal.h"

using infernt::fail;

struct infernt_page_pool {
    int page_size = 0;
    std::vector<int> holders;             // [num_pages] sequences that hold the page
    std::vector<std::vector<int>> pages;  // [max_seqs]
    int n_free = 0;
    int lowest = 0;  // no page below it is free

    int pages_for(int n_positions) const {
        return n_positions / page_size + (n_positions % page_size != 0);
    }
    // the lowest free page (there must be one)
    int take() {
        while (holders[lowest] > 0) ++lowest;
        holders[lowest] = 1;
        --n_free;
        return lowest;
    }
    void give(int p) {
        if (--holders[p] > 0) return;
        ++n_free;
        if (p < lowest) lowest = p;
    }
};

namespace {

// Runs f; a host allocation that fails becomes a status, not an exception.
template <typename F>
int guarded(const char* op, F f) {
    try {
        return f();
    } catch (const std::bad_alloc&) {
        return fail(INFERNT_ERR_OUT_OF_MEMORY, "%s: host allocation failed", op);
    }
}

}  // namespace

#define POOL_SEQ(op, s) \
    INFERNT_REQUIRE((s) >= 0 && (s) < (int)pool->pages.size(), op ": sequence %d of %zu", (s), pool->pages.size())

extern "C" {

int infernt_page_pool_create(int num_pages, int page_size, int max_seqs, infernt_page_pool** out) {
    INFERNT_REQUIRE(out, "page_pool_create: null argument");
    *out = nullptr;
    INFERNT_REQUIRE(num_pages >= 1 && page_size >= 1 && max_seqs >= 1,
                    "page_pool_create: %d pages of %d positions, %d sequences", num_pages, page_size, max_seqs);
    infernt_page_pool* p = new (std::nothrow) infernt_page_pool();
    if (!p) return fail(INFERNT_ERR_OUT_OF_MEMORY, "page_pool_create: host allocation failed");
    const int s = guarded("page_pool_create", [&] {
        p->page_size = page_size;
        p->holders.assign(num_pages, 0);
        p->pages.resize(max_seqs);
        p->n_free = num_pages;
        return (int)INFERNT_OK;
    });
    if (s) {
        delete p;
        return s;
    }
    *out = p;
    return INFERNT_OK;
}

int infernt_page_pool_destroy(infernt_page_pool* pool) {
    delete pool;
    return INFERNT_OK;
}

int infernt_page_pool_resize(infernt_page_pool* pool, int seq, int n_positions) {
    INFERNT_REQUIRE(pool, "page_pool_resize: null pool");
    POOL_SEQ("page_pool_resize", seq);
    INFERNT_REQUIRE(n_positions >= 0, "page_pool_resize: %d positions", n_positions);
    std::vector<int>& row = pool->pages[seq];
    const int want = pool->pages_for(n_positions);
    if (want - (int)row.size() > pool->n_free)
        return fail(INFERNT_ERR_OUT_OF_MEMORY, "page_pool_resize: %d pages are free, %d more are needed", pool->n_free,
                    want - (int)row.size());
    return guarded("page_pool_resize", [&] {
        row.reserve(want);
        while ((int)row.size() < want) row.push_back(pool->take());
        while ((int)row.size() > want) {
            pool->give(row.back());
            row.pop_back();
        }
        return (int)INFERNT_OK;
    });
}

int infernt_page_pool_fork(infernt_page_pool* pool, int src_seq, int dst_seq, int n_positions) {
    INFERNT_REQUIRE(pool, "page_pool_fork: null pool");
    POOL_SEQ("page_pool_fork", src_seq);
    POOL_SEQ("page_pool_fork", dst_seq);
    INFERNT_REQUIRE(n_positions >= 0 && pool->pages_for(n_positions) <= (int)pool->pages[src_seq].size(),
                    "page_pool_fork: sequence %d has no pages for %d positions", src_seq, n_positions);
    INFERNT_REQUIRE(src_seq != dst_seq && pool->pages[dst_seq].empty(), "page_pool_fork: sequence %d holds pages",
                    dst_seq);
    return guarded("page_pool_fork", [&] {
        const std::vector<int>& row = pool->pages[src_seq];
        pool->pages[dst_seq].assign(row.begin(), row.begin() + pool->pages_for(n_positions));
        for (int p : pool->pages[dst_seq]) ++pool->holders[p];
        return (int)INFERNT_OK;
    });
}

int infernt_page_pool_write(infernt_page_pool* pool, int seq, int from, int to, int* src, int* dst, int* n) {
    INFERNT_REQUIRE(pool && src && dst && n, "page_pool_write: null argument");
    POOL_SEQ("page_pool_write", seq);
    std::vector<int>& row = pool->pages[seq];
    INFERNT_REQUIRE(from >= 0 && to >= from && pool->pages_for(to) <= (int)row.size(),
                    "page_pool_write: sequence %d has no pages for [%d, %d)", seq, from, to);
    *n = 0;
    if (from == to) return INFERNT_OK;
    const int first = from / pool->page_size, last = (to - 1) / pool->page_size;
    int need = 0;
    for (int i = first; i <= last; ++i) need += pool->holders[row[i]] > 1;
    if (need > pool->n_free)
        return fail(INFERNT_ERR_OUT_OF_MEMORY, "page_pool_write: %d pages are free, %d copies are needed", pool->n_free,
                    need);
    for (int i = first; i <= last; ++i)
        if (pool->holders[row[i]] > 1) {
            const int p = pool->take();
            src[*n] = row[i];
            dst[*n] = p;
            ++*n;
            --pool->holders[row[i]];
            row[i] = p;
        }
    return INFERNT_OK;
}

int infernt_page_pool_compact(infernt_page_pool* pool, int* src, int* dst, int* n) {
    INFERNT_REQUIRE(pool && src && dst && n, "page_pool_compact: null argument");
    *n = 0;
    return guarded("page_pool_compact", [&] {
        const int num = (int)pool->holders.size(), used = num - pool->n_free;
        std::vector<int> moved(num, -1);
        // the pages in use at or above `used` go into the holes below it
        int hole = 0;
        for (int p = num - 1; p >= used; --p)
            if (pool->holders[p] > 0) {
                while (pool->holders[hole] > 0) ++hole;
                src[*n] = p;
                dst[*n] = hole;
                ++*n;
                moved[p] = hole;
                pool->holders[hole] = pool->holders[p];
                pool->holders[p] = 0;
            }
        pool->lowest = used;
        for (std::vector<int>& row : pool->pages)
            for (int& p : row)
                if (moved[p] >= 0) p = moved[p];
        return (int)INFERNT_OK;
    });
}

int infernt_page_pool_pages(infernt_page_pool* pool, int seq, int* pages, int cap, int* n) {
    INFERNT_REQUIRE(pool && n && cap >= 0 && (cap == 0 || pages), "page_pool_pages: null argument");
    POOL_SEQ("page_pool_pages", seq);
    const std::vector<int>& row = pool->pages[seq];
    *n = (int)row.size();
    for (int i = 0; i < *n && i < cap; ++i) pages[i] = row[i];
    return INFERNT_OK;
}

int infernt_page_pool_stats(infernt_page_pool* pool, int* free_pages, int* shared_pages, int* highest) {
    INFERNT_REQUIRE(pool && free_pages && shared_pages && highest, "page_pool_stats: null argument");
    *free_pages = pool->n_free;
    *shared_pages = 0;
    *highest = -1;
    for (int p = 0; p < (int)pool->holders.size(); ++p) {
        *shared_pages += pool->holders[p] > 1;
        if (pool->holders[p] > 0) *highest = p;
    }
    return INFERNT_OK;
}

}  // extern "C"
