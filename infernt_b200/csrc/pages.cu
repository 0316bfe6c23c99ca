// pages.cu — copies of pages of paged caches: page src[i] into page dst[i]
// in every pool (each layer's K and V) of a model, in one launch.  What a
// fork's partly filled page, a copy before a write to a shared page and a
// compaction need.
//
// The list of pages and the pools' addresses travel as kernel parameters, so
// the call needs no device memory of its own, no copy to the device and no
// synchronisation, and a captured call keeps its list.  Bytes: every copied
// page is read once and written once; nothing else moves.
#include <cstdint>
#include <new>
#include <vector>

#include <cudaTypedefs.h>

#include "common.cuh"
#include "internal.h"
#include "paged.cuh"

namespace infernt {
namespace {

constexpr int kCopyThreads = 256;

// Pools and page pairs of one launch (kernel parameters: 32 764 bytes at most).
template <int NP, int NM>
struct CopyList {
    char* pool[NP];
    int2 move[NM];  // (src, dst)
};

// Block (x, y): part x of the pages' bytes of move blockIdx.y; z: the pool.
template <int NP, int NM>
__global__ void __launch_bounds__(kCopyThreads) pages_copy(const __grid_constant__ CopyList<NP, NM> list,
                                                           size_t page_bytes) {
    const int2 m = list.move[blockIdx.y];
    const uint4* src = reinterpret_cast<const uint4*>(list.pool[blockIdx.z] + (size_t)m.x * page_bytes);
    uint4* dst = reinterpret_cast<uint4*>(list.pool[blockIdx.z] + (size_t)m.y * page_bytes);
    const size_t n = page_bytes / 16;
    for (size_t i = (size_t)blockIdx.x * kCopyThreads + threadIdx.x; i < n; i += (size_t)gridDim.x * kCopyThreads)
        dst[i] = src[i];
}

template <int NP, int NM>
int launch_copy(void* const* pools, int n_pools, size_t page_bytes, const int* src, const int* dst, int n,
                cudaStream_t st) {
    for (int p0 = 0; p0 < n_pools; p0 += NP)
        for (int m0 = 0; m0 < n; m0 += NM) {
            CopyList<NP, NM> list;
            const int np = n_pools - p0 < NP ? n_pools - p0 : NP, nm = n - m0 < NM ? n - m0 : NM;
            for (int i = 0; i < np; ++i) list.pool[i] = static_cast<char*>(pools[p0 + i]);
            for (int i = 0; i < nm; ++i) list.move[i] = make_int2(src[m0 + i], dst[m0 + i]);
            const size_t parts = (page_bytes / 16 + kCopyThreads * 4 - 1) / (kCopyThreads * 4);
            const dim3 grid((unsigned)(parts < 1024 ? parts : 1024), nm, np);
            pages_copy<NP, NM><<<grid, kCopyThreads, 0, st>>>(list, page_bytes);
            INFERNT_CUDA_TRY(cudaGetLastError());
        }
    return INFERNT_OK;
}

// Every pool must be memory that the current device reads in place.  Pools that
// begin in an allocation that has been looked at are: layers of one tensor,
// most often (a look at each of 64 pools takes 8 us, as long as the call).
int check_pools(void* const* pools, int n_pools) {
    static const auto range_of = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuMemGetAddressRange", &f, cudaEnableDefault, &found) != cudaSuccess) f = nullptr;
        return reinterpret_cast<PFN_cuMemGetAddressRange_v3020>(f);
    }();
    CUdeviceptr base = 0;
    size_t bytes = 0;
    for (int i = 0; i < n_pools; ++i) {
        const CUdeviceptr p = reinterpret_cast<CUdeviceptr>(pools[i]);
        if (p >= base && p - base < bytes) continue;
        if (int s = check_device_pointer("pages_copy", "a pool", pools[i])) return s;
        if (i + 1 < n_pools && (!range_of || range_of(&base, &bytes, p) != CUDA_SUCCESS)) bytes = 0;
    }
    return INFERNT_OK;
}

}  // namespace

int pages_copy_launch(void* const* pools, int n_pools, size_t page_bytes, int num_pages, const int* src, const int* dst,
                      int n, bool known, cudaStream_t st) {
    INFERNT_REQUIRE(n_pools >= 0 && n >= 0 && num_pages >= 1, "pages_copy: %d pools of %d pages, %d copies", n_pools,
                    num_pages, n);
    INFERNT_REQUIRE((n_pools == 0 || pools) && (n == 0 || (src && dst)), "pages_copy: null array");
    INFERNT_REQUIRE(page_bytes >= 16 && page_bytes % 16 == 0 && page_bytes <= SIZE_MAX / 2 / (size_t)num_pages,
                    "pages_copy: pages of %zu bytes (a multiple of 16)", page_bytes);
    for (int i = 0; i < n_pools; ++i)
        INFERNT_REQUIRE(pools[i] && aligned16(pools[i]), "pages_copy: pool %d null or not 16-byte aligned", i);
    for (int i = 0; i < n; ++i)
        INFERNT_REQUIRE(src[i] >= 0 && src[i] < num_pages && dst[i] >= 0 && dst[i] < num_pages,
                        "pages_copy: page %d into %d of %d pages", src[i], dst[i], num_pages);
    // a destination written twice, or read too, would depend on the order
    int clash = -1;
    if (n <= 32) {
        for (int i = 0; i < n; ++i)
            for (int j = 0; j < n; ++j)
                if (dst[i] == src[j] || (i != j && dst[i] == dst[j])) clash = dst[i];
    } else {
        try {
            std::vector<char> used((size_t)num_pages, 0);
            for (int i = 0; i < n; ++i) used[src[i]] = 1;
            for (int i = 0; i < n; ++i) {
                if (used[dst[i]]) clash = dst[i];
                used[dst[i]] = 1;
            }
        } catch (const std::bad_alloc&) {
            return fail(INFERNT_ERR_OUT_OF_MEMORY, "pages_copy: host allocation failed");
        }
    }
    INFERNT_REQUIRE(clash < 0, "pages_copy: page %d is a destination twice, or a source too", clash);
    if (n_pools == 0 || n == 0) return INFERNT_OK;
    if (!known)
        if (int s = check_pools(pools, n_pools)) return s;
    // a short list keeps the parameters of a fork's launch small
    if (n_pools <= 64 && n <= 32) return launch_copy<64, 32>(pools, n_pools, page_bytes, src, dst, n, st);
    return launch_copy<256, 2048>(pools, n_pools, page_bytes, src, dst, n, st);
}

}  // namespace infernt

extern "C" int infernt_pages_copy(void* const* pools, int n_pools, size_t page_bytes, int num_pages, const int* src,
                                  const int* dst, int n, void* stream) {
    return infernt::pages_copy_launch(pools, n_pools, page_bytes, num_pages, src, dst, n, false,
                                      static_cast<cudaStream_t>(stream));
}
