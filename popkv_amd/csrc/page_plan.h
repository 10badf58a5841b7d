// Device pieces shared by the page plans (pages.hip, page_evict.hip): bit maps of
// a pool's used pages, ranks and prefixes over one workgroup.
#pragma once

#include "paged.h"

namespace popkv {
namespace {

// Copies `n` words (the page table's unchanged part of an out-of-place call).
__global__ __launch_bounds__(256) void copy_words_kernel(const uint32_t* src, uint32_t* dst, int64_t n) {
    const int64_t step = int64_t{256} * gridDim.x;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += step) dst[i] = src[i];
}

unsigned blocks_for(int64_t n, int64_t per, int64_t most) {
    const int64_t b = (n + per - 1) / per;
    return static_cast<unsigned>(b < 1 ? 1 : b > most ? most : b);
}

hipError_t copy_words(const void* src, void* dst, int64_t n, hipStream_t s) {
    hipLaunchKernelGGL(copy_words_kernel, dim3(blocks_for(n, 1024, 1024)), dim3(256), 0, s,
                       static_cast<const uint32_t*>(src), static_cast<uint32_t*>(dst), n);
    return hipGetLastError();
}

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / kWave;

// Exclusive prefix over the block of one value a wave (lane-uniform), and the
// total; sh holds kPlanWaves words and is free again on return.
__device__ __forceinline__ int32_t plan_prefix(int32_t v, int32_t* sh, int32_t& total) {
    const int wave = threadIdx.x / kWave;
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) sh[wave] = v;
    __syncthreads();
    int32_t base = 0;
    total = 0;
    for (int w = 0; w < kPlanWaves; ++w) {
        base += w < wave ? sh[w] : 0;
        total += sh[w];
    }
    __syncthreads();
    return base;
}

// Copies `n` words by the whole workgroup.  (Loads come in batches before their
// stores: the compiler cannot know that the two do not overlap.)
__device__ __forceinline__ void plan_copy(const int32_t* src, int32_t* dst, int n) {
    constexpr int AHEAD = 8;
    for (int i0 = threadIdx.x; i0 < n; i0 += AHEAD * kPlanThreads) {
        int32_t x[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) x[j] = i0 + j * kPlanThreads < n ? src[i0 + j * kPlanThreads] : 0;
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            if (i0 + j * kPlanThreads < n) dst[i0 + j * kPlanThreads] = x[j];
    }
}

// The used pages of a part of the pool as bits in LDS, with how many lie before
// each word: any page's rank among the used or the free ones is a popcount
// away.  A pool of more than kMapPages goes through it part by part.
constexpr int kMapPages = 65536, kMapWords = kMapPages / 64;
static_assert(kMapWords == kPlanThreads);
struct PageMap {
    uint64_t words[kMapWords];
    int32_t before[kMapWords];
    int32_t sh[kPlanWaves];
};
// Builds the map of pages [first, first + kMapPages) of a pool; returns the used
// pages there.  Every thread of the block calls it.
template <typename F>
__device__ __forceinline__ int32_t map_pages(PageMap& m, int64_t first, int64_t pages, F&& used) {
    const int lane = threadIdx.x & (kWave - 1);
    const int n = static_cast<int>(min<int64_t>(kMapPages, pages - first));
    __syncthreads();  // nothing reads the last part's any more
    constexpr int AHEAD = 8;  // loads on their way at once
    static_assert(kMapPages % (AHEAD * kPlanThreads) == 0);
    for (int i0 = 0; i0 < n; i0 += AHEAD * kPlanThreads) {
        bool u[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int i = i0 + j * kPlanThreads + threadIdx.x;
            u[j] = i < n && used(first + i);
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const uint64_t bits = __ballot(u[j]);
            if (lane == 0) m.words[(i0 + j * kPlanThreads + threadIdx.x) / 64] = bits;
        }
    }
    __syncthreads();
    const int32_t v = static_cast<int>(threadIdx.x) * 64 < n ? __popcll(m.words[threadIdx.x]) : 0;
    const int32_t incl = static_cast<int32_t>(wave_incl_scan(static_cast<uint32_t>(v), lane));
    int32_t total;
    const int32_t base = plan_prefix(__builtin_amdgcn_readlane(incl, kWave - 1), m.sh, total);
    m.before[threadIdx.x] = base + incl - v;
    __syncthreads();
    return total;
}
// Used pages of the mapped part before page i of it.
__device__ __forceinline__ int32_t used_before(const PageMap& m, int i) {
    return m.before[i / 64] + __popcll(m.words[i / 64] & ((uint64_t{1} << (i & 63)) - 1));
}

// The lowest `want` pages without a reference, ascending, to list; returns how
// many there are in all.  Every thread of the block calls it.
template <typename F>
__device__ __forceinline__ int32_t list_free(PageMap& m, int64_t pages, int32_t want, int32_t* list, F&& used) {
    int32_t found = 0;
    for (int64_t first = 0; first < pages; first += kMapPages) {
        const int n = static_cast<int>(min<int64_t>(kMapPages, pages - first));
        const int32_t total = map_pages(m, first, pages, used);
        if (found < want)
            for (int i = threadIdx.x; i < n; i += kPlanThreads) {
                const int32_t r = found + i - used_before(m, i);
                if (!(m.words[i / 64] >> (i & 63) & 1) && r < want) list[r] = static_cast<int32_t>(first + i);
            }
        found += n - total;
    }
    return found;
}

// need[] to exclusive offsets in place (kept in global memory), total returned.
__device__ __forceinline__ int32_t scan_needs(int32_t* need, int64_t batch, int32_t* sh) {
    const int lane = threadIdx.x & (kWave - 1);
    int32_t base = 0;
    for (int64_t b0 = 0; b0 < batch; b0 += kPlanThreads) {
        const int64_t b = b0 + threadIdx.x;
        const int32_t v = b < batch ? need[b] : 0;
        const int32_t incl = static_cast<int32_t>(wave_incl_scan(static_cast<uint32_t>(v), lane));
        const int32_t wave_total = __builtin_amdgcn_readlane(incl, kWave - 1);
        int32_t total;
        const int32_t at = base + plan_prefix(wave_total, sh, total) + incl - v;
        if (b < batch) need[b] = at;
        base += total;
    }
    if (threadIdx.x == 0) need[batch] = base;
    __syncthreads();
    return base;
}

// Tables and pools up to which one workgroup does the whole plan, a thread a
// sequence, a table entry and a page: a launch or two saved are worth more than
// the other CUs.  Reserve and fork, alone against in several launches (us, with
// the pages moved): 64 sequences of 14 entries over 1031 pages 6.2 and 12.5, 9.2
// and 14.0; 128 of 113 over 8100 18.1 and 20.7, 14.2 and 18.9; 8 of 1876 16.2 and
// 15.5, 13.6 and 32.3; 512 of 26 19.2 and 47, 16.5 and 30.
constexpr int64_t kPlanAlone = 16384;

bool plan_alone(int64_t batch, int64_t width, int64_t pages) {
    return batch <= kPlanThreads && batch * width <= kPlanAlone && pages <= kPlanAlone;
}

}  // namespace
}  // namespace popkv
