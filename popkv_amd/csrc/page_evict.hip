// Eviction from the paged 4-bit K/V cache: sequences cut to the tokens of largest
// weight and the most recent ones, chosen for every layer and KV head by itself.
// Every head keeps as many, so that the rows of one page table go on holding all
// of them; kept rows move to the front of their sequence in their order, and the
// pages behind them are given back.
#include "page_plan.h"

namespace popkv {
namespace {

constexpr int32_t kFresh = -2;  // an entry whose page another sequence holds too: a free one takes its place

// Sequence b by one wave: whether it is cut, its old row kept, its new one with
// the fresh pages still to come, which are counted.
__device__ __forceinline__ void evict_row(const PageEvict& a, int64_t b) {
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t page = int64_t{1} << a.page_log2;
    const int64_t n = clamp_count(a.counts_in[b], a.width << a.page_log2);
    const int64_t k = a.keeps ? clamp_count(a.keeps[b], a.keep) : a.keep;
    const int64_t have = (n + page - 1) >> a.page_log2, stay = (k + page - 1) >> a.page_log2;
    const int32_t* row = a.table_in + b * a.width;
    auto there = [&](int32_t e) { return static_cast<uint32_t>(e) < static_cast<uint32_t>(a.pages); };
    bool cut = n > k, missing = false;
    if (cut) {
        for (int64_t i = lane; i < have; i += kWave) missing = missing || !there(row[i]);
        if (__ballot(missing) != 0) {
            cut = false;
            if (lane == 0 && a.status) atomicOr(a.status, kStatusNoPage);
        }
    }
    int32_t need = 0;
    for (int64_t i = lane; i < a.width; i += kWave) {
        const int32_t e = row[i];
        int32_t now = e;
        if (cut) {
            const bool fresh = i < stay && a.refs_in[e] > 1;
            now = i >= stay ? -1 : fresh ? kFresh : e;
            need += fresh ? 1 : 0;
        }
        a.old[b * a.width + i] = e;
        a.table[b * a.width + i] = now;
    }
    need = static_cast<int32_t>(wave_incl_scan(static_cast<uint32_t>(need), lane));
    if (lane == kWave - 1) {
        a.need[b] = need;
        a.held[b] = static_cast<int32_t>(n);
        a.cut[b] = cut ? static_cast<int32_t>(k) : -1;
    }
}

__global__ __launch_bounds__(256) void evict_rows_kernel(PageEvict a) {
    const int64_t b = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / kWave;
    if (b < a.batch) evict_row(a, b);
}

// Where there are fewer free pages than are needed: need[] (offsets that
// scan_needs made) to offsets of the shares that still fit, in order, -1 for those
// that do not.  By one wave, 64 sequences at a time.
__device__ __forceinline__ void fit_needs(int32_t* need, int64_t batch, int32_t found, int lane) {
    int32_t at = 0;
    for (int64_t b0 = 0; b0 < batch; b0 += kWave) {
        const int64_t b = b0 + lane;
        const int32_t n = b < batch ? need[b + 1] - need[b] : 0;
        int32_t mine = 0;
        for (int i = 0; i < kWave; ++i) {
            const int32_t x = __builtin_amdgcn_readlane(n, i);
            const bool fits = x <= found - at;
            if (i == lane) mine = fits ? at : -1;
            at += fits ? x : 0;
        }
        if (b < batch) need[b] = mine;  // (the next 64 read theirs and those behind)
    }
}

// Fresh pages handed out by one workgroup, lowest first, sequences in order; one
// whose share does not fit in what is left stays as it was, and the next ones go on.
__device__ __forceinline__ void evict_plan(const PageEvict& a, PageMap& map) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int32_t total = scan_needs(a.need, a.batch, map.sh);
    int32_t found = 0;
    if (total > 0)
        found = list_free(map, a.pages, static_cast<int32_t>(min<int64_t>(total, a.pages)), a.list,
                          [&](int64_t i) { return a.refs[i] != 0; });
    if (total > found && wave == 0) fit_needs(a.need, a.batch, found, lane);
    __syncthreads();
    for (int64_t b = wave; b < a.batch; b += kPlanWaves) {
        const int32_t at = a.need[b];
        int32_t* row = a.table + b * a.width;
        const int32_t* old = a.old + b * a.width;
        int32_t cut = a.cut[b];
        if (at < 0) {
            for (int64_t i = lane; i < a.width; i += kWave) row[i] = old[i];
            if (lane == 0) {
                a.cut[b] = -1;
                if (a.status) atomicOr(a.status, kStatusNoPage);
            }
            cut = -1;
        }
        if (cut >= 0) {
            int32_t r = at;
            for (int64_t i0 = 0; i0 < a.width; i0 += kWave) {
                const int64_t i = i0 + lane;
                const int32_t was = i < a.width ? old[i] : -1;
                int32_t now = i < a.width ? row[i] : -1;
                const uint64_t mask = __ballot(now == kFresh);
                if (now == kFresh) {
                    now = a.list[r + __popcll(mask & ((uint64_t{1} << lane) - 1))];
                    row[i] = now;
                    a.refs[now] = 1;
                }
                if (was != now && static_cast<uint32_t>(was) < static_cast<uint32_t>(a.pages)) atomicSub(a.refs + was, 1);
                r += __popcll(mask);
            }
        }
        if (lane == 0) a.counts[b] = cut >= 0 ? cut : a.counts_in[b];
    }
}

__global__ __launch_bounds__(kPlanThreads) void evict_plan_kernel(PageEvict a) {
    __shared__ PageMap map;
    evict_plan(a, map);
}

// The whole plan of a small table.
__global__ __launch_bounds__(kPlanThreads) void evict_alone_kernel(PageEvict a) {
    __shared__ PageMap map;
    if (a.refs != a.refs_in) plan_copy(a.refs_in, a.refs, static_cast<int>(a.pages));
    for (int64_t b = threadIdx.x / kWave; b < a.batch; b += kPlanWaves) evict_row(a, b);
    __syncthreads();
    evict_plan(a, map);
}

// Order of weights: NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
    const uint32_t u = __float_as_uint(w == 0.0f ? 0.0f : w);
    if (w != w) return 0xffffffffu;
    return u >> 31 ? ~u : u | 0x80000000u;
}

constexpr int kEvictThreads = 1024, kEvictWaves = kEvictThreads / kWave;

// One (layer, sequence, KV head) a workgroup: its tokens chosen by a radix select
// over the weights' 32 bits, then moved.  A kept row's place is never behind where
// it was: a tile of rows is read whole before any of it is written, and later
// tiles' rows lie behind everything written so far, so rows move in place.  Bound by
// the rows' stream, 2 (128 + 8R) bytes a kept token, past the caches: 32 layers of 8 heads
// and four sequences cut to 4096 tokens, 1.2 GB read and written, 296 us (4.1 TB/s; through
// the caches 318; a plain copy 4.9 to 5.2), the choice, six passes over the weights in
// L2, before it.
__global__ __launch_bounds__(kEvictThreads) void evict_move_kernel(PageEvict a) {
    __shared__ uint32_t s_hist[kEvictWaves][256];
    __shared__ uint32_t s_pick[2];
    __shared__ uint32_t s_above[kEvictWaves], s_equal[kEvictWaves];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const int64_t layer = blockIdx.y, item = layer * gridDim.x + blockIdx.x;
    const int h = static_cast<int>(blockIdx.x) % a.kv_heads;
    const int64_t b = static_cast<int>(blockIdx.x) / a.kv_heads;
    const float* w_in = a.weights_in + item * a.weight_stride;
    float* w_out = a.weights + item * a.weight_stride;
    int32_t* kept = a.kept + item * a.keep;
    const int k = a.cut[b];
    if (k < 0) {
        for (int64_t i = tid; i < a.keep; i += kEvictThreads) kept[i] = -1;
        if (w_out != w_in)
            for (int64_t i = tid; i < a.weight_stride; i += kEvictThreads) w_out[i] = w_in[i];
        return;
    }
    const int n = a.held[b];
    const int recent = static_cast<int>(min<int64_t>(a.recent, k)), m = n - recent;
    const int choose = k - recent;
    // the smallest key taken, and how many of that key
    uint32_t key = 0, want = static_cast<uint32_t>(choose);
    if (choose > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < kEvictWaves * 256; i += kEvictThreads) (&s_hist[0][0])[i] = 0;
            __syncthreads();
            const uint64_t high = uint64_t{0xffffffffu} << (shift + 8);
            for (int i = tid; i < m; i += kEvictThreads) {
                const uint32_t x = weight_key(w_in[i]);
                if (((x ^ key) & static_cast<uint32_t>(high)) == 0) atomicAdd(&s_hist[wave][x >> shift & 0xff], 1u);
            }
            __syncthreads();
            if (wave == 0) {
                // lane l: keys 255 - 4 l and down
                uint32_t n4[4], sum = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    n4[j] = 0;
                    for (int c = 0; c < kEvictWaves; ++c) n4[j] += s_hist[c][255 - 4 * lane - j];
                    sum += n4[j];
                }
                uint32_t before = wave_incl_scan(sum, lane) - sum;
                if (before < want && want <= before + sum) {
                    int j = 0;
                    while (before + n4[j] < want) before += n4[j++];
                    s_pick[0] = 255 - 4 * lane - j;
                    s_pick[1] = want - before;
                }
            }
            __syncthreads();
            key |= s_pick[0] << shift;
            want = s_pick[1];
            __syncthreads();
        }
        // ascending places: a run of the row a wave
        const int run = (m + kEvictThreads - 1) / kEvictThreads * kWave, lo = min(m, wave * run), hi = min(m, lo + run);
        uint32_t above = 0, equal = 0;
        for (int i = lo + lane; i < hi; i += kWave) {
            const uint32_t x = weight_key(w_in[i]);
            above += x > key ? 1 : 0;
            equal += x == key ? 1 : 0;
        }
        above = wave_incl_scan(above, lane);
        equal = wave_incl_scan(equal, lane);
        if (lane == kWave - 1) {
            s_above[wave] = above;
            s_equal[wave] = equal;
        }
        __syncthreads();
        above = equal = 0;
        for (int c = 0; c < wave; ++c) {
            above += s_above[c];
            equal += s_equal[c];
        }
        for (int i0 = lo; i0 < hi; i0 += kWave) {
            const int i = i0 + lane;
            const uint32_t x = i < hi ? weight_key(w_in[i]) : 0u;
            const uint64_t up = __ballot(i < hi && x > key), eq = __ballot(i < hi && x == key);
            const uint64_t below = (uint64_t{1} << lane) - 1;
            const uint32_t e = equal + __popcll(eq & below), at = above + __popcll(up & below) + min(e, want);
            if (i < hi && (x > key || (x == key && e < want))) kept[at] = i;
            above += __popcll(up);
            equal += __popcll(eq);
        }
    }
    for (int64_t i = choose + tid; i < a.keep; i += kEvictThreads)
        kept[i] = i < k ? static_cast<int32_t>(i) - choose + m : -1;
    __syncthreads();

    // eight lanes a row: sixteen bytes of codes each, of scales the first ones
    constexpr int AHEAD = 4, PASS = kEvictThreads / 8;
    const int part = tid & 7;
    const int32_t* from = a.old + b * a.width;
    const int32_t* to = a.table + b * a.width;
    const int64_t plane = layer * a.pages * a.kv_heads + h;
    const int in_page = (1 << a.page_log2) - 1;
    auto row_of = [&](const int32_t* row, int t) {
        return ((plane + static_cast<int64_t>(row[t >> a.page_log2]) * a.kv_heads) << a.page_log2) + (t & in_page);
    };
    for (int j0 = 0; j0 < k; j0 += AHEAD * PASS) {
        u32x4 codes[AHEAD], scales[AHEAD];
        float w[AHEAD];
        int64_t src[AHEAD], dst[AHEAD];
#pragma unroll
        for (int p = 0; p < AHEAD; ++p) {
            const int j = j0 + p * PASS + tid / 8;
            src[p] = dst[p] = 0;
            if (j < k) {
                const int i = kept[j];
                src[p] = row_of(from, i);
                dst[p] = row_of(to, j);
                if (part == 7) w[p] = w_in[i];
                if (src[p] != dst[p]) {
                    codes[p] = load_once(a.codes + src[p] * kCodeRow + 16 * part);
                    if (4 * part < a.scale_words)
                        scales[p] = load_once(a.scales + src[p] * a.scale_words + 4 * part);
                }
            }
        }
        // every wave's rows are there before the first is written
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
#pragma unroll
        for (int p = 0; p < AHEAD; ++p) {
            const int j = j0 + p * PASS + tid / 8;
            if (j < k) {
                if (part == 7) w_out[j] = w[p];
                if (src[p] != dst[p]) {
                    store_once(a.codes + dst[p] * kCodeRow + 16 * part, codes[p]);
                    if (4 * part < a.scale_words)
                        store_once(a.scales + dst[p] * a.scale_words + 4 * part, scales[p]);
                }
            }
        }
    }
    __syncthreads();
    for (int64_t i = k + tid; i < a.weight_stride; i += kEvictThreads) w_out[i] = 0.0f;
}

}  // namespace

hipError_t launch_page_evict(const PageEvict& a, hipStream_t s) {
    if (plan_alone(a.batch, a.width, a.pages)) {
        hipLaunchKernelGGL(evict_alone_kernel, dim3(1), dim3(kPlanThreads), 0, s, a);
    } else {
        if (a.refs != a.refs_in) {
            const hipError_t e = copy_words(a.refs_in, a.refs, a.pages, s);
            if (e != hipSuccess) return e;
        }
        hipLaunchKernelGGL(evict_rows_kernel, dim3(static_cast<unsigned>((a.batch + 3) / 4)), dim3(256), 0, s, a);
        hipLaunchKernelGGL(evict_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a);
    }
    hipLaunchKernelGGL(evict_move_kernel, dim3(static_cast<unsigned>(a.batch * a.kv_heads), static_cast<unsigned>(a.layers)),
                       dim3(kEvictThreads), 0, s, a);
    return hipGetLastError();
}

}  // namespace popkv
