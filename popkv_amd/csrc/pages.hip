// The paged 4-bit K/V cache: rows written into and read out of its pages, and
// the pages themselves -- reserved, forked, freed and compacted.  Everything a
// kernel decides (which page is free, who keeps an open page, what moves) is
// decided on the device from the page table, the token counts and the
// reference counts, so a captured graph of these calls stays valid while the
// sequences grow; choices go to the lowest index, so results do not depend on
// the order in which workgroups run.
#include "paged.h"

namespace popkv {
namespace {

// A group's extrema are held in +-57344: then low + 15 * delta, each rounded
// to fp16, stays below fp16's largest value.
constexpr float kScaleLimit = 57344.0f;

// ---- write ----------------------------------------------------------------

// low = fp16(min), delta = fp16((max - low) / 15), code = round((x - low) /
// delta) in 0 .. 15, ties to even, of this lane's eight values; the LPG lanes
// of a group hold its G = 8 * LPG values.  The quotient for delta is taken in
// fp64 (max - low need not fit fp32) and rounded to fp32, then fp16.  A group
// with a NaN or an infinity gets low = NaN: it reads back as NaN.
template <typename T, int LPG>
__device__ __forceinline__ void quantise8(const T* src, uint32_t& code, uint32_t& scale) {
    float x[8];
    load8<T>(src, x);
    float lo = x[0], hi = x[0];
    uint32_t top = 0;  // largest magnitude's bits: infinity and NaN lie above every number
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
        top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    }
    auto fold = [&](auto ctrl) {
        constexpr int C = decltype(ctrl)::value;
        lo = fminf(lo, dpp_mov<C>(lo));
        hi = fmaxf(hi, dpp_mov<C>(hi));
        top = max(top, __float_as_uint(dpp_mov<C>(__uint_as_float(top))));
    };
    fold(std::integral_constant<int, 0xB1>{});
    if constexpr (LPG >= 4) fold(std::integral_constant<int, 0x4E>{});
    if constexpr (LPG >= 8) fold(std::integral_constant<int, 0x141>{});
    if (top >= 0x7f800000u) {
        code = 0;
        scale = 0x7e00u;  // low = NaN, delta = 0
        return;
    }
    lo = fminf(fmaxf(lo, -kScaleLimit), kScaleLimit);
    hi = fminf(fmaxf(hi, -kScaleLimit), kScaleLimit);
    const uint32_t lob = f16_rne(lo);
    const float low = bits_f16(lob);
    const uint32_t deb = f16_rne(static_cast<float>((static_cast<double>(hi) - static_cast<double>(low)) / 15.0));
    const float delta = bits_f16(deb);
    scale = lob | (deb << 16);
    code = 0;
    if (delta == 0.0f) return;
    // fp32 quotients are off by less than 2^-18 (three roundings of at most
    // 2^-24 of a quotient below 16); a value that near a border between two
    // codes is decided in fp64
    const float inv = 1.0f / delta;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float q = fminf(fmaxf((x[i] - low) * inv, 0.0f), 15.0f);
        float r = rintf(q);
        if (fabsf(q - r) > 0.5f - 0x1p-16f)
            r = static_cast<float>(
                rint(fmin(fmax((static_cast<double>(x[i]) - static_cast<double>(low)) / static_cast<double>(delta), 0.0), 15.0)));
        code |= static_cast<uint32_t>(r) << (4 * i);
    }
}

// Sixteen lanes a row (eight dims each), four tokens a wave: the K and the V
// row of a token make one 128-byte line of codes.  Bound by the stream of the
// rows: 2 * 128 * sizeof(T) bytes read, 128 + 8R written per token and head.
template <typename T, int G>
__global__ __launch_bounds__(256) void paged_write_kernel(PagedWrite a, PagedView c) {
    constexpr int R = 128 / G;
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 16 + threadIdx.x / 16;
    const int h = blockIdx.y, b = blockIdx.z;
    const int64_t most = a.tokens ? clamp_count(a.tokens[b], a.rows) : a.rows;
    if (t >= most) return;  // whole 16-lane rows leave
    const int64_t limit = c.width << c.page_log2;
    const int64_t pos = clamp_count(c.counts[b], limit) + t;
    const int64_t entry = pos >> c.page_log2;
    const int32_t page = pos < limit ? c.table[b * c.width + entry] : -1;
    if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(c.pages)) {
        if (a.status && (lane & 15) == 0 && h == 0) atomicOr(a.status, pos < limit ? kStatusNoPage : kStatusFull);
        return;
    }
    const int d = (lane & 15) * 8;
    const int64_t row = ((static_cast<int64_t>(page) * c.kv_heads + h) << c.page_log2) + (pos & ((1 << c.page_log2) - 1));
    uint32_t* codes = reinterpret_cast<uint32_t*>(c.codes + row * kCodeRow);
    uint32_t* scales = c.scales + row * (2 * R);
    const T* src[2] = {static_cast<const T*>(a.k) + b * a.k_bs + h * a.k_hs + t * a.k_ts + d,
                       static_cast<const T*>(a.v) + b * a.v_bs + h * a.v_hs + t * a.v_ts + d};
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        uint32_t code, scale;
        quantise8<T, G / 8>(src[w], code, scale);
        codes[16 * w + (lane & 15)] = code;
        if (d % G == 0) scales[R * w + d / G] = scale;
    }
}

// ---- read -----------------------------------------------------------------

// The inverse: rows [0, count) of every sequence as K/V rows of T; rows past a
// count are cleared when `fill`, else left as they are.
template <typename T, int G>
__global__ __launch_bounds__(256) void paged_read_kernel(PagedRead a, PagedView c) {
    constexpr int R = 128 / G;
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 16 + threadIdx.x / 16;
    const int h = blockIdx.y, b = blockIdx.z;
    if (t >= a.rows) return;
    const int64_t count = clamp_count(c.counts[b], c.width << c.page_log2);
    const int32_t page = t < count ? c.table[b * c.width + (t >> c.page_log2)] : -1;
    const bool live = static_cast<uint32_t>(page) < static_cast<uint32_t>(c.pages);
    if (!live && !a.fill && t >= count) return;
    const int d = (lane & 15) * 8;
    const int64_t row =
        (((live ? static_cast<int64_t>(page) : 0) * c.kv_heads + h) << c.page_log2) + (t & ((1 << c.page_log2) - 1));
    const uint32_t* codes = reinterpret_cast<const uint32_t*>(c.codes + row * kCodeRow);
    const uint32_t* scales = c.scales + row * (2 * R);
    T* dst[2] = {static_cast<T*>(a.k), static_cast<T*>(a.v)};
    const int64_t at = ((static_cast<int64_t>(b) * c.kv_heads + h) * a.rows + t) * 128 + d;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        float x[8];
        const uint32_t s = scales[R * w + d / G];
        codes8(codes[16 * w + (lane & 15)], x);
        const float low = f16_lo(s), delta = f16_hi(s);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = live ? fmaf(x[i], delta, low) : 0.0f;
        store8<T>(dst[w] + at, x);
    }
}

// ---- reserve --------------------------------------------------------------

// Copies `n` words (the page table's unchanged part of an out-of-place call).
__global__ __launch_bounds__(256) void copy_words_kernel(const uint32_t* src, uint32_t* dst, int64_t n) {
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += int64_t{256} * gridDim.x) dst[i] = src[i];
}

// The entries of sequence b that `new_tokens` more tokens need: [lo, hi).
// Entries before the next token's page are never touched (a program may have
// dropped them).
__device__ __forceinline__ void reserve_range(const PageReserve& a, int64_t b, int64_t& lo, int64_t& hi, bool& fits) {
    const int64_t limit = a.width << a.page_log2;
    const int64_t n = clamp_count(a.counts_in[b], limit);
    const int64_t want = a.tokens ? a.tokens[b] : a.each;
    const int64_t more = want < 0 ? 0 : want;
    lo = n >> a.page_log2;
    fits = more <= limit - n;
    hi = fits ? (n + more + (int64_t{1} << a.page_log2) - 1) >> a.page_log2 : lo;
}

// Sequence b by one wave: its row and count to the output, its missing entries
// counted.
__device__ __forceinline__ void reserve_row(const PageReserve& a, int64_t b) {
    const int lane = threadIdx.x & (kWave - 1);
    int64_t lo, hi;
    bool fits;
    reserve_range(a, b, lo, hi, fits);
    const int32_t* row = a.table_in + b * a.width;
    int32_t need = 0;
    for (int64_t i = lo + lane; i < hi; i += kWave) need += row[i] < 0 ? 1 : 0;
    need = static_cast<int32_t>(wave_incl_scan(static_cast<uint32_t>(need), lane));
    if (lane == kWave - 1) {
        a.need[b] = need;
        if (!fits && a.status) atomicOr(a.status, kStatusFull);
    }
    if (a.table != a.table_in) {
        for (int64_t i = lane; i < a.width; i += kWave) a.table[b * a.width + i] = row[i];
        if (lane == 0) a.counts[b] = a.counts_in[b];
    }
}

__global__ __launch_bounds__(256) void reserve_rows_kernel(PageReserve a) {
    const int64_t b = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / kWave;
    if (b < a.batch) reserve_row(a, b);
}

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / kWave;

// The pages [0, n) cut among the plan's waves, a whole number of 64 each.
__device__ __forceinline__ void plan_segment(int64_t n, int wave, int64_t& first, int64_t& last) {
    const int64_t per = ((n + kPlanWaves - 1) / kPlanWaves + kWave - 1) / kWave * kWave;
    first = min(per * wave, n);
    last = min(first + per, n);
}

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

// The lowest `want` pages without a reference, ascending, to list; returns how
// many there are in all.  Every thread of the block calls it.
// COH: this workgroup's own atomics changed them in this launch, so the loads
// read past the cache that may still hold what was there before.
template <bool COH>
__device__ __forceinline__ int32_t list_free(const int32_t* refs, int64_t pages, int32_t want, int32_t* list, int32_t* sh) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    auto is_free = [&](int64_t i, int64_t end) {
        if (i >= end) return false;
        if constexpr (COH) return __hip_atomic_load(refs + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == 0;
        else return refs[i] == 0;
    };
    int64_t first, last;
    plan_segment(pages, wave, first, last);
    int32_t mine = 0;
    for (int64_t i = first; i < last; i += kWave) mine += __popcll(__ballot(is_free(i + lane, last)));
    int32_t total;
    int32_t at = plan_prefix(mine, sh, total);
    for (int64_t i = first; i < last && at < want; i += kWave) {
        const bool free = is_free(i + lane, last);
        const uint64_t mask = __ballot(free);
        const int32_t r = at + __popcll(mask & ((uint64_t{1} << lane) - 1));
        if (free && r < want) list[r] = static_cast<int32_t>(i + lane);
        at += __popcll(mask);
    }
    return total;
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

// Tables and pools up to which one workgroup does the whole plan: a launch
// saved is worth more than the other CUs.  Reserve and fork, out of place, one
// launch against two or three (us):
constexpr int64_t kPlanAlone = 16384;

bool plan_alone(int64_t batch, int64_t width, int64_t pages) {
    return batch * width <= kPlanAlone && pages <= kPlanAlone;
}

// One workgroup: the missing entries of the sequences, in order, take the
// lowest free pages; a sequence whose share does not fit gets none.  ALONE:
// the rows and references are its work too.
template <bool ALONE>
__global__ __launch_bounds__(kPlanThreads) void reserve_plan_kernel(PageReserve a) {
    __shared__ int32_t sh[kPlanWaves];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    if constexpr (ALONE) {
        for (int64_t b = wave; b < a.batch; b += kPlanWaves) reserve_row(a, b);
        if (a.refs != a.refs_in)
            for (int64_t i = threadIdx.x; i < a.pages; i += kPlanThreads) a.refs[i] = a.refs_in[i];
        __syncthreads();
    }
    const int32_t total = scan_needs(a.need, a.batch, sh);
    if (total == 0) return;
    const int32_t want = static_cast<int32_t>(min<int64_t>(total, a.pages));
    const int32_t found = list_free<false>(a.refs, a.pages, want, a.list, sh);
    __syncthreads();  // the list is this workgroup's own: the barrier orders it
    for (int64_t b = wave; b < a.batch; b += kPlanWaves) {
        const int32_t at = a.need[b], end = a.need[b + 1];
        if (end == at) continue;
        if (end > found) {
            if (lane == 0 && a.status) atomicOr(a.status, kStatusNoPage);
            continue;
        }
        int64_t lo, hi;
        bool fits;
        reserve_range(a, b, lo, hi, fits);
        int32_t* row = a.table + b * a.width;
        int32_t r = at;
        for (int64_t i = lo; i < hi; i += kWave) {
            const bool missing = i + lane < hi && row[i + lane] < 0;
            const uint64_t mask = __ballot(missing);
            if (missing) {
                const int32_t page = a.list[r + __popcll(mask & ((uint64_t{1} << lane) - 1))];
                row[i + lane] = page;
                a.refs[page] = 1;
            }
            r += __popcll(mask);
        }
    }
}

// ---- fork -----------------------------------------------------------------

__device__ __forceinline__ int64_t parent_of(const PageFork& a, int64_t b) {
    const int64_t p = a.parents[b];
    return p >= 0 && p < a.batch ? p : -1;
}

// Sequence b by one wave: its new row (in the workspace: another sequence may
// still read the old one) and the reference counts' changes.  The lowest child
// of a parent keeps its whole row; the others share the full pages and get an
// open page of their own (need = 1).
__device__ __forceinline__ void fork_row(const PageFork& a, int64_t b) {
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t p = parent_of(a, b);
    bool earlier = false;
    if (p >= 0)
        for (int64_t i = lane; i < b; i += kWave) earlier = earlier || a.parents[i] == p;
    const bool first = __ballot(earlier) == 0;
    const int64_t count = p >= 0 ? clamp_count(a.counts_in[p], a.width << a.page_log2) : 0;
    const int64_t full = count >> a.page_log2;
    const bool open = (count & ((int64_t{1} << a.page_log2) - 1)) != 0;
    const int32_t* from = a.table_in + (p >= 0 ? p : 0) * a.width;
    const int32_t* old = a.table_in + b * a.width;
    int32_t* to = a.rows + b * a.width;
    const int64_t kept = p < 0 ? 0 : first ? a.width : full;
    for (int64_t i = lane; i < a.width; i += kWave) {
        const int32_t was = old[i];
        const int32_t now = i < kept ? from[i] : -1;
        to[i] = now;
        if (was != now) {
            if (static_cast<uint32_t>(was) < static_cast<uint32_t>(a.pages)) atomicSub(a.refs + was, 1);
            if (static_cast<uint32_t>(now) < static_cast<uint32_t>(a.pages)) atomicAdd(a.refs + now, 1);
        }
    }
    if (lane == 0) {
        const int32_t source = p >= 0 && !first && open ? from[full] : -1;
        const bool need = static_cast<uint32_t>(source) < static_cast<uint32_t>(a.pages);
        a.need[b] = need ? 1 : 0;
        a.source[b] = source;
        a.new_counts[b] = count;
        if (a.status && p < 0 && a.parents[b] != -1) atomicOr(a.status, kStatusBadParent);
    }
}

__global__ __launch_bounds__(256) void fork_rows_kernel(PageFork a) {
    const int64_t b = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / kWave;
    if (b < a.batch) fork_row(a, b);
}

// One workgroup: the open pages wanted take the lowest free pages; a sequence
// that finds none is left empty.  ALONE: the rows and references are its work
// too.
template <bool ALONE>
__global__ __launch_bounds__(kPlanThreads) void fork_plan_kernel(PageFork a) {
    __shared__ int32_t sh[kPlanWaves];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    if constexpr (ALONE) {
        if (a.refs != a.refs_in) {
            for (int64_t i = threadIdx.x; i < a.pages; i += kPlanThreads) a.refs[i] = a.refs_in[i];
            __syncthreads();
        }
        for (int64_t b = wave; b < a.batch; b += kPlanWaves) fork_row(a, b);
        __syncthreads();
    }
    const int32_t total = scan_needs(a.need, a.batch, sh);
    if (threadIdx.x == 0) *a.moves = total;
    if (total == 0) return;
    const int32_t found = list_free<ALONE>(a.refs, a.pages, static_cast<int32_t>(min<int64_t>(total, a.pages)), a.list, sh);
    if (threadIdx.x == 0 && found < total) *a.moves = found;
    __syncthreads();
    for (int64_t b = wave; b < a.batch; b += kPlanWaves) {
        const int32_t at = a.need[b];
        if (a.need[b + 1] == at) continue;
        int32_t* row = a.rows + b * a.width;
        const int64_t full = a.new_counts[b] >> a.page_log2;
        if (at < found) {
            if (lane == 0) {
                const int32_t page = a.list[at];
                row[full] = page;
                a.refs[page] = 1;
                a.pairs[at] = make_int2(a.source[b], page);
            }
        } else {
            for (int64_t i = lane; i < a.width; i += kWave) {
                if (static_cast<uint32_t>(row[i]) < static_cast<uint32_t>(a.pages)) atomicSub(a.refs + row[i], 1);
                row[i] = -1;
            }
            if (lane == 0) {
                a.new_counts[b] = 0;
                if (a.status) atomicOr(a.status, kStatusNoPage);
            }
        }
    }
}

// ---- compact --------------------------------------------------------------

// One workgroup: n = the live pages; the live pages from n on, ascending, move
// to the free ones before n, ascending (as many).
__global__ __launch_bounds__(kPlanThreads) void compact_plan_kernel(PageCompact a) {
    __shared__ int32_t sh[kPlanWaves];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    int64_t first, last;
    plan_segment(a.pages, wave, first, last);
    int32_t live = 0;
    for (int64_t i = first; i < last; i += kWave)
        live += __popcll(__ballot(i + lane < last && a.refs_in[i + lane] > 0));
    int32_t n;
    plan_prefix(live, sh, n);
    int32_t holes = 0, movers = 0;
    for (int64_t i = first; i < last; i += kWave) {
        const bool in = i + lane < last, used = in && a.refs_in[i + lane] > 0;
        holes += __popcll(__ballot(in && !used && i + lane < n));
        movers += __popcll(__ballot(used && i + lane >= n));
    }
    int32_t moves, same;
    int32_t hole_at = plan_prefix(holes, sh, moves), mover_at = plan_prefix(movers, sh, same);
    int32_t* pair = reinterpret_cast<int32_t*>(a.pairs);  // (source, target) of move j at 2j, 2j + 1
    for (int64_t i = first; i < last; i += kWave) {
        const bool in = i + lane < last;
        const int32_t refs = in ? a.refs_in[i + lane] : 0;
        const bool hole = in && refs <= 0 && i + lane < n, mover = refs > 0 && i + lane >= n;
        const uint64_t hm = __ballot(hole), mm = __ballot(mover), below = (uint64_t{1} << lane) - 1;
        if (hole) pair[2 * (hole_at + __popcll(hm & below)) + 1] = static_cast<int32_t>(i + lane);
        if (mover) pair[2 * (mover_at + __popcll(mm & below))] = static_cast<int32_t>(i + lane);
        if (in) {
            a.map[i + lane] = refs > 0 ? static_cast<int32_t>(i + lane) : -1;
            if (a.refs != a.refs_in) a.refs[i + lane] = refs;
        }
        hole_at += __popcll(hm);
        mover_at += __popcll(mm);
    }
    if (threadIdx.x == 0) *a.moves = moves;
    __syncthreads();
    for (int32_t j = threadIdx.x; j < moves; j += kPlanThreads) {
        const int32_t source = pair[2 * j], target = pair[2 * j + 1];
        a.map[source] = target;
        a.refs[target] = a.refs[source];
        a.refs[source] = 0;
    }
}

// ---- the pages of a plan, and its table -----------------------------------

// Copies the plan's pages in every layer, and lays the new table down in the
// first workgroups.  Sources are live pages and targets pages nothing else
// holds, so no workgroup reads what another writes.
__global__ __launch_bounds__(256) void move_pages_kernel(PageMoves m) {
    const int64_t step = int64_t{256} * gridDim.x, me = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    for (int64_t i = me; i < m.entries; i += step) {
        int32_t e = m.table_in[i];
        if (m.map && static_cast<uint32_t>(e) < static_cast<uint32_t>(m.pages)) e = m.map[e];
        m.table[i] = e;
    }
    if (m.counts)
        for (int64_t i = me; i < m.batch; i += step) m.counts[i] = m.counts_in[i];
    const int64_t units = static_cast<int64_t>(*m.moves) * m.layers * m.parts;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int64_t part = u % m.parts, rest = u / m.parts;
        const int64_t layer = rest % m.layers;
        const int2 pair = m.pairs[rest / m.layers];
        const bool codes = part < m.code_parts;
        const int64_t bytes = codes ? m.code_bytes : m.scale_bytes;
        const int64_t off = (codes ? part : part - m.code_parts) * kMoveBytes;
        char* pool = codes ? m.codes : m.scales;
        const int64_t base = layer * m.pages * bytes + off;
        const uint4* src = reinterpret_cast<const uint4*>(pool + base + pair.x * bytes);
        uint4* dst = reinterpret_cast<uint4*>(pool + base + pair.y * bytes);
        const int64_t n = min<int64_t>(kMoveBytes, bytes - off) / 16;
        for (int64_t i = threadIdx.x; i < n; i += 256) dst[i] = src[i];
    }
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

}  // namespace

#define POPKV_PAGED_G(KERNEL, T)                                                                  \
    switch (dim_group) {                                                                          \
        case 16: hipLaunchKernelGGL((KERNEL<T, 16>), grid, dim3(256), 0, stream, a, c); break;    \
        case 32: hipLaunchKernelGGL((KERNEL<T, 32>), grid, dim3(256), 0, stream, a, c); break;    \
        default: hipLaunchKernelGGL((KERNEL<T, 64>), grid, dim3(256), 0, stream, a, c); break;    \
    }
#define POPKV_PAGED_T(KERNEL)                                                \
    switch (dtype) {                                                         \
        case POPKV_DTYPE_F32: POPKV_PAGED_G(KERNEL, float) break;            \
        case POPKV_DTYPE_F16: POPKV_PAGED_G(KERNEL, f16_t) break;            \
        default: POPKV_PAGED_G(KERNEL, bf16_t) break;                        \
    }

hipError_t launch_paged_write(const PagedWrite& a, const PagedView& c, int dtype, int dim_group, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>((a.rows + 15) / 16), static_cast<unsigned>(c.kv_heads),
                    static_cast<unsigned>(c.batch));
    POPKV_PAGED_T(paged_write_kernel)
    return hipGetLastError();
}

hipError_t launch_paged_read(const PagedRead& a, const PagedView& c, int dtype, int dim_group, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>((a.rows + 15) / 16), static_cast<unsigned>(c.kv_heads),
                    static_cast<unsigned>(c.batch));
    POPKV_PAGED_T(paged_read_kernel)
    return hipGetLastError();
}
#undef POPKV_PAGED_T
#undef POPKV_PAGED_G

hipError_t launch_page_reserve(const PageReserve& a, hipStream_t s) {
    if (plan_alone(a.batch, a.width, a.pages)) {
        hipLaunchKernelGGL(reserve_plan_kernel<true>, dim3(1), dim3(kPlanThreads), 0, s, a);
        return hipGetLastError();
    }
    if (a.refs != a.refs_in) {
        const hipError_t e = copy_words(a.refs_in, a.refs, a.pages, s);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(reserve_rows_kernel, dim3(static_cast<unsigned>((a.batch + 3) / 4)), dim3(256), 0, s, a);
    hipLaunchKernelGGL(reserve_plan_kernel<false>, dim3(1), dim3(kPlanThreads), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_page_fork(const PageFork& a, const PageMoves& m, hipStream_t s) {
    if (plan_alone(a.batch, a.width, a.pages)) {
        hipLaunchKernelGGL(fork_plan_kernel<true>, dim3(1), dim3(kPlanThreads), 0, s, a);
    } else {
        if (a.refs != a.refs_in) {
            const hipError_t e = copy_words(a.refs_in, a.refs, a.pages, s);
            if (e != hipSuccess) return e;
        }
        hipLaunchKernelGGL(fork_rows_kernel, dim3(static_cast<unsigned>((a.batch + 3) / 4)), dim3(256), 0, s, a);
        hipLaunchKernelGGL(fork_plan_kernel<false>, dim3(1), dim3(kPlanThreads), 0, s, a);
    }
    hipLaunchKernelGGL(move_pages_kernel, dim3(blocks_for(a.batch * m.layers * m.parts, 1, 2048)), dim3(256), 0, s, m);
    return hipGetLastError();
}

hipError_t launch_page_compact(const PageCompact& a, const PageMoves& m, hipStream_t s) {
    hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a);
    hipLaunchKernelGGL(move_pages_kernel, dim3(blocks_for(a.pages / 2 * m.layers * m.parts, 1, 2048)), dim3(256), 0, s, m);
    return hipGetLastError();
}

}  // namespace popkv
