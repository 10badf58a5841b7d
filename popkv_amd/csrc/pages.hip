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

// Eight neighbouring elements as loaded, and what the encode asks of them.
template <typename T>
struct Eight {
    Raw8<T> raw;
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (sizeof(T) == 4) {
            raw.a = __builtin_bit_cast(float4, load_once(p));
            raw.b = __builtin_bit_cast(float4, load_once(p + 4));
        } else {
            raw.u = __builtin_bit_cast(uint4, load_once(p));
        }
    }
    // the largest magnitude's bits: at least kNotFinite for infinity and NaN
    static constexpr uint32_t kNotFinite = Elem<T>::kDtype == POPKV_DTYPE_F32 ? 0x7f800000u
                                           : Elem<T>::kDtype == POPKV_DTYPE_BF16 ? 0x7f80u : 0x7c00u;
    __device__ __forceinline__ uint32_t top() const {
        if constexpr (sizeof(T) == 4) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(raw.get(i)) & 0x7fffffffu);
            return m;
        } else {
            typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
            const uint32_t w[4] = {raw.u.x, raw.u.y, raw.u.z, raw.u.w};
            u16x2 m = __builtin_bit_cast(u16x2, w[0] & 0x7fff7fffu);
#pragma unroll
            for (int i = 1; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
            return max(m[0], m[1]);
        }
    }
};

// low = fp16(min), delta = fp16((max - low) / 15), code = round((x - low) /
// delta) in 0 .. 15, ties to even, of this lane's eight values; the LPG lanes
// of a group hold its G = 8 * LPG values.  A group with a NaN or an infinity
// gets low = NaN: it reads back as NaN.
template <typename T, int LPG>
__device__ __forceinline__ void quantise8(const Eight<T>& in, uint32_t& code, uint32_t& scale) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = in.raw.get(i);
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
    }
    uint32_t top = in.top();
    auto fold = [&](auto ctrl) {
        constexpr int C = decltype(ctrl)::value;
        lo = fminf(lo, dpp_mov<C>(lo));
        hi = fmaxf(hi, dpp_mov<C>(hi));
        top = max(top, __float_as_uint(dpp_mov<C>(__uint_as_float(top))));
    };
    fold(std::integral_constant<int, 0xB1>{});
    if constexpr (LPG >= 4) fold(std::integral_constant<int, 0x4E>{});
    if constexpr (LPG >= 8) fold(std::integral_constant<int, 0x141>{});
    lo = fminf(fmaxf(lo, -kScaleLimit), kScaleLimit);
    hi = fminf(fmaxf(hi, -kScaleLimit), kScaleLimit);
    const uint32_t lob = f16_rne(lo);
    const float low = bits_f16(lob);
    // (max - low) / 15 in fp64, as max - low need not fit fp32: the product with
    // 1 / 15 and one correction by its exact remainder is the division's result
    // (Markstein), in three instructions
    const double t = static_cast<double>(hi) - static_cast<double>(low), fifteenth = 1.0 / 15.0;
    double d15 = t * fifteenth;
    d15 = fma(fma(-15.0, d15, t), fifteenth, d15);
    const uint32_t deb = f16_rne(static_cast<float>(d15));
    const float delta = bits_f16(deb);
    const bool bad = top >= Eight<T>::kNotFinite, flat = bad || delta == 0.0f;
    scale = bad ? 0x7e00u : lob | (deb << 16);
    // fp32 quotients are off by less than 2^-18 (a reciprocal within 2^-23 and two
    // roundings of 2^-24, of a quotient below 16); a value that near a border
    // between two codes is decided in fp64.  Adding 2^23 rounds to an integer.
    const float inv = flat ? 0.0f : __builtin_amdgcn_rcpf(delta);
    constexpr float kMagic = 8388608.0f;
    float r[8], off = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float q = fminf(fmaxf((x[i] - low) * inv, 0.0f), 15.0f);
        r[i] = (q + kMagic) - kMagic;
        off = fmaxf(off, fabsf(q - r[i]));
    }
    if (__ballot(off > 0.5f - 0x1p-16f) != 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float q = fminf(fmaxf((x[i] - low) * inv, 0.0f), 15.0f);
            if (fabsf(q - r[i]) > 0.5f - 0x1p-16f && !flat) {
                const double e = (static_cast<double>(x[i]) - static_cast<double>(low)) / static_cast<double>(delta);
                r[i] = static_cast<float>(rint(fmin(fmax(e, 0.0), 15.0)));
            }
        }
    }
    // four codes at a time as one number of 16 bits
    const float even = fmaf(fmaf(fmaf(r[3], 16.0f, r[2]), 16.0f, r[1]), 16.0f, r[0]);
    const float odd = fmaf(fmaf(fmaf(r[7], 16.0f, r[6]), 16.0f, r[5]), 16.0f, r[4]);
    code = bad ? 0u : static_cast<uint32_t>(even) | (static_cast<uint32_t>(odd) << 16);
}

// Sixteen lanes a row, eight dims of its K and of its V each: the K and the V
// row of a token make one 128-byte line of codes.  Bound by the stream of the
// rows, 2 * 128 * sizeof(T) bytes read, which pass the caches by, and 128 + 8R
// written per token and head: 32768 tokens of 8 heads bf16, 64-dim groups, 172 MB
// in 35 us (4.9 TB/s), fp32 with 32-dim groups 310 MB in 61 (5.1); two rows a lane
// 35 and 61, at 8192 tokens 13.2 and 16.8 against 12.0 and 16.3.
template <typename T, int G>
__global__ __launch_bounds__(256) void paged_write_kernel(PagedWrite a, PagedView c) {
    constexpr int R = 128 / G;
    const int lane16 = threadIdx.x & 15;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 16 + threadIdx.x / 16;
    const int h = blockIdx.y, b = blockIdx.z;
    const int64_t most = a.tokens ? clamp_count(a.tokens[b], a.rows) : a.rows;
    if (static_cast<int64_t>(blockIdx.x) * 16 >= most) return;
    const int64_t limit = c.width << c.page_log2;
    const int64_t pos = clamp_count(c.counts[b], limit) + t;
    const int d = lane16 * 8;
    const int64_t from = min(t, most - 1);  // (rows past the last repeat it)
    Eight<T> k, v;
    k.load(static_cast<const T*>(a.k) + b * a.k_bs + h * a.k_hs + from * a.k_ts + d);
    v.load(static_cast<const T*>(a.v) + b * a.v_bs + h * a.v_hs + from * a.v_ts + d);
    const int32_t page = pos < limit ? c.table[b * c.width + (pos >> c.page_log2)] : -1;
    uint32_t code[2], scale[2];
    quantise8<T, G / 8>(k, code[0], scale[0]);
    quantise8<T, G / 8>(v, code[1], scale[1]);
    if (t >= most) return;
    if (static_cast<uint32_t>(page) < static_cast<uint32_t>(c.pages)) {
        const int64_t row =
            ((static_cast<int64_t>(page) * c.kv_heads + h) << c.page_log2) + (pos & ((1 << c.page_log2) - 1));
        uint32_t* codes = reinterpret_cast<uint32_t*>(c.codes + row * kCodeRow);
        uint32_t* scales = c.scales + row * (2 * R);
        codes[lane16] = code[0];
        codes[16 + lane16] = code[1];
        if (d % G == 0) {
            scales[d / G] = scale[0];
            scales[R + d / G] = scale[1];
        }
    } else if (a.status && lane16 == 0 && h == 0) {
        atomicOr(a.status, pos < limit ? kStatusNoPage : kStatusFull);
    }
}

// ---- read -----------------------------------------------------------------

// The inverse: rows [0, count) of every sequence as K/V rows of T; rows past a
// count are cleared when `fill`, else left as they are.  Sixteen lanes a row,
// each two pieces of 16 bytes: of 16-bit rows its eight dims of K and of V, of
// fp32 rows four dims in either half, so that a store instruction fills whole
// lines (32 bytes a lane instead left half of each line for the next one).
// Bound by the rows written, which pass the caches by: a prompt of 32767 tokens
// of 8 heads bf16, 64-dim groups, written and read back in turn with others,
// 71.3 us against 80.5 with plain loads and stores; fp32 rows of 268 MB 45.6
// against 73.1 (5.9 TB/s; 32 bytes a lane past the caches are slower than either).
template <typename T, int G>
__global__ __launch_bounds__(256) void paged_read_kernel(PagedRead a, PagedView c) {
    constexpr int R = 128 / G, DIMS = 16 / sizeof(T), PIECES = sizeof(T) / 2;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 16 + threadIdx.x / 16;
    const int h = blockIdx.y, b = blockIdx.z;
    if (t >= a.rows) return;
    const int64_t count = clamp_count(c.counts[b], c.width << c.page_log2);
    const int32_t page = t < count ? c.table[b * c.width + (t >> c.page_log2)] : -1;
    const bool live = static_cast<uint32_t>(page) < static_cast<uint32_t>(c.pages);
    if (!live && !a.fill && t >= count) return;
    const int64_t row =
        (((live ? static_cast<int64_t>(page) : 0) * c.kv_heads + h) << c.page_log2) + (t & ((1 << c.page_log2) - 1));
    const char* codes = c.codes + row * kCodeRow;
    const uint32_t* scales = c.scales + row * (2 * R);
    T* dst[2] = {static_cast<T*>(a.k), static_cast<T*>(a.v)};
    const int64_t at = ((static_cast<int64_t>(b) * c.kv_heads + h) * a.rows + t) * 128;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
#pragma unroll
        for (int piece = 0; piece < PIECES; ++piece) {
            const int d = 128 / PIECES * piece + DIMS * (threadIdx.x & 15);
            float x[DIMS];
            const uint32_t s = scales[R * w + d / G];
            const float low = f16_lo(s), delta = f16_hi(s);
            if constexpr (sizeof(T) == 4) {
                const uint32_t code = *reinterpret_cast<const uint16_t*>(codes + 64 * w + d / 2);
#pragma unroll
                for (int i = 0; i < DIMS; ++i) x[i] = static_cast<float>(code >> (4 * i) & 15u);
            } else {
                codes8(*reinterpret_cast<const uint32_t*>(codes + 64 * w + d / 2), x);
            }
#pragma unroll
            for (int i = 0; i < DIMS; ++i) x[i] = live ? fmaf(x[i], delta, low) : 0.0f;
            u32x4 out;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(T) == 4) out[i] = __float_as_uint(x[i]);
                else out[i] = pack2<T>(x[2 * i], x[2 * i + 1]);
            }
            store_once(dst[w] + at + d, out);
        }
    }
}

// ---- reserve --------------------------------------------------------------

// Copies `n` words (the page table's unchanged part of an out-of-place call).
__global__ __launch_bounds__(256) void copy_words_kernel(const uint32_t* src, uint32_t* dst, int64_t n) {
    const int64_t step = int64_t{256} * gridDim.x;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += step) dst[i] = src[i];
}

// The entries of sequence b that `new_tokens` more tokens need: [lo, hi).
// Entries before the next token's page are never touched (a program may have
// dropped them); of the others, one outside the pool is no page and is missing.
__device__ __forceinline__ bool is_missing(const PageReserve& a, int32_t page) {
    return static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.pages);
}
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
    for (int64_t i = lo + lane; i < hi; i += kWave) need += is_missing(a, row[i]) ? 1 : 0;
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

// One workgroup: the missing entries of the sequences, in order, take the
// lowest free pages; a sequence whose share does not fit gets none.
__global__ __launch_bounds__(kPlanThreads) void reserve_plan_kernel(PageReserve a) {
    __shared__ PageMap map;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int32_t total = scan_needs(a.need, a.batch, map.sh);
    if (total == 0) return;
    const int32_t want = static_cast<int32_t>(min<int64_t>(total, a.pages));
    const int32_t found = list_free(map, a.pages, want, a.list, [&](int64_t i) { return a.refs[i] != 0; });
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
            const bool missing = i + lane < hi && is_missing(a, row[i + lane]);
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

// i / width of an entry of such a table, inverse = 1 / width: (i + 1/2) / width
// lies at least 1 / (2 width) from an integer, and its fp32 rounding is off by
// less, i being below 2^14.
__device__ __forceinline__ int row_of(int i, float inverse) {
    return static_cast<int>((static_cast<float>(i) + 0.5f) * inverse);
}

// The r-th free page (r below how many there are) of a mapped pool.
__device__ __forceinline__ int nth_free(const PageMap& m, int pages, int r) {
    int lo = 0, hi = (pages + 63) / 64 - 1;  // the last word with at most r free pages before it
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (mid * 64 - m.before[mid] <= r) lo = mid;
        else hi = mid - 1;
    }
    uint64_t free = ~m.words[lo];
    int left = r - (lo * 64 - m.before[lo]), at = 0;
#pragma unroll
    for (int half = 32; half; half /= 2) {
        const int n = __popcll(free & ((uint64_t{1} << half) - 1));
        if (left >= n) {
            left -= n;
            at += half;
            free >>= half;
        }
    }
    return lo * 64 + at;
}

__global__ __launch_bounds__(kPlanThreads) void reserve_alone_kernel(PageReserve a) {
    __shared__ PageMap map;
    __shared__ uint64_t s_missing[kPlanAlone / 64];
    __shared__ int32_t s_before[kPlanAlone / 64], s_lo[kPlanThreads], s_hi[kPlanThreads], s_need[kPlanThreads];
    const int tid = threadIdx.x, lane = tid & (kWave - 1);
    const int batch = static_cast<int>(a.batch), width = static_cast<int>(a.width), pages = static_cast<int>(a.pages);
    const int entries = batch * width, words = (entries + 63) / 64;
    const float inverse = 1.0f / static_cast<float>(width);
    s_need[tid] = 0;
    if (tid < batch) {
        int64_t lo, hi;
        bool fits;
        reserve_range(a, tid, lo, hi, fits);
        s_lo[tid] = static_cast<int32_t>(lo);
        s_hi[tid] = static_cast<int32_t>(hi);
        if (!fits && a.status) atomicOr(a.status, kStatusFull);
        if (a.counts != a.counts_in) a.counts[tid] = a.counts_in[tid];
    }
    const int32_t used = map_pages(map, 0, pages, [&](int64_t i) { return a.refs_in[i] != 0; });
    if (a.refs != a.refs_in) plan_copy(a.refs_in, a.refs, pages);
    constexpr int AHEAD = 4;
    for (int i0 = 0; i0 < entries; i0 += AHEAD * kPlanThreads) {
        int32_t page[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int i = i0 + j * kPlanThreads + tid;
            page[j] = i < entries ? a.table_in[i] : 0;
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int i = i0 + j * kPlanThreads + tid;
            bool missing = false;
            if (i < entries) {
                const int b = row_of(i, inverse), e = i - b * width;
                if (a.table != a.table_in) a.table[i] = page[j];
                missing = is_missing(a, page[j]) && e >= s_lo[b] && e < s_hi[b];
                if (missing) atomicAdd(s_need + b, 1);
            }
            const uint64_t bits = __ballot(missing);
            if (lane == 0 && i / 64 < words) s_missing[i / 64] = bits;
        }
    }
    __syncthreads();
    // ranks: of the missing entries before each word, and of each sequence's last
    auto scan = [&](int32_t v, int32_t& total) {
        const int32_t incl = static_cast<int32_t>(wave_incl_scan(static_cast<uint32_t>(v), lane));
        return plan_prefix(__builtin_amdgcn_readlane(incl, kWave - 1), map.sh, total) + incl;
    };
    int32_t total;
    const int32_t n = tid < words ? __popcll(s_missing[tid]) : 0, incl = scan(n, total);
    if (tid < words) s_before[tid] = incl - n;
    if (total == 0) return;
    const int32_t need = s_need[tid], end = scan(need, total), found = pages - used;
    if (need > 0 && end > found && a.status) atomicOr(a.status, kStatusNoPage);
    s_need[tid] = end;
    __syncthreads();
    for (int i = tid; i < entries; i += kPlanThreads) {
        const uint64_t bits = s_missing[i / 64];
        if (!(bits >> (i & 63) & 1) || s_need[row_of(i, inverse)] > found) continue;
        const int page = nth_free(map, pages, s_before[i / 64] + __popcll(bits & ((uint64_t{1} << (i & 63)) - 1)));
        a.table[i] = page;
        a.refs[page] = 1;
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

// A child for whose open page none is free: empty, its shared pages given back.
__device__ __forceinline__ void fork_drop(const PageFork& a, int64_t b, int32_t* refs) {
    int32_t* row = a.rows + b * a.width;
    for (int64_t i = threadIdx.x & (kWave - 1); i < a.width; i += kWave) {
        if (static_cast<uint32_t>(row[i]) < static_cast<uint32_t>(a.pages)) atomicSub(refs + row[i], 1);
        row[i] = -1;
    }
    if ((threadIdx.x & (kWave - 1)) == 0) {
        a.new_counts[b] = 0;
        if (a.status) atomicOr(a.status, kStatusNoPage);
    }
}

// One workgroup: the open pages wanted take the lowest free pages; a sequence
// that finds none is left empty.
__global__ __launch_bounds__(kPlanThreads) void fork_plan_kernel(PageFork a) {
    __shared__ PageMap map;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int32_t total = scan_needs(a.need, a.batch, map.sh);
    if (total == 0) {
        if (threadIdx.x == 0) *a.moves = 0;
        return;
    }
    const int32_t found = list_free(map, a.pages, static_cast<int32_t>(min<int64_t>(total, a.pages)), a.list,
                                    [&](int64_t i) { return a.refs[i] != 0; });
    if (threadIdx.x == 0) *a.moves = min(found, total);
    __syncthreads();
    for (int64_t b = wave; b < a.batch; b += kPlanWaves) {
        const int32_t at = a.need[b];
        if (a.need[b + 1] == at) continue;
        if (at >= found) {
            fork_drop(a, b, a.refs);
        } else if (lane == 0) {
            const int32_t page = a.list[at];
            a.rows[b * a.width + (a.new_counts[b] >> a.page_log2)] = page;
            a.refs[page] = 1;
            a.pairs[at] = make_int2(a.source[b], page);
        }
    }
}

// The whole plan of a small table by one workgroup, a thread a sequence and a
// thread a table entry, the reference counts in LDS.
constexpr int kForkPages = 8192;
__global__ __launch_bounds__(kPlanThreads) void fork_alone_kernel(PageFork a) {
    __shared__ PageMap map;
    __shared__ int32_t s_refs[kForkPages], s_first[kPlanThreads], s_parent[kPlanThreads], s_kept[kPlanThreads];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const int batch = static_cast<int>(a.batch), width = static_cast<int>(a.width), pages = static_cast<int>(a.pages);
    const float inverse = 1.0f / static_cast<float>(width);
    const int p = tid < batch ? static_cast<int>(parent_of(a, tid)) : -1;
    const int count = p >= 0 ? static_cast<int>(clamp_count(a.counts_in[p], a.width << a.page_log2)) : 0;
    s_first[tid] = kPlanThreads;
    plan_copy(a.refs_in, s_refs, pages);
    __syncthreads();
    if (p >= 0) atomicMin(s_first + p, tid);
    __syncthreads();
    const bool first = p >= 0 && s_first[p] == tid;
    const int full = count >> a.page_log2;
    s_parent[tid] = p;
    s_kept[tid] = p < 0 ? 0 : first ? width : full;
    const bool open = p >= 0 && !first && (count & ((1 << a.page_log2) - 1)) != 0;
    const int32_t source = open ? a.table_in[p * width + full] : -1;
    const int need = static_cast<uint32_t>(source) < static_cast<uint32_t>(pages) ? 1 : 0;
    if (tid < batch) {
        a.new_counts[tid] = count;
        if (a.status && p < 0 && a.parents[tid] != -1) atomicOr(a.status, kStatusBadParent);
    }
    __syncthreads();
    constexpr int AHEAD = 4;
    for (int i0 = 0; i0 < batch * width; i0 += AHEAD * kPlanThreads) {
        int32_t was[AHEAD], now[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int i = i0 + j * kPlanThreads + tid;
            was[j] = now[j] = -1;
            if (i < batch * width) {
                const int b = row_of(i, inverse), e = i - b * width;
                was[j] = a.table_in[i];
                if (e < s_kept[b]) now[j] = a.table_in[s_parent[b] * width + e];
            }
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int i = i0 + j * kPlanThreads + tid;
            if (i < batch * width) a.rows[i] = now[j];
            if (was[j] != now[j]) {
                if (static_cast<uint32_t>(was[j]) < static_cast<uint32_t>(pages)) atomicSub(s_refs + was[j], 1);
                if (static_cast<uint32_t>(now[j]) < static_cast<uint32_t>(pages)) atomicAdd(s_refs + now[j], 1);
            }
        }
    }
    const int32_t incl = static_cast<int32_t>(wave_incl_scan(static_cast<uint32_t>(need), lane));
    int32_t total;
    const int32_t at = plan_prefix(__builtin_amdgcn_readlane(incl, kWave - 1), map.sh, total) + incl - need;
    int32_t found = 0;
    if (total > 0) {
        found = list_free(map, pages, min(total, pages), a.list, [&](int64_t i) { return s_refs[i] != 0; });
        __syncthreads();
        if (need && at < found) {
            const int32_t page = a.list[at];
            a.rows[tid * width + full] = page;
            s_refs[page] = 1;
            a.pairs[at] = make_int2(source, page);
        }
        s_first[tid] = need && at >= found ? 1 : 0;  // (read as the parents' no more)
        __syncthreads();
        if (found < total)
            for (int b = wave; b < batch; b += kPlanWaves)
                if (s_first[b] != 0) fork_drop(a, b, s_refs);
        __syncthreads();
    }
    if (tid == 0) *a.moves = min(found, total);
    plan_copy(s_refs, a.refs, pages);
}

// ---- compact --------------------------------------------------------------

// One workgroup: n = the live pages; the live pages from n on, ascending, move
// to the free ones before n, ascending (as many).  A live page from n on is the
// (live pages before it - live pages before n)-th mover, a free page before n the
// (its number - live pages before it)-th hole.
__global__ __launch_bounds__(kPlanThreads) void compact_plan_kernel(PageCompact a) {
    __shared__ PageMap map;
    auto used = [&](int64_t i) { return a.refs_in[i] > 0; };
    int64_t n = 0;
    int32_t whole = 0;
    for (int64_t first = 0; first < a.pages; first += kMapPages) n += whole = map_pages(map, first, a.pages, used);
    // the live pages before n: those of the parts before n's, and what the map
    // of its part says
    int64_t below = 0;
    if (a.pages <= kMapPages) {
        below = n < a.pages ? used_before(map, static_cast<int>(n)) : n;
    } else {
        for (int64_t first = 0; first < n; first += kMapPages) {
            const int32_t part = map_pages(map, first, a.pages, used);
            below += n - first < kMapPages ? used_before(map, static_cast<int>(n - first)) : part;
        }
    }
    int32_t* pair = reinterpret_cast<int32_t*>(a.pairs);  // (source, target) of move j at 2j, 2j + 1
    int64_t before = 0;
    for (int64_t first = 0; first < a.pages; first += kMapPages) {
        const int32_t part = a.pages <= kMapPages ? whole : map_pages(map, first, a.pages, used);
        const int size = static_cast<int>(min<int64_t>(kMapPages, a.pages - first));
        constexpr int AHEAD = 8;
        for (int i0 = threadIdx.x; i0 < size; i0 += AHEAD * kPlanThreads) {
            int32_t refs[AHEAD];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
                refs[j] = i0 + j * kPlanThreads < size ? a.refs_in[first + i0 + j * kPlanThreads] : 0;
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const int i = i0 + j * kPlanThreads;
                if (i >= size) break;
                const bool live = refs[j] > 0;
                const int64_t page = first + i, rank = before + used_before(map, i);
                if (!live && page < n) pair[2 * (page - rank) + 1] = static_cast<int32_t>(page);
                if (live && page >= n) pair[2 * (rank - below)] = static_cast<int32_t>(page);
                a.map[page] = live ? static_cast<int32_t>(page) : -1;
                if (a.refs != a.refs_in) a.refs[page] = refs[j];
            }
        }
        before += part;
    }
    const int32_t moves = static_cast<int32_t>(n - below);
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

// Copies the plan's pages in every layer, 16 KB a workgroup at a time, and lays
// the new table down in the first workgroups.  Sources are live pages and
// targets pages nothing else holds, so no workgroup reads what another writes.
// Bound by the copy: half of 640 pages of 16 layers, 206 MB read and written, 84
// us with the plan (91 through the caches, a load at a time); units of 4 or 64 KB
// cost a fork of 28 pages 3 and 2 us.  ONCE: pages pass the caches by, as a
// compaction's do; a fork's few stay there (34 MB 8 us, 14 past the caches).
template <bool ONCE>
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
        const u32x4* src = reinterpret_cast<const u32x4*>(pool + base + pair.x * bytes) + threadIdx.x;
        u32x4* dst = reinterpret_cast<u32x4*>(pool + base + pair.y * bytes) + threadIdx.x;
        const int n = static_cast<int>(min<int64_t>(kMoveBytes, bytes - off) / 16) - threadIdx.x;
        constexpr int LOADS = kMoveBytes / (256 * 16);  // a thread's, all on their way before the first store
        u32x4 x[LOADS];
#pragma unroll
        for (int j = 0; j < LOADS; ++j)
            if (256 * j < n) x[j] = ONCE ? load_once(src + 256 * j) : src[256 * j];
#pragma unroll
        for (int j = 0; j < LOADS; ++j)
            if (256 * j < n) {
                if constexpr (ONCE) store_once(dst + 256 * j, x[j]);
                else dst[256 * j] = x[j];
            }
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
        hipLaunchKernelGGL(reserve_alone_kernel, dim3(1), dim3(kPlanThreads), 0, s, a);
        return hipGetLastError();
    }
    if (a.refs != a.refs_in) {
        const hipError_t e = copy_words(a.refs_in, a.refs, a.pages, s);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(reserve_rows_kernel, dim3(static_cast<unsigned>((a.batch + 3) / 4)), dim3(256), 0, s, a);
    hipLaunchKernelGGL(reserve_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_page_fork(const PageFork& a, const PageMoves& m, hipStream_t s) {
    if (plan_alone(a.batch, a.width, a.pages) && a.pages <= kForkPages) {
        hipLaunchKernelGGL(fork_alone_kernel, dim3(1), dim3(kPlanThreads), 0, s, a);
    } else {
        if (a.refs != a.refs_in) {
            const hipError_t e = copy_words(a.refs_in, a.refs, a.pages, s);
            if (e != hipSuccess) return e;
        }
        hipLaunchKernelGGL(fork_rows_kernel, dim3(static_cast<unsigned>((a.batch + 3) / 4)), dim3(256), 0, s, a);
        hipLaunchKernelGGL(fork_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a);
    }
    const unsigned grid = blocks_for(a.batch * m.layers * m.parts, 1, 2048);
    hipLaunchKernelGGL(move_pages_kernel<false>, dim3(grid), dim3(256), 0, s, m);
    return hipGetLastError();
}

hipError_t launch_page_compact(const PageCompact& a, const PageMoves& m, hipStream_t s) {
    hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a);
    const unsigned grid = blocks_for(a.pages / 2 * m.layers * m.parts, 1, 2048);
    hipLaunchKernelGGL(move_pages_kernel<true>, dim3(grid), dim3(256), 0, s, m);
    return hipGetLastError();
}

}  // namespace popkv
