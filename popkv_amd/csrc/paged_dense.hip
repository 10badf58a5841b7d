// Dense decode attention over the paged 4-bit K/V cache: every cached token and
// the current one.
#include "paged_attention.h"

namespace popkv {
namespace {

// Adds `n` states, `stride` floats apart, to a wave's running (m, l, a); a lane
// owns dims 2 lane and 2 lane + 1.
__device__ __forceinline__ void fold_states(const float* ps, int64_t stride, int n, float& m, float& l, float2& a) {
    constexpr int NF = 32;
    const int lane = threadIdx.x & (kWave - 1);
    for (int s0 = 0; s0 < n; s0 += NF) {
        float2 state = make_float2(-INFINITY, 0.0f), x[NF];
        const int k = min(NF, n - s0);
        if (lane < k) state = ld_pair(ps + (s0 + lane) * stride);
#pragma unroll
        for (int j0 = 0; j0 < NF; j0 += 8) {
            if (j0 >= k) break;
#pragma unroll
            for (int j = j0; j < j0 + 8; ++j) x[j] = ld_pair(ps + (s0 + min(j, k - 1)) * stride + 2 + 2 * lane);
        }
        const float mx = fmaxf(m, wave_max(state.x));
        const float w = state_weight(state.x, state.y, mx);
        const float f = state_weight(m, l, mx);
        l = fmaf(l, f, wave_sum(state.y * w));
        a.x *= f;
        a.y *= f;
#pragma unroll
        for (int j = 0; j < NF; ++j) {
            if (j < k) {
                const float wj = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), j));
                a.x = fmaf(wj, x[j].x, a.x);
                a.y = fmaf(wj, x[j].y, a.y);
            }
        }
        m = mx;
    }
}

// A row's query and its current token, lanes as in fold_states.
template <typename T>
struct CurrentRow {
    float2 q, k, v;
    __device__ __forceinline__ void load(const T* q_row, const T* k_row, const T* v_row) {
        const int d = 2 * (threadIdx.x & (kWave - 1));
        q = load2<T>(q_row + d);
        k = load2<T>(k_row + d);
        v = load2<T>(v_row + d);
    }
    __device__ __forceinline__ float logit() const { return scaled_logit(wave_sum(fmaf(q.x, k.x, q.y * k.y))); }
    // the row's output from its merged state and the current token (NaN logits stay)
    __device__ __forceinline__ void finish(float m, float l, float2 a, T* out) const {
        const float s = logit(), mx = fmaxf(m, s);
        const float f = state_weight(m, l, mx), w = s == -INFINITY && mx != -INFINITY ? 0.0f : exp2_fast(s - mx);
        l = fmaf(l, f, w);
        store2<T>(out + 2 * (threadIdx.x & (kWave - 1)), fmaf(a.x, f, w * v.x) / l, fmaf(a.y, f, w * v.y) / l);
    }
};

// Workgroups of eight waves, one a CU.  (Four waves three times a CU, with as
// many bytes again on their way, were slower, 137 against 116 us at 8 x 64K and
// 43 against 35 at 131071 tokens: three times as many states to merge, and more
// places of memory read at once.)
constexpr int kDenseWaves = 8;
constexpr int kDenseThreads = kDenseWaves * kWave;
constexpr int kDenseBlocks = 256;

// What a further sequence costs a workgroup beside its tiles, in tiles: the
// queries, the join of the waves, the state or output.  Sequences 0, 14, 24 and 30
// tiles apart: a ragged batch of five up to 20001, fp16 8 queries a KV head, 32.5,
// 29.0, 28.0 and 27.8 us; 64 up to 2000 42.0, 35.5, 33.6 and 33.2; 16 up to 1000
// 19.9, 13.1, 13.5 and 14.5; 64 of one token 34.7, 11.0, 11.0 and 10.8.
constexpr int kSequenceCost = 24;

// Workgroups of a KV head: one a CU in all, with a tile for each wave (with two
// 4095 tokens of 8 KV heads take 12.4 us instead of 10.9).
int dense_workgroups(int64_t batch, int64_t kv_heads, int64_t max_tokens) {
    const int64_t target = kDenseBlocks / kv_heads < 1 ? 1 : kDenseBlocks / kv_heads;
    const int64_t tiles = (max_tokens + kPageTile - 1) / kPageTile;
    const int64_t most = (batch * ((tiles < 1 ? 1 : tiles) + kSequenceCost) + kDenseWaves - 1) / kDenseWaves;
    const int64_t one = (tiles + kDenseWaves - 1) / kDenseWaves;  // (a sequence alone has no further one)
    const int64_t n = batch == 1 ? one : most;
    return static_cast<int>(n < 1 ? 1 : n < target ? n : target);
}

// A workgroup's part of a sequence: tokens [t0, t1) of sequence b, part s of n;
// its state goes to place first + s.
struct DenseShare {
    int b, s, n, first, t0, t1;
};

// The work of one KV head is the batch's tiles of 32 tokens laid end to end
// (one at least a sequence, kSequenceCost places apart), cut among the grid's
// workgroups by the real lengths, which are read on the device: every workgroup
// takes as many places (one a wave at least), whether they are part of one long
// sequence or several short ones.  (Splits of each sequence by itself left a few
// workgroups more than fit at once, a second round: a ragged batch of five up to
// 20001, 64 query heads over 8 KV heads fp16 35 us.)  Workgroup w's state for
// sequence b has place w + b: one of the two grows from a part to the next, so
// places differ.  Each wave works its parts out by itself from the counts.  (The
// entry refuses batches of 2^30 places and more.)
struct DenseWalk {
    const PagedView& c;
    const int64_t most;
    const int lane, w;
    int per, r0, r1, b0, base;
    int count, tiles, start;  // lane i: sequence b0 + i
    uint64_t mask;            // its sequences still to come, of the 64 from b0 on

    __device__ __forceinline__ DenseWalk(const PagedView& view, int64_t max_tokens, int groups)
        : c(view), most(min(view.width << view.page_log2, max_tokens)), lane(threadIdx.x & (kWave - 1)),
          w(div_nonneg(blockIdx.x, view.kv_heads)), b0(0), base(0) {
        load();
        int total = __builtin_amdgcn_readlane(incl(), kWave - 1);
        for (int b = kWave; b < c.batch; b += kWave) {
            const uint32_t n = static_cast<uint32_t>(cost(b + lane, tiles_of(count_of(b + lane))));
            total += __builtin_amdgcn_readlane(static_cast<int>(wave_incl_scan(n, lane)), kWave - 1);
        }
        total -= kSequenceCost;
        per = max(div_nonneg(total + groups - 1, groups), kDenseWaves);
        r0 = static_cast<int>(min<int64_t>(static_cast<int64_t>(w) * per, int64_t{1} << 30));
        r1 = r0 + per;
        find();
    }
    __device__ __forceinline__ int count_of(int b) const {
        return b < c.batch ? static_cast<int>(clamp_count(c.counts[b], most)) : 0;
    }
    static __device__ __forceinline__ int tiles_of(int n) { return max((n + kPageTile - 1) / kPageTile, 1); }
    __device__ __forceinline__ int cost(int b, int n) const { return b < c.batch ? n + kSequenceCost : 0; }
    __device__ __forceinline__ void load() {
        count = count_of(b0 + lane);
        tiles = tiles_of(count);
    }
    __device__ __forceinline__ int incl() const {
        return static_cast<int>(wave_incl_scan(static_cast<uint32_t>(cost(b0 + lane, tiles)), lane));
    }
    __device__ __forceinline__ void find() {
        const int n = incl();
        start = base + n - cost(b0 + lane, tiles);
        mask = __ballot(b0 + lane < c.batch && start < r1 && start + tiles > r0);
        base += __builtin_amdgcn_readlane(n, kWave - 1);
    }
    // the next sequence that the workgroup has a part of
    __device__ __forceinline__ bool next(DenseShare& sh) {
        while (mask == 0) {
            b0 += kWave;
            if (b0 >= c.batch || base >= r1) return false;
            load();
            find();
        }
        const int src = __ffsll(static_cast<unsigned long long>(mask)) - 1;
        mask &= mask - 1;
        const int from = __builtin_amdgcn_readlane(start, src), to = from + __builtin_amdgcn_readlane(tiles, src);
        sh.b = b0 + src;
        const int w0 = from >= r0 ? w : from / per, w1 = to <= r1 ? w : (to - 1) / per;
        sh.s = w - w0;
        sh.n = w1 - w0 + 1;
        sh.first = w0 + sh.b;
        sh.t0 = (max(from, r0) - from) * kPageTile;
        sh.t1 = min(__builtin_amdgcn_readlane(count, src), (min(to, r1) - from) * kPageTile);
        return true;
    }
};

// The workgroup's waves hold the states of rows r0 .. r0 + rows - 1 of the
// group in LDS (s_m, s_l [W][ROWS], s_acc [W][ROWS][PITCH]): one state each to
// the partials, or, where the part is the whole sequence, the rows' outputs.
template <typename T, int ROWS, int PITCH>
__device__ __forceinline__ void emit_rows(const PagedAttend& a, const PagedView& c, const DenseShare& sh, int h,
                                          int group, int r0, const float (*s_m)[ROWS], const float (*s_l)[ROWS],
                                          const float (*s_acc)[ROWS][PITCH]) {
    constexpr int W = kDenseWaves;
    static_assert(ROWS <= W);
    __shared__ float s_cur[ROWS];
    const int rows = min(ROWS, group - r0);
    const int64_t kv = (static_cast<int64_t>(sh.b) * c.kv_heads + h) * 128;
    const int64_t row0 = static_cast<int64_t>(sh.b) * a.q_heads + static_cast<int64_t>(h) * group + r0;
    CurrentRow<T> cur;  // of the wave's own row, where the outputs are written here
    const int lane = threadIdx.x & (kWave - 1), own = threadIdx.x / kWave;
    if (sh.n == 1) {
        const T* q = static_cast<const T*>(a.q) + (row0 + min(own, rows - 1)) * 128;
        cur.load(q, static_cast<const T*>(a.cur_k) + kv, static_cast<const T*>(a.cur_v) + kv);
        const float x = cur.logit();
        if (lane == 0 && own < rows) s_cur[own] = x;
        __syncthreads();
    }
    // a row's maximum and the factors of its waves, once
    __shared__ float s_f[ROWS][W + 3];  // factors, maximum, sum, the current token's weight
    if (threadIdx.x < rows * W) {
        const int j = threadIdx.x / W, w = threadIdx.x % W;
        float mx = s_m[w][j];
        mx = fmaxf(mx, dpp_mov<0xB1>(mx));
        mx = fmaxf(mx, dpp_mov<0x4E>(mx));
        mx = fmaxf(mx, dpp_mov<0x141>(mx));
        if (sh.n == 1) mx = fmaxf(mx, s_cur[j]);
        const float f = state_weight(s_m[w][j], s_l[w][j], mx), l = row_sum<8>(f * s_l[w][j]);
        s_f[j][w] = f;
        if (w == 0) {
            float cur = 0.0f;
            if (sh.n == 1) cur = s_cur[j] == -INFINITY && mx != -INFINITY ? 0.0f : exp2_fast(s_cur[j] - mx);
            s_f[j][W] = mx;
            s_f[j][W + 1] = l + cur;
            s_f[j][W + 2] = cur;
        }
    }
    __syncthreads();
    if (own >= rows) return;
    float2 x = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const float2 y = *reinterpret_cast<const float2*>(&s_acc[w][own][2 * lane]);
        x.x = fmaf(s_f[own][w], y.x, x.x);
        x.y = fmaf(s_f[own][w], y.y, x.y);
    }
    if (sh.n == 1) {
        const float l = s_f[own][W + 1], w = s_f[own][W + 2];
        store2<T>(static_cast<T*>(a.out) + (row0 + own) * 128 + 2 * lane, fmaf(w, cur.v.x, x.x) / l,
                  fmaf(w, cur.v.y, x.y) / l);
    } else {
        float* p = a.partials + ((static_cast<int64_t>(sh.first + sh.s) * c.kv_heads + h) * group + r0 + own) * kState;
        st_pair(p + 2 + 2 * lane, x.x, x.y);
        if (lane == 0) st_pair(p, s_f[own][W], s_f[own][W + 1]);
    }
}
static_assert(kDenseWaves == 8, "a row's waves are eight neighbouring lanes, a wave for each of eight rows");

// Waves a row in the merge of a group's `n` states.
__device__ __forceinline__ int merge_share(int n, int group) {
    int share = 1;
    while (share * 2 * group <= kDenseWaves && share * 2 <= n) share *= 2;
    return share;
}

// Merges `n` states of each of the group's rows, `stride` floats apart: a row
// takes a wave, or several waves' shares of its states where the group has fewer
// rows than the workgroup waves.  done(r, m, l, a) by the wave that has row r's
// state.
template <typename F>
__device__ __forceinline__ void merge_rows(const float* ps, int64_t stride, int n, int group, F&& done) {
    constexpr int W = kDenseWaves;
    __shared__ __align__(8) float s_part[W][kState];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int share = merge_share(n, group);
    const int at_once = W / share;
    for (int r0 = 0; r0 < group; r0 += at_once) {
        const int r = r0 + wave / share, part = wave % share;
        float m = -INFINITY, l = 0.0f;
        float2 a = make_float2(0.0f, 0.0f);
        if (r < group) {
            const int s0 = n * part / share, s1 = n * (part + 1) / share;
            fold_states(ps + s0 * stride + static_cast<int64_t>(r) * kState, stride, s1 - s0, m, l, a);
        }
        if (share > 1) {
            __syncthreads();
            if (lane == 0) {
                s_part[wave][0] = m;
                s_part[wave][1] = l;
            }
            *reinterpret_cast<float2*>(&s_part[wave][2 + 2 * lane]) = a;
            __syncthreads();
            if (part == 0 && r < group) {
                for (int w = 1; w < share; ++w) {
                    const float m2 = s_part[wave + w][0], l2 = s_part[wave + w][1], mx = fmaxf(m, m2);
                    const float f = state_weight(m, l, mx), g = state_weight(m2, l2, mx);
                    l = fmaf(l, f, l2 * g);
                    a.x = fmaf(a.x, f, s_part[wave + w][2 + 2 * lane] * g);
                    a.y = fmaf(a.y, f, s_part[wave + w][3 + 2 * lane] * g);
                    m = mx;
                }
            }
        }
        if (part == 0 && r < group) done(r, m, l, a);
    }
}

// The last workgroup of a (sequence, KV head) in several parts merges them.
// More than kOneLevel merge in two levels, as one workgroup's reading of them is
// what takes the time: the last workgroup of every kSet leaves the set's state
// in the place of its first, and the last of those merges the sets' (157 parts,
// 40000 tokens of one KV head with 8 query heads: 15.6 us against 22.1 in one
// level; up to 32 parts one level is faster, 13.7 us against 15.7 at 16000
// tokens of 8 KV heads).  A (sequence, KV head) in several parts has kTickets
// tickets, the sets' from 1 on, in the place of the workgroup of its first part: no
// other goes on past that workgroup's end.  (A KV head has several workgroups only
// where they all are kDenseBlocks at most.)
constexpr int kOneLevel = 32, kSet = 16, kTickets = 32;
static_assert(kDenseBlocks / kSet + 1 <= kTickets);
static_assert(int64_t{kDenseBlocks} * kTickets * 4 <= kPagedTicketBytes);

template <typename T>
__device__ __forceinline__ void dense_merge(const PagedAttend& a, const PagedView& c, const DenseShare& sh, int h,
                                            int group) {
    __shared__ uint32_t s_last;
    if (sh.n == 1) return;
    const int lane = threadIdx.x & (kWave - 1);
    uint32_t* tickets = a.tickets + (static_cast<int64_t>(sh.first - sh.b) * c.kv_heads + h) * kTickets;
    const int64_t stride = static_cast<int64_t>(c.kv_heads) * group * kState;
    float* ps = a.partials + (static_cast<int64_t>(sh.first) * c.kv_heads + h) * group * kState;
    int n = sh.n, step = 1;
    if (n > kOneLevel) {
        const int set = sh.s / kSet, in_set = min(kSet, n - set * kSet);
        float* dst = ps + set * kSet * stride;
        if (!last_of(tickets + 1 + set, in_set, &s_last)) return;
        merge_rows(dst, stride, in_set, group, [&](int r, float m, float l, float2 a) {
            float* p = dst + static_cast<int64_t>(r) * kState;
            if (lane == 0) st_pair(p, m, l);
            st_pair(p + 2 + 2 * lane, a.x, a.y);
        });
        n = (n + kSet - 1) / kSet;
        step = kSet;
    }
    // the current token of the wave's first row on its way with the ticket
    CurrentRow<T> cur;
    const int64_t row0 = static_cast<int64_t>(sh.b) * a.q_heads + static_cast<int64_t>(h) * group;
    const int64_t kv = (static_cast<int64_t>(sh.b) * c.kv_heads + h) * 128;
    auto load = [&](int r) {
        cur.load(static_cast<const T*>(a.q) + (row0 + r) * 128, static_cast<const T*>(a.cur_k) + kv,
                 static_cast<const T*>(a.cur_v) + kv);
    };
    const int first = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) / merge_share(n, group);
    load(min(first, group - 1));
    if (!last_of(tickets, n, &s_last)) return;
    merge_rows(ps, step * stride, n, group, [&](int r, float m, float l, float2 acc) {
        if (r != first) load(r);
        cur.finish(m, l, acc, static_cast<T*>(a.out) + (row0 + r) * 128);
    });
}

__device__ __forceinline__ f32x4_t mfma_f16(const uint32_t (&a)[4], const uint32_t (&b)[4], f32x4_t c) {
    const half8_t x = __builtin_bit_cast(half8_t, make_uint4(a[0], a[1], a[2], a[3]));
    const half8_t y = __builtin_bit_cast(half8_t, make_uint4(b[0], b[1], b[2], b[3]));
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0);
}

// d[s] of lane group g becomes d[g] of lane group s.
__device__ __forceinline__ void exchange_quarters(uint32_t (&d)[4]) {
    const auto a = __builtin_amdgcn_permlane32_swap(d[0], d[2], false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(d[1], d[3], false, false);
    const auto x = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    const auto y = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    d[0] = x[0];
    d[1] = x[1];
    d[2] = y[0];
    d[3] = y[1];
}

// One workgroup a (share, KV head) for the whole group: its query heads are the
// 16 rows of matrix products (those past the group zero), so any group of 1 to
// 16 costs the same.  A wave takes tiles of 32 tokens, two of 16 for the logits:
//   dot_g[head, token] = q . (c - 8)   one 16 x 16 x 32 step per 32 dims, each
//                                    scale group by itself
//   S = sum_g delta_g dot_g + sum_g (low_g + 8 delta_g) qsum_g   in fp32, the
//                                    second sum by one more product (qsum in two
//                                    fp16 terms)
//   O[head, dim] += P . V            V as low + c delta in fp16 (bf16 tensors), or
//                                    exactly, in parts: low, 8 delta, and c - 8
//                                    times delta's upper seven and lower four bits
// so keys enter the logits unrounded: with the outlier channels that keys have,
// their rounding to fp16 was four times fp16's own in the result.  Codes are taken
// from their middle so that the two sums cancel little: with 1024 + c, the bits as
// they come, sum(q) a thousandfold went through the fp32 sums, and fp16 results of
// queries of one sign were 1.5 to 2.6 times as far off as their own rounding (now
// 1.00 of it, for 5 % of the time at 8 x 65535; sums that start at minus the
// thousandfold cost nothing and were still 1.8 times as far off).  (C layout: lane
// l holds rows 4 (l / 16) .. + 3 of column l % 16; A and B: lane l holds k-elements
// 8 (l / 16) .. + 7 of row / column l % 16.)
// A code becomes fp16 by its bits: 0x6400 | c is 1024 + c, and 0x6400 | 16 c
// is 1024 + 16 c; a packed subtraction, or an fma by 1/16, leaves c - 8 (nine
// instructions a dword of eight).  A token's 16-byte quarters are exchanged among
// the four lane groups (lane swaps), so that a step's 32 dims are one group's.
// What is held in fewer bits than fp32:
//   queries: scaled by a power of two per head, 16-bit ones exact down to 2^-18
//     (fp16) and 2^-21 (bf16) of the head's largest, fp32 ones two terms, off by at
//     most 2^-23 of themselves; below that any by 2^-29 of the largest.
//   weights: kept around 2^8, where fp16 keeps 11 bits, a second term for the
//     rest (22 bits) with fp16 and fp32 tensors.  bf16 ones have no such term and V
//     rounded to fp16: each off by at most half a step, 2^-11 of it, an eighth of
//     what the result's own rounding may be.  Both exact, as for fp16, 8 x 65535
//     took 140 us against 112 and the ragged batch 27.9 against 24.1, for a norm of
//     the error of 1.634e-3 of the result's instead of 1.652e-3.
// fp32 results are as far off as fp32 products of dequantised values, or less,
// where queries have no mean (relative 1.0e-6 against 2.1e-6 at 20001 tokens), and
// two to three times as far where they have one sign (3.1e-6 against 2.0e-6, at
// 64-dim groups 5.2e-6 and 1.7e-6): the two sums of S then cancel.
// 8 x 65536 tokens of 8 KV heads, 64-dim groups, 604 MB: bf16 112 to 118 us with
// the card (5.4 to 5.1 TB/s, where a plain read of as many bytes takes 86 us), fp16
// 138 to 145, fp32 154: bound by the vector instructions around the products, 325 a
// tile beside 18 matrix instructions in bf16.  A ragged batch of five up to 20001
// with 64 query heads, 32-dim groups, 77 MB: bf16 24.1, fp16 27.8, fp32 30 (94 by
// fp32 vector products).  4095 tokens, 5 MB, 10.9: a chain of reads, one tile a
// wave, the hand-off.
template <typename T, int G>
__global__ __launch_bounds__(kDenseThreads) void paged_dense_kernel(PagedAttend a, PagedView c, int64_t max_tokens,
                                                                         int groups) {
    constexpr int R = 128 / G;
    constexpr bool F32 = std::is_same_v<T, float>;
    constexpr int HALVES = R == 8 ? 2 : 1;        // groups of a 32-dim step
    // Query registers: fp32 two terms; 16-bit types a set for each half of a step,
    // zero in the other (31.2 us at 16-dim groups, a ragged fp16 batch, against 32.7
    // with the codes masked; fp32 has no registers left for that and masks them).
    constexpr int QSETS = F32 ? 2 : HALVES;
    constexpr int LOWS = R == 8 ? 2 : 1;          // products for the low terms (four groups each)
    constexpr int TERMS = std::is_same_v<T, bf16_t> ? 1 : 2;
    constexpr int QTOP = 5;                       // queries lie below 2^QTOP
    constexpr float kBase = 8.0f, kTop = 15.0f;   // weights start at 2^8 and may grow to 2^15
    constexpr float kNone = -3e38f;               // no weight yet
    constexpr int W = kDenseWaves, ROWS = 8, PITCH = 132;
    constexpr int ROWB = 8 * R;                                     // bytes of a token's scales
    constexpr int SLOADS = R == 8 ? 2 : 1, LOADS = 4 + SLOADS;      // 1 KB loads of a tile's scales, of a tile
    constexpr int STAGE = LOADS * 1024, STAGES = 2, PP = 20;
    constexpr int WAVE_BYTES = STAGES * STAGE + TERMS * 16 * PP * 4;
    // a wave's two stages, then its weights on their way from the logits' lanes
    // to the product's: [term][head][token pair (t, 16 + t) at 4 (t % 4) + t / 4]
    // (20 words a head: writes and reads meet different banks)
    __shared__ __align__(16) unsigned char s_mem[W * WAVE_BYTES];
    __shared__ float s_m[W][ROWS], s_l[W][ROWS];
    __shared__ __align__(16) float s_acc[W][ROWS][PITCH];
    const int h = blockIdx.x - div_nonneg(blockIdx.x, c.kv_heads) * c.kv_heads;
    const int group = a.q_heads / c.kv_heads;
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col = lane & 15, grp = lane >> 4;
    // A tile's codes and scales go from memory to LDS without passing through
    // registers, 1 KB an instruction, two tiles ahead of the one in work: lane
    // l's 16 bytes of load i are quarter (l % 8) ^ swz(token) of token 8 i + l /
    // 8, so that the reads below (16 tokens' equal quarters; four tokens' 64
    // bytes of V) meet 64 different banks.  swz(t) = 4 (t / 2 % 2) + t / 4 % 4.
    // Codes pass the caches by (8 x 65535 tokens 112.8 us against 118.0; what stays
    // in the last-level cache from call to call, 131071 and 4095 tokens and a ragged
    // batch, 0 to 3 % slower).
    struct Tile {
        uint4 k[2];
        uint32_t ks[2][R], v[8], vs[8];
    };
    const int64_t per_page = static_cast<int64_t>(c.kv_heads) << c.page_log2;
    const int64_t head_row = static_cast<int64_t>(h) << c.page_log2;
    const int in_page = (1 << c.page_log2) - 1;
    DenseShare sh;  // the part whose tiles are loaded
    int first = 0, tiles = 0;
    unsigned char* const mine = s_mem + wave * WAVE_BYTES;
    const uint32_t lds = __builtin_amdgcn_readfirstlane(
        static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char*)mine)));
    const int t8 = lane / 8, swz = 4 * ((t8 >> 1) & 1) + ((t8 >> 2) & 1);
    const uint32_t even = t8 * kCodeRow + 16 * ((lane % 8) ^ swz), odd = even ^ 32u;
    const uint32_t flat = R == 2 ? (lane & 31) * 16 : lane * 16;  // (R = 2: 512 bytes, twice)
    int32_t entries = -1;  // lane i: the page of this wave's tile i of a block of 64
    // starts tile i's loads into a stage; returns its live tokens
    auto issue = [&](int i, int stage) {
        if ((i & (kWave - 1)) == 0) {
            const int t = first + (i + lane) * (W * kPageTile);
            entries = t < sh.t1 && t >= 0 ? c.table[sh.b * c.width + (t >> c.page_log2)] : -1;
        }
        const int t = first + i * (W * kPageTile);
        const int32_t e = __builtin_amdgcn_readlane(entries, i & (kWave - 1));
        const bool there = static_cast<uint32_t>(e) < static_cast<uint32_t>(c.pages);
        const int64_t row = (there ? e : 0) * per_page + head_row + (t & in_page);
        const char* code = c.codes + row * kCodeRow;
        const char* sc = reinterpret_cast<const char*>(c.scales) + row * ROWB;
        // (the wave has read what the stage held; the loads write LDS behind the
        // compiler's back.  All of a tile's in one statement, which leaves m0, where
        // the LDS address stands, as it found it: the compiler takes no notice of m0
        // between statements.)
        uint32_t m0;
#define POPKV_TILE_LOADS(LAST)                                                                                      \
    asm volatile(                                                                                                   \
        "s_waitcnt lgkmcnt(0)\n\t"                                                                                  \
        "s_mov_b32 %0, m0\n\t"                                                                                      \
        "s_mov_b32 m0, %1\n\t"                                                                                      \
        "s_nop 1\n\t"                                                                                               \
        "global_load_lds_dwordx4 %2, %4 nt\n\t"                                                                     \
        "global_load_lds_dwordx4 %3, %4 offset:1024 nt\n\t"                                                         \
        "global_load_lds_dwordx4 %2, %4 offset:2048 nt\n\t"                                                         \
        "global_load_lds_dwordx4 %3, %4 offset:3072 nt\n\t"                                                         \
        "s_mov_b32 m0, %5\n\t"                                                                                      \
        "s_nop 1\n\t"                                                                                               \
        "global_load_lds_dwordx4 %6, %7\n\t" LAST                                                                   \
        "s_mov_b32 m0, %0"                                                                                          \
        : "=&s"(m0)                                                                                                 \
        : "s"(lds + stage * STAGE), "v"(even), "v"(odd), "s"(code), "s"(lds + stage * STAGE + 4096), "v"(flat),     \
          "s"(sc)                                                                                                   \
        : "memory")
        if constexpr (SLOADS == 2) POPKV_TILE_LOADS("global_load_lds_dwordx4 %6, %7 offset:1024\n\t");
        else POPKV_TILE_LOADS("");
#undef POPKV_TILE_LOADS
        return there ? min(kPageTile, sh.t1 - t) : 0;
    };
    // lane addresses in a stage: K of token col (+ 16), V dword col of tokens
    // grp + 4 j (+ 16), and their scales
    const int kswz = 4 * ((col >> 1) & 1) + ((col >> 2) & 3);
    const int ka = col * kCodeRow + 16 * (grp ^ kswz);
    const int va = grp * kCodeRow + 16 * ((4 ^ (4 * (grp >> 1))) + (col >> 2)) + 4 * (col & 3);
    const int ksa = 4096 + col * ROWB, vsa = 4096 + grp * ROWB + 4 * (R + 8 * col / G);
    auto read_tile = [&](int stage, Tile& x) {
        const unsigned char* p = mine + stage * STAGE;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            x.k[u] = *reinterpret_cast<const uint4*>(p + ka + 16 * u * kCodeRow);
            if constexpr (R == 2) {
                const uint2 w = *reinterpret_cast<const uint2*>(p + ksa + 16 * u * ROWB);
                x.ks[u][0] = w.x;
                x.ks[u][1] = w.y;
            } else {
#pragma unroll
                for (int g = 0; g < R; g += 4) {
                    const uint4 w = *reinterpret_cast<const uint4*>(p + ksa + 16 * u * ROWB + 4 * g);
                    x.ks[u][g] = w.x;
                    x.ks[u][g + 1] = w.y;
                    x.ks[u][g + 2] = w.z;
                    x.ks[u][g + 3] = w.w;
                }
            }
        }
        // v[2 j], v[2 j + 1]: tokens grp + 4 j and 16 + grp + 4 j
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int tok = 4 * (j >> 1) + 16 * (j & 1);
            x.v[j] = *reinterpret_cast<const uint32_t*>(p + (va ^ (16 * (j >> 1))) + tok * kCodeRow);
            x.vs[j] = *reinterpret_cast<const uint32_t*>(p + vsa + tok * ROWB);
        }
    };
    uint32_t* const s_p = reinterpret_cast<uint32_t*>(mine + STAGES * STAGE);
    const int pair = 4 * (col & 3) + (col >> 2);  // where the weights of tokens col and 16 + col go

    const CodeBits bits;
    const uint32_t half_mask[2] = {grp < 2 ? ~0u : 0u, grp < 2 ? 0u : ~0u};  // (fp32 at 16-dim groups)
    const uint32_t low_or_delta = grp == 1 ? 0x03020302u : 0x01000100u;  // byte picks of a scale pair

    // Starts a part: its first two tiles on their way, then its queries (row
    // `col`, dims 32 s + 8 grp .. + 7 in step s).
    Raw8<T> raw[4];
    int left = 0, next = 0;
    auto start_part = [&] {
        first = sh.t0 + wave * kPageTile;
        tiles = first < sh.t1 ? (sh.t1 - first + W * kPageTile - 1) / (W * kPageTile) : 0;
        left = tiles > 0 ? issue(0, 0) : 0;
        next = tiles > 1 ? issue(1, 1) : 0;
        const int64_t row =
            static_cast<int64_t>(sh.b) * a.q_heads + static_cast<int64_t>(h) * group + min(col, group - 1);
#pragma unroll
        for (int s = 0; s < 4; ++s) raw[s].load(static_cast<const T*>(a.q) + row * 128 + 8 * grp + 32 * s);
    };

    DenseWalk walk(c, max_tokens, groups);
    while (walk.next(sh)) {
        start_part();
        f32x4_t acc[8], low_acc = {0.0f, 0.0f, 0.0f, 0.0f};
        float ref[4], l[4];  // rows 4 grp + i: weights are 2^(logit - ref)
        // the queries in fp16, the largest magnitude of a head in [1/2, 1) 2^QTOP
        uint32_t qa[QSETS][4][4], ql[LOWS][4];
        float factor[4];  // of rows 4 grp + i
        {
            float q[4][8], top = 0.0f;
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    q[s][i] = col < group ? raw[s].get(i) : 0.0f;
                    top = fmaxf(top, fabsf(q[s][i]));
                }
            top = fmaxf(top, lane_xor<16>(top));
            top = fmaxf(top, lane_xor<32>(top));
            const int e = static_cast<int>((__float_as_uint(top) >> 23) & 0xffu) - 127;
            const float mine = ldexpf(kScaleHigh, e + 1 - QTOP);
#pragma unroll
            for (int i = 0; i < 4; ++i) factor[i] = __shfl(mine, 4 * grp + i);
            float sum[4];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                sum[s] = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    q[s][i] = ldexpf(q[s][i], QTOP - 1 - e);
                    sum[s] += q[s][i];
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t x = pack_half2(q[s][j], q[s][j + 4]);
                    if constexpr (F32) {
                        qa[0][s][j] = x;
                        qa[1][s][j] = pack_half2(q[s][j] - static_cast<float>(as_half2(x)[0]),
                                                 q[s][j + 4] - static_cast<float>(as_half2(x)[1]));
                    } else if constexpr (HALVES == 2) {
                        qa[0][s][j] = grp < 2 ? x : 0u;
                        qa[1][s][j] = grp < 2 ? 0u : x;
                    } else {
                        qa[0][s][j] = x;
                    }
                }
                sum[s] += lane_xor<16>(sum[s]);
            }
            // the low terms' product: lane group 0 holds the groups' sums of queries
            // for low, lane group 1 eight times them for delta (what codes lack in c
            // - 8), each as (high, rest)
            float qs[R];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const float other = lane_xor<32>(sum[s]);
                if constexpr (R == 8) {
                    qs[2 * s] = grp < 2 ? sum[s] : other;
                    qs[2 * s + 1] = grp < 2 ? other : sum[s];
                } else if constexpr (R == 4) {
                    qs[s] = sum[s] + other;
                } else {
                    qs[s / 2] = s & 1 ? qs[s / 2] + (sum[s] + other) : sum[s] + other;
                }
            }
#pragma unroll
            for (int g = 0; g < 4 * LOWS; ++g) {
                uint32_t x = 0;
                if (g < R) {
                    const float term = grp == 0 ? qs[g % R] : 8.0f * qs[g % R];
                    const float high = static_cast<float>(static_cast<_Float16>(term));
                    x = pack_half2(high, term - high);
                }
                ql[g / 4][g % 4] = grp < 2 ? x : 0u;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            ref[i] = kNone;
            l[i] = 0.0f;
        }
        auto fold = [&](Tile& x, int left) {
            f32x4_t s[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                uint32_t w[4] = {x.k[u].x, x.k[u].y, x.k[u].z, x.k[u].w};
                exchange_quarters(w);
                s[u] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int n = 0; n < LOWS; ++n) {
                    uint32_t lows[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                    for (int g = 0; g < 4 && g < R; ++g)
                        lows[g] = __builtin_amdgcn_perm(x.ks[u][4 * n + g], x.ks[u][4 * n + g], low_or_delta);
                    s[u] = mfma_f16(ql[n], lows, s[u]);
                }
                f32x4_t dot[R];
#pragma unroll
                for (int st = 0; st < 4; ++st) {
                    uint32_t cb[4];
                    half2_t code[4];
                    centred_pairs(bits, w[st], code);
#pragma unroll
                    for (int i = 0; i < 4; ++i) cb[i] = __builtin_bit_cast(uint32_t, code[i]);
#pragma unroll
                    for (int n = 0; n < HALVES; ++n) {
                        f32x4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
                        if (R == 2 && (st & 1)) sum = dot[st / 2];
                        if constexpr (F32) {
                            uint32_t x[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) x[i] = HALVES == 2 ? cb[i] & half_mask[n] : cb[i];
                            sum = mfma_f16(qa[0][st], x, mfma_f16(qa[1][st], x, sum));
                        } else {
                            sum = mfma_f16(qa[n][st], cb, sum);
                        }
                        dot[R == 2 ? st / 2 : HALVES * st + n] = sum;
                    }
                }
#pragma unroll
                for (int g = 0; g < R; ++g) {
                    const float delta = static_cast<float>(as_half2(x.ks[u][g])[1]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[u][i] = fmaf(delta, dot[g][i], s[u][i]);
                }
            }
            const bool whole = left == kPageTile;  // uniform; the branches stay branches
            const bool live[2] = {col < left, col + 16 < left};
            if (!whole) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    // what lies behind the last token may be anything
                    if (grp + 4 * (j >> 1) + 16 * (j & 1) >= left) x.vs[j] = 0u;
                    asm volatile("" : "+v"(x.vs[j]));
                }
            }
            float e[4][2], top = -INFINITY;
            auto exponents = [&] {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        e[i][u] = fmaf(s[u][i], factor[i], -ref[i]);
                        if constexpr (F32) e[i][u] = fmaf(s[u][i] * factor[i], kScaleLow / kScaleHigh, e[i][u]);
                    }
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            e[i][u] = live[u] ? e[i][u] : -INFINITY;
                            asm volatile("" : "+v"(e[i][u]));
                        }
                }
            };
            exponents();
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(e[i][0], e[i][1]));
            if (__ballot(top > kTop) != 0) {  // some weight would pass 2^15
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float mx = fmaxf(live[0] ? s[0][i] * factor[i] : -INFINITY,
                                     live[1] ? s[1][i] * factor[i] : -INFINITY);
                    mx = fmaxf(mx, dpp_mov<0xB1>(mx));
                    mx = fmaxf(mx, dpp_mov<0x4E>(mx));
                    mx = fmaxf(mx, dpp_mov<0x141>(mx));
                    mx = fmaxf(mx, dpp_mov<0x140>(mx));
                    const float to = fmaxf(mx - kBase, ref[i]);
                    const float f = exp2_fast(ref[i] - to);
                    l[i] *= f;
#pragma unroll
                    for (int d = 0; d < 8; ++d) acc[d][i] *= f;
                    if constexpr (TERMS == 2) low_acc[i] *= f;
                    ref[i] = to;
                }
                exponents();
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p0 = exp2_fast(e[i][0]), p1 = exp2_fast(e[i][1]);
                l[i] += p0 + p1;
                const uint32_t p = pack_half2(p0, p1);
                s_p[PP * (4 * grp + i) + pair] = p;
                if constexpr (TERMS == 2)
                    s_p[PP * (16 + 4 * grp + i) + pair] = pack_half2(p0 - static_cast<float>(as_half2(p)[0]),
                                                                p1 - static_cast<float>(as_half2(p)[1]));
            }
            // the wave reads its own weights next: one wave's LDS operations complete in order
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            uint32_t pa[TERMS][4];
#pragma unroll
            for (int n = 0; n < TERMS; ++n) {
                const uint4 w = *reinterpret_cast<const uint4*>(s_p + PP * (16 * n + col) + 4 * grp);
                pa[n][0] = w.x;
                pa[n][1] = w.y;
                pa[n][2] = w.z;
                pa[n][3] = w.w;
            }
            // a lane's eight dims 8 col .. + 7 of V: the low halves of the tokens'
            // dwords hold dims 0 .. 3, the high ones 4 .. 7
            if constexpr (TERMS == 1) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t vf[4][4];  // [dim][token pair]
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t v0 = x.v[2 * j], v1 = x.v[2 * j + 1];
                        uint32_t d[4];
                        dequantise_pairs(bits, half ? high_halves(v0, v1) : low_halves(v0, v1),
                                         as_half2(high_halves(x.vs[2 * j], x.vs[2 * j + 1])),
                                         as_half2(low_halves(x.vs[2 * j], x.vs[2 * j + 1])), d);
#pragma unroll
                        for (int i = 0; i < 4; ++i) vf[i][j] = d[i];
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[4 * half + i] = mfma_f16(pa[0], vf[i], acc[4 * half + i]);
                }
            } else {
                // exactly: codes as c - 8, times delta in two parts of at most seven
                // and four bits (products that fp16 holds, as deltas reach 7646 and
                // 15 times one may pass fp16's largest number), and low and 8 delta
                // by themselves (the same sums for each of a lane's dims)
                uint32_t lows[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) lows[j] = low_halves(x.vs[2 * j], x.vs[2 * j + 1]);
#pragma unroll
                for (int n = 0; n < TERMS; ++n) low_acc = mfma_f16(pa[n], lows, low_acc);
                uint32_t eights[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    eights[j] = __builtin_bit_cast(
                        uint32_t, as_half2(high_halves(x.vs[2 * j], x.vs[2 * j + 1])) * half2_t{8.0f16, 8.0f16});
#pragma unroll
                for (int n = 0; n < TERMS; ++n) low_acc = mfma_f16(pa[n], eights, low_acc);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t vh[4][4], vl[4][4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t v0 = x.v[2 * j], v1 = x.v[2 * j + 1];
                        const half2_t delta = as_half2(high_halves(x.vs[2 * j], x.vs[2 * j + 1]));
                        const half2_t top7 = as_half2(__builtin_bit_cast(uint32_t, delta) & 0xfff0fff0u);
                        half2_t code[4];
                        centred_pairs(bits, half ? high_halves(v0, v1) : low_halves(v0, v1), code);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            vh[i][j] = __builtin_bit_cast(uint32_t, code[i] * top7);
                            vl[i][j] = __builtin_bit_cast(uint32_t, code[i] * (delta - top7));
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        f32x4_t& sum = acc[4 * half + i];
                        sum = mfma_f16(pa[0], vh[i], sum);
                        sum = mfma_f16(pa[TERMS - 1], vh[i], sum);
                        sum = mfma_f16(pa[0], vl[i], sum);
                        if constexpr (F32) sum = mfma_f16(pa[1], vl[i], sum);
                    }
                }
            }
            // the next tile's weights overwrite s_p only after every lane has read
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        };
        // tile i is whole once at most the next one's loads are outstanding
        auto arrived = [&](bool next) {
            if (next) asm volatile("s_waitcnt vmcnt(%0)" : : "n"(LOADS) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
        };
#pragma unroll 1
        for (int i = 0; i < tiles; ++i) {
            // the two waves of a SIMD go first in turn: left to itself the older one
            // ends early and leaves the other alone (131071 tokens: 20 and 28 us; the
            // launch at 8 x 65535 112.8 us, without turns 117.1)
            if (((i ^ (wave >> 2)) & 1) != 0) __builtin_amdgcn_s_setprio(1);
            else __builtin_amdgcn_s_setprio(0);
            Tile x;
            arrived(i + 1 < tiles);
            read_tile(i & 1, x);
            const int after = i + 2 < tiles ? issue(i + 2, i & 1) : 0;
            fold(x, left);
            left = next;
            next = after;
        }

        __builtin_amdgcn_s_setprio(0);
#pragma unroll
        for (int i = 0; i < 4; ++i) l[i] = row_sum<16>(l[i]);
        if constexpr (TERMS == 2)
#pragma unroll
            for (int d = 0; d < 8; ++d) acc[d] += low_acc;
        // the waves' states meet in LDS, eight heads at a time
        for (int r0 = 0; r0 < group; r0 += ROWS) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 4 * grp + i - r0;
                if (r >= 0 && r < ROWS) {
                    if (col == 0) {
                        s_m[wave][r] = l[i] == 0.0f ? -INFINITY : ref[i];
                        s_l[wave][r] = l[i];
                    }
                    float4* dst = reinterpret_cast<float4*>(&s_acc[wave][r][8 * col]);
                    dst[0] = make_float4(acc[0][i], acc[1][i], acc[2][i], acc[3][i]);
                    dst[1] = make_float4(acc[4][i], acc[5][i], acc[6][i], acc[7][i]);
                }
            }
            __syncthreads();
            emit_rows<T, ROWS, PITCH>(a, c, sh, h, group, r0, s_m, s_l, s_acc);
            __syncthreads();
        }
        dense_merge<T>(a, c, sh, h, group);
    }
}

template <typename T, int G>
hipError_t launch_dense_t(const PagedAttend& a, const PagedView& c, int64_t max_tokens, hipStream_t stream) {
    const int per_head = dense_workgroups(c.batch, c.kv_heads, max_tokens);
    hipLaunchKernelGGL((paged_dense_kernel<T, G>), dim3(static_cast<unsigned>(per_head * c.kv_heads)),
                       dim3(kDenseThreads), 0, stream, a, c, max_tokens, per_head);
    return hipGetLastError();
}

}  // namespace

int64_t paged_dense_items(int64_t batch, int64_t kv_heads, int64_t max_tokens) {
    return dense_workgroups(batch, kv_heads, max_tokens) + batch;
}

hipError_t launch_paged_dense(const PagedAttend& a, const PagedView& c, int64_t max_tokens, int dtype, int dim_group,
                              hipStream_t stream) {
#define POPKV_CALL(T, G) launch_dense_t<T, G>(a, c, max_tokens, stream)
    POPKV_PAGED_T(POPKV_CALL)
#undef POPKV_CALL
}

}  // namespace popkv
