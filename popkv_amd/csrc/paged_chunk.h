// Kernels of the chunk attention over the paged 4-bit K/V cache, instantiated for
// each element type by a source of its own (paged_chunk_*.hip).
#pragma once

#include "paged_attention.h"

namespace popkv {
namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

constexpr int kFrag = 1024;                   // bytes of one operand of a 32 x 32 x 16 product

__device__ __forceinline__ f32x16_t mfma_h(const uint4& a, const uint4& b, f32x16_t c) {
    const half8_t x = __builtin_bit_cast(half8_t, a), y = __builtin_bit_cast(half8_t, b);
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16_t mfma_b(const uint4& a, const uint4& b, f32x16_t c) {
    const bf16x8_t x = __builtin_bit_cast(bf16x8_t, a), y = __builtin_bit_cast(bf16x8_t, b);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
}

// Two floats as N pairs of bf16 terms that add up to them.  Of several terms the first
// is held in bf16's range, which the largest floats round past; infinities and NaN then
// stand in the others.
typedef __bf16 bf16x2_raw __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
template <int N>
__device__ __forceinline__ void bf16_terms(float x, float y, uint32_t (&t)[N]) {
    f32x2_t held = {x, y};
    if constexpr (N > 1) {
        constexpr float kTop = 0x1.fep127f;
        held = f32x2_t{__builtin_amdgcn_fmed3f(x, -kTop, kTop), __builtin_amdgcn_fmed3f(y, -kTop, kTop)};
    }
    t[0] = __builtin_bit_cast(uint32_t, __builtin_convertvector(held, bf16x2_raw));
#pragma unroll
    for (int i = 1; i < N; ++i) {
        x -= __uint_as_float(t[i - 1] << 16);
        y -= __uint_as_float(t[i - 1] & 0xffff0000u);
        t[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{x, y}), bf16x2_raw));
    }
}
// Eight elements of an operand.
template <int N, typename F>
__device__ __forceinline__ void bf16_operand(F&& x, uint4 (&q)[N]) {
    uint32_t t[4][N];
#pragma unroll
    for (int j = 0; j < 4; ++j) bf16_terms<N>(x(2 * j), x(2 * j + 1), t[j]);
#pragma unroll
    for (int n = 0; n < N; ++n) q[n] = make_uint4(t[0][n], t[1][n], t[2][n], t[3][n]);
}

// Whether one of eight elements is an infinity or NaN.
template <typename T>
__device__ __forceinline__ bool odd_values(const Raw8<T>& x) {
    bool odd = false;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) odd = odd || (__float_as_uint(x.get(i)) & 0x7f800000u) == 0x7f800000u;
    } else {
        constexpr uint32_t kTop = Elem<T>::kDtype == POPKV_DTYPE_BF16 ? 0x7f80u : 0x7c00u;
        typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
        u16x2 m = __builtin_bit_cast(u16x2, x.u.x & 0x7fff7fffu);
        m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, x.u.y & 0x7fff7fffu));
        m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, x.u.z & 0x7fff7fffu));
        m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, x.u.w & 0x7fff7fffu));
        odd = max(m[0], m[1]) >= kTop;
    }
    return odd;
}
__device__ __forceinline__ bool is_odd(float x) { return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u; }
template <typename T>
__device__ __forceinline__ void clear_odd(Raw8<T>& x) {
    if constexpr (sizeof(T) == 4) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = is_odd(x.get(i)) ? 0.0f : x.get(i);
        x.a = make_float4(y[0], y[1], y[2], y[3]);
        x.b = make_float4(y[4], y[5], y[6], y[7]);
    } else {
        auto word = [&](uint32_t w, int i) {
            return (is_odd(x.get(i)) ? 0u : w & 0xffffu) | (is_odd(x.get(i + 1)) ? 0u : w & 0xffff0000u);
        };
        x.u = make_uint4(word(x.u.x, 0), word(x.u.y, 2), word(x.u.z, 4), word(x.u.w, 6));
    }
}

// What the kernel holds of each element type.  EXACT: cached keys enter the logits
// unrounded (else in fp16).
template <typename T, bool EXACT>
struct ChunkTypes {
    static constexpr bool F32 = std::is_same_v<T, float>;
    static constexpr bool F16 = std::is_same_v<T, f16_t>;
    static constexpr int QT = F32 ? 2 : 1;         // fp16 terms of the queries
    static constexpr int KT = EXACT ? 2 : 1;       // of the cached keys
    static constexpr int VT = F32 ? 2 : 1;         // of the cached values
    static constexpr int CT = F32 || F16 ? 2 : 1;  // of their weights
    static constexpr int NT = F32 ? 3 : 1;         // planes of the new tokens (fp32: bf16 terms)
    static constexpr int PT = F32 ? 3 : F16 ? 2 : 1;  // terms of the weights on new tokens
    static constexpr int QPLANES = F32 ? 3 : 1;
    // query operands kept for the second pass: for cached tokens, for new ones, the low
    // terms' (of 1 KB, eight a plane)
    static constexpr int STORED = 8 * (QT + QPLANES) + 2;
    static constexpr int PLANES = KT + VT > 2 * NT ? KT + VT : 2 * NT;
};

static_assert(ChunkTypes<float, true>::STORED == kChunkStored32 && ChunkTypes<bf16_t, true>::STORED == kChunkStored16 &&
              ChunkTypes<f16_t, true>::STORED == kChunkStored16);

// Where lane l's sixteen bytes of value operand i of four lie in its KB: writers
// of one instruction (16 dwords of codes) meet different banks, readers too.
__device__ __forceinline__ int value_slot(int l, int i) { return (l ^ (i | ((l >> 4 & 1) << 3))) * 16; }

// A workgroup's shape: WR waves of 32 rows (a row is a token and a head of the
// group, heads innermost) times WT waves that share a tile's tokens.
template <int WR_, int WT_>
struct ChunkShape {
    static constexpr int WR = WR_, WT = WT_, W = WR * WT, THREADS = W * kWave;
    static constexpr int ROWS = 32 * WR;
    static constexpr int TILE = WT == 4 ? 128 : 64, SUB = TILE / 32;  // tokens of a tile
    static constexpr int UNITS = 4 * TILE;              // quarters of keys, or dwords of four tokens' values
    static constexpr bool ROLES = THREADS >= 2 * UNITS;               // half of the threads stage keys, half values
    static constexpr int PER = ROLES ? 1 : UNITS / THREADS;
    static constexpr int STATE = WR * (32 * 128 + 64);                // floats of a part's state
};

// Sequence b's chunk: its new tokens, cached tokens, and per tile of rows j the
// tiles of both.
struct ChunkSizes {
    int rows, count;
    __device__ __forceinline__ ChunkSizes(const PagedChunk& a, const PagedView& c, int64_t max_tokens, int b)
        : rows(static_cast<int>(a.tokens ? clamp_count(a.tokens[b], a.rows) : a.rows)),
          count(static_cast<int>(clamp_count(c.counts[b], min(c.width << c.page_log2, max_tokens)))) {}
};

struct ChunkPart {
    int b, j, rows, count, x0, x1, s, n, first;
};

// The work of one KV head is the batch's tiles of rows laid end to end, each as long
// as its tiles of tokens, cut among the grid's workgroups by the real lengths, which
// are read on the device.  Workgroup w's state of a tile of rows that goes on from
// the workgroup before has place 2 w, of one that begins in it 2 w + 1.  Each wave
// works its parts out by itself.
template <typename S>
struct ChunkWalk {
    const PagedChunk& a;
    const PagedView& c;
    const int64_t most;
    const int lane, w, items, blocks, group;
    int4* const held;  // entry i: item i0 + i's rows, count, tiles and start (in LDS: no registers between parts)
    int per, r0, r1, i0, base;
    uint64_t mask;
    struct Item {
        int rows, count, tiles;
    };

    __device__ __forceinline__ ChunkWalk(const PagedChunk& a_, const PagedView& c_, int64_t max_tokens, int w_, int groups,
                                         int4* held_)
        : a(a_), c(c_), most(max_tokens), lane(threadIdx.x & (kWave - 1)), w(w_),
          items(c.batch * static_cast<int>(a.row_blocks)), blocks(static_cast<int>(a.row_blocks)),
          group(div_nonneg(a.q_heads, c.kv_heads)), held(held_), i0(0), base(0) {
        int total = 0;
        Item x{};
        for (int i = (items - 1) & ~(kWave - 1); i >= 0; i -= kWave) {  // (the first ones stay)
            x = load(i);
            total += __builtin_amdgcn_readlane(incl(x), kWave - 1);
        }
        per = max(div_nonneg(total + groups - 1, groups), a.least);
        r0 = static_cast<int>(min<int64_t>(static_cast<int64_t>(w) * per, int64_t{1} << 30));
        r1 = r0 + per;
        find(x);
    }
    __device__ __forceinline__ Item load(int first) const {
        const int i = first + lane, b = min(blocks == 1 ? i : i / blocks, c.batch - 1), j = i - b * blocks;
        const ChunkSizes z(a, c, most, b);
        const int all = z.rows * group;  // (the entry holds rows * heads below 2^30)
        const int seen = min(((j + 1) * S::ROWS - 1) / group + 1, z.rows);
        const int tiles = (z.count + S::TILE - 1) / S::TILE + (seen + S::TILE - 1) / S::TILE;
        return {z.rows, z.count, i < items && j * S::ROWS < all ? tiles : 0};
    }
    __device__ __forceinline__ int cost(const Item& x) const { return x.tiles > 0 ? x.tiles + a.item_cost : 0; }
    __device__ __forceinline__ int incl(const Item& x) const {
        return static_cast<int>(wave_incl_scan(static_cast<uint32_t>(cost(x)), lane));
    }
    // (every wave of the workgroup writes the same; all are past reading the last)
    __device__ __forceinline__ void find(const Item& x) {
        const int n = incl(x), start = base + n - cost(x);
        mask = __ballot(x.tiles > 0 && start < r1 && start + x.tiles > r0);
        held[lane] = make_int4(x.rows, x.count, x.tiles, start);
        base += __builtin_amdgcn_readlane(n, kWave - 1);
    }
    __device__ __forceinline__ bool next(ChunkPart& p) {
        while (mask == 0) {
            i0 += kWave;
            if (i0 >= items || base >= r1) return false;
            __syncthreads();
            find(load(i0));
        }
        const int src = __ffsll(static_cast<unsigned long long>(mask)) - 1;
        mask &= mask - 1;
        const int4 x = held[src];
        const int from = __builtin_amdgcn_readfirstlane(x.w), to = from + __builtin_amdgcn_readfirstlane(x.z);
        p.b = div_nonneg(i0 + src, blocks);
        p.j = i0 + src - p.b * blocks;
        p.rows = __builtin_amdgcn_readfirstlane(x.x);
        p.count = __builtin_amdgcn_readfirstlane(x.y);
        const int w0 = from >= r0 ? w : div_nonneg(from, per), w1 = to <= r1 ? w : div_nonneg(to - 1, per);
        p.s = w - w0;
        p.n = w1 - w0 + 1;
        p.first = w0;
        p.x0 = max(from, r0) - from;
        p.x1 = min(to, r1) - from;
        return true;
    }
};

// The lane's number, worked out where it stands: for rare paths in loops that have no
// register left to keep it in.
__device__ __forceinline__ int fresh_lane() {
    uint32_t all = ~0u;
    asm volatile("" : "+s"(all));
    return static_cast<int>(__builtin_amdgcn_mbcnt_hi(all, __builtin_amdgcn_mbcnt_lo(all, 0u)));
}

// Weights of 32 tokens as operands of two products of 16 tokens each, in N terms of a
// type (QK, PV: the products of an operand beside them).  SUM: their sum is the rounded
// ones' (two a step).
template <int N, bool SUM_, int QK_>
struct HalfWeights {
    static constexpr bool SUM = SUM_;
    static constexpr int QK = QK_, PV = N;
    uint4 at[N][2];
    __device__ __forceinline__ void pack(const float (&p)[16]) {
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            uint32_t w[4], rest[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p0 = p[8 * st + 2 * j], p1 = p[8 * st + 2 * j + 1];
                w[j] = pack_half2(p0, p1);
                rest[j] = pack_half2(p0 - static_cast<float>(as_half2(w[j])[0]),
                                     p1 - static_cast<float>(as_half2(w[j])[1]));
            }
            at[0][st] = make_uint4(w[0], w[1], w[2], w[3]);
            if constexpr (N == 2) at[1][st] = make_uint4(rest[0], rest[1], rest[2], rest[3]);
        }
    }
    // of the first terms
    __device__ __forceinline__ float sum() const {
        const half2_t one = {1.0f16, 1.0f16};
        float x = 0.0f;
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            x = __builtin_amdgcn_fdot2(as_half2(at[0][st].x), one, x, false);
            x = __builtin_amdgcn_fdot2(as_half2(at[0][st].y), one, x, false);
            x = __builtin_amdgcn_fdot2(as_half2(at[0][st].z), one, x, false);
            x = __builtin_amdgcn_fdot2(as_half2(at[0][st].w), one, x, false);
        }
        return x;
    }
};
template <int N, bool SUM_, int QK_>
struct Bf16Weights {
    static constexpr bool SUM = SUM_;
    static constexpr int QK = QK_, PV = N;
    uint4 at[N][2];
    __device__ __forceinline__ void pack(const float (&p)[16]) {
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            uint4 t[N];
            bf16_operand<N>([&](int j) { return p[8 * st + j]; }, t);
#pragma unroll
            for (int n = 0; n < N; ++n) at[n][st] = t[n];
        }
    }
    __device__ __forceinline__ float sum() const {
        const bf16x2_t one = __builtin_bit_cast(bf16x2_t, 0x3f803f80u);
        float x = 0.0f;
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            x = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, at[0][st].x), one, x, false);
            x = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, at[0][st].y), one, x, false);
            x = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, at[0][st].z), one, x, false);
            x = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, at[0][st].w), one, x, false);
        }
        return x;
    }
};

// Eight operands of products, four of them read ahead: products(at, product) calls
// product(i, operand) with the sixteen bytes at(i), i = 0 .. 7.
template <typename A, typename F>
__device__ __forceinline__ void products(A&& at, F&& product) {
    uint4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const uint4*>(at(i));
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        product(i, x[i % 4]);
        if (i < 4) x[i] = *reinterpret_cast<const uint4*>(at(i + 4));
    }
}
// For the scheduler, of such products and other work: M products an operand, V vector
// instructions and E exponentials behind each.
template <int M, int V, int E>
__device__ __forceinline__ void interleave() {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, M, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, V, 0);
        if (E) __builtin_amdgcn_sched_group_barrier(0x400, E, 0);
        if (i < 4) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
}

// What a row's weights are 2^(logit - x) y with: its largest weights' logits less x lie
// about zero, where a float's step is small.  (Rows past the last one weigh nothing.)
constexpr float kBase = 8.0f;  // weights start at 2^kBase
__device__ __forceinline__ float2 row_sums(float ref, float l, bool live) {
    return live ? make_float2(ref + kBase, exp2_fast(kBase) / l) : make_float2(INFINITY, 0.0f);
}

// Sixteen neighbouring values of a row, times f.
template <typename T>
__device__ __forceinline__ void store16(T* p, const f32x16_t& x, float f) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 16; j += 4)
            *reinterpret_cast<float4*>(p + j) = make_float4(x[j] * f, x[j + 1] * f, x[j + 2] * f, x[j + 3] * f);
    } else {
#pragma unroll
        for (int j = 0; j < 16; j += 8)
            *reinterpret_cast<uint4*>(p + j) =
                make_uint4(pack2<T>(x[j] * f, x[j + 1] * f), pack2<T>(x[j + 2] * f, x[j + 3] * f),
                           pack2<T>(x[j + 4] * f, x[j + 5] * f), pack2<T>(x[j + 6] * f, x[j + 7] * f));
    }
}

// 4 N of them.
template <typename T, int N>
__device__ __forceinline__ void store4s(T* p, const float4 (&x)[N], float f) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int k = 0; k < N; ++k)
            *reinterpret_cast<float4*>(p + 4 * k) = make_float4(x[k].x * f, x[k].y * f, x[k].z * f, x[k].w * f);
    } else {
        uint32_t w[2 * N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            w[2 * k] = pack2<T>(x[k].x * f, x[k].y * f);
            w[2 * k + 1] = pack2<T>(x[k].z * f, x[k].w * f);
        }
        if constexpr (N == 1) {
            *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        } else {
#pragma unroll
            for (int k = 0; k < 2 * N; k += 4)
                *reinterpret_cast<uint4*>(p + 2 * k) = make_uint4(w[k], w[k + 1], w[k + 2], w[k + 3]);
        }
    }
}

// One pass over the tokens with each row's running reference and sum.  A workgroup has
// a block of rows of one (sequence, KV head) and goes through its part's tiles: first
// cached ones, dequantised once a workgroup into operands of the matrix instructions,
// then the chunk's own.  Products stand transposed,
//   S[token, row] = K q    P = 2^(S f - ref)    O[dim, row] += V P
// so that a lane holds one row's logits of 16 tokens, which are, in their order, what
// the second product takes from it: weights never leave the lane, and which token is
// which place of an operand is settled where values are staged.  (C layout of 32 x 32
// products: lane l holds column l % 32, rows 8 (i / 4) + 4 (l / 32) + i % 4; A and B:
// lane l holds elements 8 (l / 32) .. + 7 of row / column l % 32.)
// Cached keys: in fp16, low + c delta rounded once, for bf16 rows; EXACT, for fp16 and
// fp32 rows and wherever weights are gathered, as (c - 8) times delta's upper seven and
// lower four bits, which fp16 holds, and low and 8 delta by the queries' sums.
// What is held in fewer bits than fp32, half a step each, and why:
//   queries of cached tokens: scaled by a power of two a row, 16-bit ones exact down to
//     2^-18 of the row's largest, fp32 ones two terms;
//   keys of bf16 rows, 2^-11: exact ones are another plane and 17 products instead of 8;
//   values, 2^-11, with 16-bit rows: fp32 ones are two terms;
//   weights: bf16 rows fp16 on cached tokens and bf16 on new ones; fp16 rows two fp16
//     terms; fp32 rows two fp16 and three bf16 terms.
// Error of the results against 64 bits, norm over norm, beside plain float32 products of
// dequantised rows: bf16 1.64e-3 to 1.72e-3 over cached tokens, 1.78e-3 to 2.06e-3 over new
// ones (1.66e-3, its own rounding), fp16 2.7e-4 to 2.9e-4 and 2.0e-4 (2.1e-4; with cached
// values in two terms too, for 20 % of the time), fp32 2e-7 to 2.4e-6 with the logits'
// size (1.1e-6 to 2.7e-6 where keys have outlier channels).  A bf16 row's result has
// other bits where weights are gathered, its keys then being exact.
// Sums are fp32 of weights up to 2^16: they hold values up to about 2^90.
// Eight waves of 32 rows, one workgroup a CU, where a sequence has the rows: dequantised
// tiles are shared by 256 rows, two waves a SIMD, tiles staged one ahead into the other
// half of LDS and their codes loaded two ahead, page entries three.  The vector work of
// 32 tokens (16 exponentials a lane among it) stands beside the products of the next 32,
// operands read four ahead: 2048 rows of 4 heads behind 30719 tokens 1295 us against
// 1393 with one after the other.  Values masked where they are staged and not where they are
// loaded (1210 against 1295): nothing waits for a load.  1.2 ms, 900 TFLOP/s, where a
// product of 8192 reaches 1190 to 1280.  Bound by how far the vector instructions, about
// 250 a wave and tile of 64 tokens, stand beside its 32 matrix ones with two waves a SIMD:
// of a pass's 2.76M cycles the vector unit is active for 1.24M (the matrix instructions'
// issue among them) and the matrix unit for 1.02M, and waves wait for 35 % of their time.
// All 256 registers are taken: the eight-wave kernels spill 48 to 69 more (188 to 264 bytes
// of scratch a lane), most outside the loops over tiles; the exact form reads some back
// inside them.
// Fewer rows: waves share a tile's tokens instead (WT), and join by dims in LDS.  (The
// 32-row bf16 form spills 8 registers, the others none; fp32 rows and the exact 32-row form
// take 350 to 440, one wave a SIMD.)
template <typename T, int G, bool EXACT, typename S>
__global__ __launch_bounds__(S::THREADS, (sizeof(T) == 4 || (EXACT && S::WT == 4) ? 1 : 2)) void paged_chunk_kernel(
    PagedChunk a, PagedView c, int64_t max_tokens, int groups) {
    using C = ChunkTypes<T, EXACT>;
    constexpr int R = 128 / G;
    constexpr int LOWS = R == 8 ? 2 : 1;
    constexpr int QTOP = 5;
    constexpr float kNone = -3e38f, kFull = 65504.0f;
    constexpr int PLANE = S::SUB * 8 * kFrag, BUF = C::PLANES * PLANE;
    constexpr int BUFS = S::WR == 8 && 2 * BUF <= 140 * 1024 ? 2 : 1;
    static_assert(BUF <= 150 * 1024);
    constexpr int JOIN = S::WT == 1 ? 0 : S::W * (16384 + 256);  // the waves' states
    __shared__ __align__(16) unsigned char s_mem[BUFS * BUF > JOIN ? BUFS * BUF : JOIN];
    __shared__ __align__(16) uint32_t s_scale[BUFS][EXACT ? S::TILE : 1][R];
    __shared__ float s_bias[BUFS][S::TILE];
    __shared__ int s_ragged[BUFS][S::W], s_odd_keys[BUFS][S::W];

    const int h = blockIdx.x - div_nonneg(blockIdx.x, c.kv_heads) * c.kv_heads;
    const int w_id = div_nonneg(blockIdx.x, c.kv_heads);
    const int tid = threadIdx.x, lane = tid & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int wr = wave % S::WR, wt = wave / S::WR;
    const int col = lane & 31, half = lane >> 5;
    const int group = div_nonneg(a.q_heads, c.kv_heads);

    // rows behind a sequence's last one
    if (a.fill && a.tokens)
        for (int64_t i = blockIdx.x; i < static_cast<int64_t>(c.batch) * a.q_heads; i += gridDim.x) {
            const int64_t b = i / a.q_heads;
            T* const out = static_cast<T*>(a.out) + b * a.o_bs + (i - b * a.q_heads) * a.o_hs;
            constexpr int V = 128 * sizeof(T) / 16;
            for (int64_t k = clamp_count(a.tokens[b], a.rows) * V + tid; k < a.rows * V; k += S::THREADS)
                reinterpret_cast<uint4*>(out + k / V * a.o_ts)[k % V] = make_uint4(0u, 0u, 0u, 0u);
        }

    // a thread's part of a tile: a quarter of a token's key, a dword of four tokens'
    // values, which share a page
    constexpr int VALUES_FROM = S::ROLES ? S::UNITS : 0;
    const bool keys = !S::ROLES || wave < S::UNITS / kWave, vals = !S::ROLES || wave >= S::UNITS / kWave;
    const int64_t per_page = static_cast<int64_t>(c.kv_heads) << c.page_log2;
    const int64_t head_row = static_cast<int64_t>(h) << c.page_log2;
    const int in_page = (1 << c.page_log2) - 1;
    const CodeBits bits;
    // where dim 0 of a unit's dword goes, its quad's eight bytes; dim e at value_dim(, e)
    auto value_at = [&](int unit) {
        const int dw = unit % 16, quad = unit / 16, u = quad / 8, s = quad % 8 / 4, r = quad % 4;
        const int i = dw % 8 / 2, m = 16 * (dw % 2) + 4 * (dw / 8);
        return ((u * 2 + s) * 4 + i) * kFrag + value_slot((r & 1) * 32 + m, i) + 8 * (r >> 1);
    };
    auto value_dim = [&](unsigned char* base, int at, int e) {
        return reinterpret_cast<uint2*>(base + (at ^ ((e % 4) * 16 | e / 4 * 128)));
    };
    auto key_at = [&](unsigned char* base, int unit, int e) {  // eight dims 32 quarter + 8 e
        const int token = unit / 4, quarter = unit % 4;
        return reinterpret_cast<uint4*>(base + (token / 32 * 8 + 4 * (quarter & 1) + e) * kFrag +
                                        (quarter / 2 * 32 + token % 32) * 16);
    };
    auto new_key_at = [&](unsigned char* base, int unit, int e) {  // eight dims 8 quarter + 32 e (four threads 64 bytes)
        const int token = unit / 4, quarter = unit % 4;
        return reinterpret_cast<uint4*>(base + (token / 32 * 8 + 4 * (e & 1) + quarter) * kFrag +
                                        (e / 2 * 32 + token % 32) * 16);
    };

    __shared__ int4 s_items[kWave];
    ChunkWalk<S> walk(a, c, max_tokens, w_id, groups, s_items);
    ChunkPart part;
    while (walk.next(part)) {
        const int b = part.b;
        const int rows = part.rows, count = part.count;
        const int cached_tiles = (count + S::TILE - 1) / S::TILE;
        const int all = rows * group, row0 = part.j * S::ROWS;  // (below 2^30)
        // (a lane's row, worked out where it is needed: registers between are dear)
        struct Row {
            int t, head;
            bool live;
        };
        auto own_row = [&] {
            int k = col;
            asm volatile("" : "+v"(k));
            const int row = min(row0 + 32 * wr + k, all - 1);
            const int t = (group & (group - 1)) == 0 ? row >> __builtin_ctz(group) : row / group;
            return Row{t, h * group + row - t * group, row0 + 32 * wr + k < all};
        };
        auto query = [&](const Row& r) {
            return static_cast<const T*>(a.q) + b * a.q_bs + r.head * a.q_hs + static_cast<int64_t>(r.t) * a.q_ts +
                   64 * half;
        };
        // what the second pass reads of these rows: the query operands of both kinds of
        // tokens, their factors, their sums
        const int64_t row_tile = (static_cast<int64_t>(b) * c.kv_heads + h) * a.row_blocks * S::WR + part.j * S::WR + wr;
        const bool store_rows = a.weights && part.s == 0 && wt == 0 && row0 + 32 * wr < all;

        f32x16_t acc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[i][j] = 0.0f;
        float ref = kNone, l = 0.0f, lost = 0.0f;
        uint4 q[C::QPLANES][8];

        // Weights 2^(logit - ref) of 32 tokens from their products, as operands of the
        // second product: lane's own row, tokens 8 (i / 4) + 4 half + i % 4; and their
        // sum.  They are kept below fp16's largest number: ref moves where one would
        // pass it, and starts so that the first tile's largest is 2^kBase.
        auto soft = [&](const f32x16_t& s, float f, auto& out) {
            float p[16], sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) p[i] = exp2_fast(fmaf(s[i], f, -ref));
            out.pack(p);
            if constexpr (std::decay_t<decltype(out)>::SUM) {
                sum = out.sum();
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) sum += p[i];
            }
            return sum;
        };
        auto settle = [&](const f32x16_t& s, float f, auto& out, float sum) {
            if (__ballot(!(sum < kFull)) != 0) {
                float mx = -INFINITY;
#pragma unroll
                for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[i] * f);
                mx = fmaxf(mx, lane_xor<32>(mx));
                const float to = fmaxf(mx - kBase, ref), g = exp2_fast(ref - to);
                l *= g;
                lost *= g;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 16; ++j) acc[i][j] *= g;
                ref = to;
                sum = soft(s, f, out);
            }
            if constexpr (EXACT) {  // (what a tile's sum loses goes to the next)
                const float some = sum - lost, all_of = l + some;
                lost = (all_of - l) - some;
                l = all_of;
            } else {
                l += sum;
            }
        };
        // A wave's one or two 32-token parts of a tile: the vector work of one beside the
        // matrix products of the other.
        auto fold_tile = [&](auto weights_of, float f, auto&& qk, auto&& mask, auto&& pv) {
            decltype(weights_of) p0, p1;
            f32x16_t s0 = qk(wt);
            mask(wt, s0);
            if constexpr (S::SUB / S::WT == 2) {
                f32x16_t s1 = qk(1);
                const float sum0 = soft(s0, f, p0);
                interleave<std::decay_t<decltype(p0)>::QK, 4, 2>();
                settle(s0, f, p0, sum0);
                mask(1, s1);
                pv(0, p0);
                const float sum1 = soft(s1, f, p1);
                interleave<std::decay_t<decltype(p0)>::PV, 4, 2>();
                settle(s1, f, p1, sum1);
                pv(1, p1);
            } else {
                settle(s0, f, p0, soft(s0, f, p0));
                pv(wt, p0);
            }
        };

        __syncthreads();  // nothing reads the last part's LDS any more
        // ---- cached tokens
        if (part.x0 < cached_tiles) {
            // codes and scales on their way (with roles, of keys or of values)
            constexpr int SETS = S::ROLES ? 1 : 2, VALS = SETS - 1;
            uint32_t x[S::PER][SETS][4], xs[S::PER][SETS][4];
            int left[S::PER];  // of a quad's four tokens, those that are there
            // (a tile's page entries are on their way while the one before is loaded)
            int32_t entry[S::PER];
            auto find = [&](int tile) {
#pragma unroll
                for (int p = 0; p < S::PER; ++p) {
                    const int unit = tid - (vals && S::ROLES ? VALUES_FROM : 0) + p * S::THREADS;
                    const int t = tile * S::TILE + unit / 16 * 4;  // the quad of both
                    entry[p] = t < count ? c.table[b * c.width + (t >> c.page_log2)] : -1;
                }
            };
            auto load = [&](int tile) {
#pragma unroll
                for (int p = 0; p < S::PER; ++p) {
                    const int unit = tid - (vals && S::ROLES ? VALUES_FROM : 0) + p * S::THREADS;
                    const int t = tile * S::TILE + unit / 16 * 4;
                    const bool there = static_cast<uint32_t>(entry[p]) < static_cast<uint32_t>(c.pages);
                    const int64_t at = (there ? entry[p] : 0) * per_page + head_row + (t & in_page);
                    const char* const code = c.codes + at * kCodeRow;
                    const uint32_t* const sc = c.scales + at * (2 * R);
                    left[p] = there ? count - t : 0;
                    if (keys) {
                        const int quarter = unit % 4, k = unit / 4 % 4;
                        const uint4 w = *reinterpret_cast<const uint4*>(code + k * kCodeRow + 16 * quarter);
                        x[p][0][0] = w.x;
                        x[p][0][1] = w.y;
                        x[p][0][2] = w.z;
                        x[p][0][3] = w.w;
                        if constexpr (R == 8) {
                            xs[p][0][0] = sc[k * 2 * R + 2 * quarter];
                            xs[p][0][1] = sc[k * 2 * R + 2 * quarter + 1];
                        } else {
                            xs[p][0][0] = sc[k * 2 * R + (R == 4 ? quarter : quarter / 2)];
                        }
                    }
                    if (vals) {
                        const int dw = unit % 16;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            x[p][VALS][j] = *reinterpret_cast<const uint32_t*>(code + 4 * dw + (j * kCodeRow + 64));
                            xs[p][VALS][j] = sc[8 * dw / G + (j * 2 * R + R)];
                        }
                    }
                }
            };
            uint4 ql[LOWS];
            float factor;
            {
                find(part.x0);
                Raw8<T> raw[8];
                const T* const q_row = query(own_row());
#pragma unroll
                for (int s = 0; s < 8; ++s) raw[s].load(q_row + 8 * s);
                load(part.x0);
                find(part.x0 + 1);
                float top = 0.0f;
#pragma unroll
                for (int s = 0; s < 8; ++s)
#pragma unroll
                    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(raw[s].get(i)));
                top = fmaxf(top, lane_xor<32>(top));
                const int e = static_cast<int>((__float_as_uint(top) >> 23) & 0xffu) - 127;
                factor = ldexpf(kScaleHigh, e + 1 - QTOP);
                float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // of this half's scale groups
#pragma unroll
                for (int s = 0; s < 8; ++s) {
                    float x[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        x[i] = ldexpf(raw[s].get(i), QTOP - 1 - e);
                        sums[8 * s / G] += x[i];
                    }
                    uint32_t w[4], rest[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        w[j] = pack_half2(x[j], x[j + 4]);
                        rest[j] = pack_half2(x[j] - static_cast<float>(as_half2(w[j])[0]),
                                             x[j + 4] - static_cast<float>(as_half2(w[j])[1]));
                    }
                    q[0][s] = make_uint4(w[0], w[1], w[2], w[3]);
                    if constexpr (C::QT == 2) q[1][s] = make_uint4(rest[0], rest[1], rest[2], rest[3]);
                }
                if constexpr (EXACT) {
                    // sums of the queries, for the scales' low and 8 delta (what codes lack in c - 8)
                    float qs[8];
#pragma unroll
                    for (int g = 0; g < 8; ++g) qs[g] = 0.0f;
#pragma unroll
                    for (int g = 0; g < R / 2; ++g) {
                        const float other = lane_xor<32>(sums[g]);
                        qs[g] = half == 0 ? sums[g] : other;
                        qs[R / 2 + g] = half == 0 ? other : sums[g];
                    }
#pragma unroll
                    for (int n = 0; n < LOWS; ++n) {
                        uint32_t w[4];
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const float term = half == 0 ? qs[4 * n + g] : 8.0f * qs[4 * n + g];
                            const float high = static_cast<float>(static_cast<_Float16>(term));
                            w[g] = pack_half2(high, term - high);
                        }
                        ql[n] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
                if (store_rows) {
                    if (half == 0) a.factors[row_tile * 32 + col] = factor;
#pragma unroll
                    for (int n = 0; n < C::QT; ++n)
#pragma unroll
                        for (int s = 0; s < 8; ++s) a.queries[(row_tile * C::STORED + 8 * n + s) * kWave + lane] = q[n][s];
                    if constexpr (EXACT)
#pragma unroll
                        for (int n = 0; n < LOWS; ++n)
                            a.queries[(row_tile * C::STORED + 8 * (C::QT + C::QPLANES) + n) * kWave + lane] = ql[n];
                }
            }
            auto stage = [&](int buf) {
                unsigned char* const s_k = s_mem + buf * BUF;
                unsigned char* const s_v = s_k + C::KT * PLANE;
                bool any = false;
#pragma unroll
                for (int p = 0; p < S::PER; ++p) {
                    const int unit = tid - (vals && S::ROLES ? VALUES_FROM : 0) + p * S::THREADS;
                    if (__ballot(left[p] < 4) != 0) {
                        // what lies behind the last token, or in no page, may be anything
                        any = true;
                        if (keys) {
                            const int rare = (wave * kWave + fresh_lane() + p * S::THREADS);
                            const bool there = rare / 4 % 4 < left[p];
                            if (!there) xs[p][0][0] = xs[p][0][1] = 0u;
                            if (rare % 4 == 0) s_bias[buf][rare / 4] = there ? 0.0f : 1.0f;
                        }
                        if (vals) {
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (j >= left[p]) xs[p][VALS][j] = 0u;
                        }
                    } else if (keys) {
                        const int rare = (wave * kWave + fresh_lane() + p * S::THREADS);
                        if (rare % 4 == 0) s_bias[buf][rare / 4] = 0.0f;
                    }
                    if (keys) {
                        const int token = unit / 4, quarter = unit % 4;
                        const uint32_t (&w)[4] = x[p][0];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t sc = xs[p][0][R == 8 ? e / 2 : 0];
                            const half2_t delta = as_half2(high_halves(sc, sc));
                            if constexpr (EXACT) {
                                const half2_t top7 = as_half2(__builtin_bit_cast(uint32_t, delta) & 0xfff0fff0u);
                                const half2_t low4 = delta - top7;
                                half2_t code[4];
                                centred_pairs(bits, w[e], code);
                                uint32_t hi[4], lo[4];
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    hi[i] = __builtin_bit_cast(uint32_t, code[i] * top7);
                                    lo[i] = __builtin_bit_cast(uint32_t, code[i] * low4);
                                }
                                *key_at(s_k, unit, e) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                                *key_at(s_k + PLANE, unit, e) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                            } else {
                                uint32_t x[4];
                                dequantise_pairs(bits, w[e], delta, as_half2(low_halves(sc, sc)), x);
                                *key_at(s_k, unit, e) = make_uint4(x[0], x[1], x[2], x[3]);
                            }
                        }
                        if constexpr (EXACT) {
                            if constexpr (R == 8) {
                                s_scale[buf][token][2 * quarter] = xs[p][0][0];
                                s_scale[buf][token][2 * quarter + 1] = xs[p][0][1];
                            } else if (R == 4 || quarter % 2 == 0) {
                                s_scale[buf][token][R == 4 ? quarter : quarter / 2] = xs[p][0][0];
                            }
                        }
                    }
                    if (vals) {
                        int place = value_at(unit);
                        asm volatile("" : "+v"(place));  // (its eight forms need no registers between tiles)
                        uint32_t out[8][2], low[8][2];  // [dim][token pair]
#pragma unroll
                        for (int t2 = 0; t2 < 2; ++t2) {
                            const uint32_t v0 = x[p][VALS][2 * t2], v1 = x[p][VALS][2 * t2 + 1];
                            const half2_t delta = as_half2(high_halves(xs[p][VALS][2 * t2], xs[p][VALS][2 * t2 + 1]));
                            const half2_t base = as_half2(low_halves(xs[p][VALS][2 * t2], xs[p][VALS][2 * t2 + 1]));
#pragma unroll
                            for (int hw = 0; hw < 2; ++hw) {
                                const uint32_t w = hw ? high_halves(v0, v1) : low_halves(v0, v1);
                                if constexpr (C::VT == 1) {
                                    uint32_t x[4];
                                    dequantise_pairs(bits, w, delta, base, x);
#pragma unroll
                                    for (int i = 0; i < 4; ++i) out[4 * hw + i][t2] = x[i];
                                } else {
                                    // low + code * delta to 22 bits
                                    half2_t code[4];
                                    code_pairs(bits, w, code);
#pragma unroll
                                    for (int i = 0; i < 4; ++i) {
                                        float y[2], rest[2];
#pragma unroll
                                        for (int k = 0; k < 2; ++k) {
                                            y[k] = fmaf(static_cast<float>(code[i][k]), static_cast<float>(delta[k]),
                                                        static_cast<float>(base[k]));
                                            rest[k] = y[k] - static_cast<float>(static_cast<_Float16>(y[k]));
                                        }
                                        out[4 * hw + i][t2] = pack_half2(y[0], y[1]);
                                        low[4 * hw + i][t2] = pack_half2(rest[0], rest[1]);
                                    }
                                }
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            *value_dim(s_v, place, e) = make_uint2(out[e][0], out[e][1]);
                            if constexpr (C::VT == 2) *value_dim(s_v + PLANE, place, e) = make_uint2(low[e][0], low[e][1]);
                        }
                    }
                }
                if (lane == 0) s_ragged[buf][wave] = any ? 1 : 0;
            };
            auto fold = [&](int buf) {
                const unsigned char* const s_k = s_mem + buf * BUF;
                const unsigned char* const s_v = s_k + C::KT * PLANE;
                int flags = 0;
#pragma unroll
                for (int i = 0; i < S::W; ++i) flags |= s_ragged[buf][i];
                const bool ragged = __builtin_amdgcn_readfirstlane(flags) != 0;
                auto qk = [&](int u) {
                    f32x16_t s;
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] = 0.0f;
                    if constexpr (EXACT) {
                        const uint32_t pick = half == 0 ? 0x01000100u : 0x03020302u;
#pragma unroll
                        for (int n = 0; n < LOWS; ++n) {
                            uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                            for (int g = 0; g < 4 && g < R; ++g) {
                                const uint32_t sc = s_scale[buf][32 * u + col][4 * n + g];
                                w[g] = __builtin_amdgcn_perm(sc, sc, pick);
                            }
                            s = mfma_h(make_uint4(w[0], w[1], w[2], w[3]), ql[n], s);
                        }
                    }
#pragma unroll
                    for (int kt = C::KT - 1; kt >= 0; --kt)
                        products([&](int st) { return s_k + kt * PLANE + (u * 8 + st) * kFrag + lane * 16; },
                                 [&](int st, const uint4& k) {
#pragma unroll
                                     for (int qt = C::QT - 1; qt >= 0; --qt) s = mfma_h(k, q[qt][st], s);
                                 });
                    return s;
                };
                auto mask = [&](int u, f32x16_t& s) {
                    if (ragged) {
                        const float* const bias = &s_bias[buf][32 * u + fresh_lane() / 32 * 4];
#pragma unroll
                        for (int i = 0; i < 16; ++i) s[i] = bias[8 * (i / 4) + i % 4] != 0.0f ? -INFINITY : s[i];
                    }
                };
                auto pv = [&](int u, const HalfWeights<C::CT, C::CT == 1 && !EXACT, C::QT * C::KT>& p) {
#pragma unroll
                    for (int vt = 0; vt < C::VT; ++vt)
                        products(
                            [&](int n) { return s_v + vt * PLANE + (u * 8 + n) * kFrag + value_slot(lane, n % 4); },
                            [&](int n, const uint4& v) {
#pragma unroll
                                for (int pt = 0; pt < C::CT - vt; ++pt) acc[n % 4] = mfma_h(v, p.at[pt][n / 4], acc[n % 4]);
                            });
                };
                fold_tile(HalfWeights<C::CT, C::CT == 1 && !EXACT, C::QT * C::KT>{}, factor, qk, mask, pv);
            };
            const int x1 = min(part.x1, cached_tiles);
            if constexpr (BUFS == 2) {
                stage(0);
                load(part.x0 + 1);
                find(part.x0 + 2);
                __syncthreads();
                for (int x = part.x0; x < x1; ++x) {
                    const int buf = (x - part.x0) & 1;
                    // (behind the part's last tile: what nothing reads)
                    fold(buf);
                    stage(buf ^ 1);
                    load(x + 2);
                    find(x + 3);
                    __syncthreads();
                }
            } else {
                for (int x = part.x0; x < x1; ++x) {
                    stage(0);
                    if (x + 1 < x1) load(x + 1);
                    find(x + 2);
                    __syncthreads();
                    fold(0);
                    __syncthreads();
                }
            }
        }

        // ---- the new tokens, in their own type (fp32: three bf16 terms)
        if (store_rows || part.x1 > cached_tiles) {
            Raw8<T> raw[8];
            const T* const q_row = query(own_row());
#pragma unroll
            for (int s = 0; s < 8; ++s) raw[s].load(q_row + 8 * s);
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                if constexpr (C::F32) {
                    uint4 t[3];
                    bf16_operand<3>([&](int i) { return raw[s].get(i); }, t);
#pragma unroll
                    for (int n = 0; n < 3; ++n) q[n][s] = t[n];
                } else {
                    q[0][s] = raw[s].u;
                }
            }
            if (store_rows) {
#pragma unroll
                for (int n = 0; n < C::QPLANES; ++n)
#pragma unroll
                    for (int s = 0; s < 8; ++s)
                        a.queries[(row_tile * C::STORED + 8 * (C::QT + n) + s) * kWave + lane] = q[n][s];
            }
        }
        if (part.x1 > cached_tiles) {
            const int t_row = own_row().t;
            const T* const k_head = static_cast<const T*>(a.k) + b * a.k_bs + h * a.k_hs;
            const T* const v_head = static_cast<const T*>(a.v) + b * a.v_bs + h * a.v_hs;
            auto mfma_t = [&](const uint4& x, const uint4& y, f32x16_t z) {
                if constexpr (C::F16) return mfma_h(x, y, z);
                else return mfma_b(x, y, z);
            };
            constexpr int SETS = S::ROLES ? 1 : 2, VALS = SETS - 1;
            Raw8<T> x[S::PER][SETS][4];
            auto load = [&](int tile) {
#pragma unroll
                for (int p = 0; p < S::PER; ++p) {
                    const int unit = tid - (vals && S::ROLES ? VALUES_FROM : 0) + p * S::THREADS;
                    if (keys) {
                        const int t = tile * S::TILE + unit / 4;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            x[p][0][e].load(k_head + static_cast<int64_t>(min(t, rows - 1)) * a.k_ts + 8 * (unit % 4) + 32 * e);
                        }
                    }
                    if (vals) {
                        const int t = tile * S::TILE + unit / 16 * 4;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            x[p][VALS][j].load(v_head + static_cast<int64_t>(min(t + j, rows - 1)) * a.v_ts + 8 * (unit % 16));
                        }
                    }
                }
            };
            auto stage = [&](int tile, int buf) {
                unsigned char* const s_k = s_mem + buf * BUF;
                unsigned char* const s_v = s_k + C::NT * PLANE;
                bool odd = false, odd_key = false;
#pragma unroll
                for (int p = 0; p < S::PER; ++p) {
                    const int unit = tid - (vals && S::ROLES ? VALUES_FROM : 0) + p * S::THREADS;
                    if ((tile + 1) * S::TILE > rows) {  // what lies behind the chunk's last token may be anything
                        if (keys && tile * S::TILE + unit / 4 >= rows) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[p][0][e].zero();
                        }
                        if (vals) {
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (tile * S::TILE + unit / 16 * 4 + j >= rows) x[p][VALS][j].zero();
                        }
                    }
                    if (keys) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if constexpr (C::F32) {
                                odd_key = odd_key || odd_values<T>(x[p][0][e]);
                                uint4 t[3];
                                bf16_operand<3>([&](int i) { return x[p][0][e].get(i); }, t);
#pragma unroll
                                for (int n = 0; n < 3; ++n) *new_key_at(s_k + n * PLANE, unit, e) = t[n];
                            } else {
                                *new_key_at(s_k, unit, e) = x[p][0][e].u;
                            }
                        }
                    }
                    if (vals) {
                        int place = value_at(unit);
                        asm volatile("" : "+v"(place));
                        bool mine = false;
#pragma unroll
                        for (int j = 0; j < 4; ++j) mine = mine || odd_values<T>(x[p][VALS][j]);
                        odd = odd || mine;
                        if (__ballot(mine) != 0) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) clear_odd<T>(x[p][VALS][j]);
                        }
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            if constexpr (C::F32) {
                                uint32_t t[2][3];
                                bf16_terms<3>(x[p][VALS][0].get(e), x[p][VALS][1].get(e), t[0]);
                                bf16_terms<3>(x[p][VALS][2].get(e), x[p][VALS][3].get(e), t[1]);
#pragma unroll
                                for (int n = 0; n < 3; ++n) *value_dim(s_v + n * PLANE, place, e) = make_uint2(t[0][n], t[1][n]);
                            } else {
                                uint32_t w[4];
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    const uint4& y = x[p][VALS][j].u;
                                    w[j] = e < 2 ? y.x : e < 4 ? y.y : e < 6 ? y.z : y.w;
                                }
                                *value_dim(s_v, place, e) = e & 1 ? make_uint2(high_halves(w[0], w[1]), high_halves(w[2], w[3]))
                                                                : make_uint2(low_halves(w[0], w[1]), low_halves(w[2], w[3]));
                            }
                        }
                    }
                }
                const bool any = __ballot(odd) != 0, any_key = __ballot(odd_key) != 0;
                if (lane == 0) {
                    s_ragged[buf][wave] = any ? 1 : 0;
                    s_odd_keys[buf][wave] = any_key ? 1 : 0;
                }
            };
            // Infinite and NaN values: times a weight of zero they would reach rows that do
            // not see their token, so the products take them as zero, and their dims of the
            // rows that do see it get them here.
            auto add_odd = [&](int first, int last) {
#pragma unroll 1
                for (int t = first; t < min(last, rows); ++t) {
                    const T* v_row = v_head + static_cast<int64_t>(t) * a.v_ts + 64 * half;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        Raw8<T> v;
                        v.load(v_row + 8 * i);
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            acc[i / 2][8 * (i & 1) + j] += t <= t_row && is_odd(v.get(j)) ? v.get(j) : 0.0f;
                    }
                }
            };
            // Logits of fp32 keys with an infinite element: its product with the lower
            // terms of a query is no part of the sum.
            auto odd_logits = [&](int first, f32x16_t& s) {
#pragma unroll 1
                for (int t = 0; t < min(32, rows - first); ++t) {
                    const T* k_row = k_head + static_cast<int64_t>(first + t) * a.k_ts + 64 * half;
                    const T* const q_row = query(own_row());
                    float dot = 0.0f;
                    bool odd = false;
#pragma unroll 1
                    for (int i = 0; i < 8; ++i) {
                        Raw8<T> k, x;
                        k.load(k_row + 8 * i);
                        x.load(q_row + 8 * i);
                        odd = odd || odd_values<T>(k);
#pragma unroll
                        for (int j = 0; j < 8; ++j) dot = fmaf(x.get(j), k.get(j), dot);
                    }
                    if (__ballot(odd) == 0) continue;
                    dot += lane_xor<32>(dot);
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] = 8 * (i / 4) + 4 * half + i % 4 == t ? dot : s[i];
                }
            };
            // (of the wave's rows)
            const int t_first = __builtin_amdgcn_readfirstlane(t_row), t_last = __builtin_amdgcn_readlane(t_row, 31);
            using Weights = std::conditional_t<C::F16, HalfWeights<C::PT, false, 1>,
                                               Bf16Weights<C::PT, C::PT == 1 && !EXACT, 1>>;
            bool odd = false;
            auto fold = [&](int tile, int buf) {
                const unsigned char* const s_k = s_mem + buf * BUF;
                const unsigned char* const s_v = s_k + C::NT * PLANE;
                int flags = 0, key_flags = 0;
#pragma unroll
                for (int i = 0; i < S::W; ++i) {
                    flags |= s_ragged[buf][i];
                    if constexpr (C::F32) key_flags |= s_odd_keys[buf][i];
                }
                odd = odd || __builtin_amdgcn_readfirstlane(flags) != 0;
                const bool odd_keys = __builtin_amdgcn_readfirstlane(key_flags) != 0;
                auto qk = [&](int u) {
                    f32x16_t s;
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
                    for (int n = C::NT - 1; n >= 0; --n)
                        products([&](int st) { return s_k + n * PLANE + (u * 8 + st) * kFrag + lane * 16; },
                                 [&](int st, const uint4& k) {
#pragma unroll
                                     for (int m = C::NT - 1 - n; m >= 0; --m) s = mfma_t(k, q[m][st], s);
                                 });
                    return s;
                };
                auto mask = [&](int u, f32x16_t& s) {
                    const int first = tile * S::TILE + 32 * u, t0 = first + 4 * half;
                    if constexpr (C::F32)
                        if (odd_keys) odd_logits(first, s);
                    // (tokens behind the chunk's last are ahead of every row)
                    if (first + 31 > t_first) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) s[i] = t0 + 8 * (i / 4) + i % 4 <= t_row ? s[i] : -INFINITY;
                    }
                };
                auto pv = [&](int u, const Weights& p) {
#pragma unroll
                    for (int n = 0; n < C::NT; ++n)
                        products(
                            [&](int k) { return s_v + n * PLANE + (u * 8 + k) * kFrag + value_slot(lane, k % 4); },
                            [&](int k, const uint4& v) {
#pragma unroll
                                for (int m = 0; m < C::PT - n; ++m) acc[k % 4] = mfma_t(v, p.at[m][k / 4], acc[k % 4]);
                            });
                };
                // (a wave's rows may lie before its part of the tile)
                if (tile * S::TILE + 32 * wt <= t_last) fold_tile(Weights{}, kScaleHigh, qk, mask, pv);
            };
            const int x0 = max(part.x0 - cached_tiles, 0), x1 = part.x1 - cached_tiles;
            load(x0);
            if constexpr (BUFS == 2) {
                stage(x0, 0);
                load(x0 + 1);
                __syncthreads();
                for (int x = x0; x < x1; ++x) {
                    const int buf = (x - x0) & 1;
                    fold(x, buf);
                    stage(x + 1, buf ^ 1);
                    load(x + 2);
                    __syncthreads();
                }
            } else {
                for (int x = x0; x < x1; ++x) {
                    stage(x, 0);
                    if (x + 1 < x1) load(x + 1);
                    __syncthreads();
                    fold(x, 0);
                    __syncthreads();
                }
            }
            // (by one of the waves that share a tile's tokens)
            if (odd && wt == 0) add_odd(x0 * S::TILE, x1 * S::TILE);
        }

        l += lane_xor<32>(l);
        // Waves that shared the tokens: each takes D of the four tiles of dims from all of
        // them.
        constexpr int D = 4 / S::WT;
        if constexpr (S::WT > 1) {
            float* const states = reinterpret_cast<float*>(s_mem);
            float* const sums = states + S::W * 4096;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                *reinterpret_cast<float4*>(states + (wave * 16 + i) * 256 + lane * 4) =
                    make_float4(acc[i / 4][4 * (i % 4)], acc[i / 4][4 * (i % 4) + 1], acc[i / 4][4 * (i % 4) + 2],
                                acc[i / 4][4 * (i % 4) + 3]);
            if (half == 0) {
                sums[wave * 64 + col] = ref;
                sums[wave * 64 + 32 + col] = l;
            }
            __syncthreads();
            float f[S::WT];
#pragma unroll
            for (int n = 0; n < S::WT; ++n) f[n] = sums[(n * S::WR + wr) * 64 + col];
            ref = f[0];
#pragma unroll
            for (int n = 1; n < S::WT; ++n) ref = fmaxf(ref, f[n]);
            l = 0.0f;
#pragma unroll
            for (int n = 0; n < S::WT; ++n) {
                f[n] = exp2_fast(f[n] - ref);
                l = fmaf(f[n], sums[(n * S::WR + wr) * 64 + 32 + col], l);
            }
#pragma unroll
            for (int i = 0; i < 4 * D; ++i) {
                float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int n = 0; n < S::WT; ++n) {
                    const float4 y = *reinterpret_cast<const float4*>(
                        states + ((n * S::WR + wr) * 16 + wt * 4 * D + i) * 256 + lane * 4);
                    x.x = fmaf(f[n], y.x, x.x);
                    x.y = fmaf(f[n], y.y, x.y);
                    x.z = fmaf(f[n], y.z, x.z);
                    x.w = fmaf(f[n], y.w, x.w);
                }
                const int j = 4 * (i % 4);
                acc[i / 4][j] = x.x;
                acc[i / 4][j + 1] = x.y;
                acc[i / 4][j + 2] = x.z;
                acc[i / 4][j + 3] = x.w;
            }
        }
        if (part.n == 1) {
            const Row r = own_row();
            if (r.live) {
                T* const out = static_cast<T*>(a.out) + b * a.o_bs + r.head * a.o_hs + static_cast<int64_t>(r.t) * a.o_ts +
                               64 * half + 16 * D * wt;
                const float f = 1.0f / l;
#pragma unroll
                for (int i = 0; i < D; ++i) store16<T>(out + 16 * i, acc[i], f);
            }
            // (rows past the last one weigh nothing)
            if (store_rows && half == 0) a.sums[row_tile * 32 + col] = row_sums(ref, l, r.live);
        } else {
            const int64_t place = 2 * static_cast<int64_t>(w_id) + (part.s == 0 ? 1 : 0);
            float* const state = a.partials + (place * c.kv_heads + h) * S::STATE + wr * (4096 + 64);
#pragma unroll
            for (int i = 0; i < 4 * D; ++i)
                *reinterpret_cast<float4*>(state + ((4 * D * wt + i) * kWave + lane) * 4) = make_float4(
                    acc[i / 4][4 * (i % 4)], acc[i / 4][4 * (i % 4) + 1], acc[i / 4][4 * (i % 4) + 2],
                    acc[i / 4][4 * (i % 4) + 3]);
            if (half == 0 && wt == 0) {
                state[4096 + col] = ref;
                state[4096 + 32 + col] = l;
            }
        }
        if (h == 0 && part.s == 0 && tid == 0) a.parts[b * a.row_blocks + part.j] = make_int2(part.first, part.n);
    }
}

// Blocks of rows in several parts: a wave for 4 N of each half's 64 dims of 32 rows.  A
// launch of its own: the parts' states are up to 68 MB (34 MB where each workgroup has
// one, 133 KB), which one workgroup a block would read too slowly.  Bound by its chain of
// reads (sizes, part, states), 5 us, and for 256 parts of 256 rows by the states, 14 us.
// Few tiles of rows have many parts each: then
// a wave has 4 dims and 16 parts on their way (64 tiles of 8 to 13 parts 9.5 us, with 16
// dims 11.4; of 32 parts 14.2 and 17.7; 288 tiles 6.2 both ways).
constexpr int kFewTiles = 256;
template <typename T, typename S, int N>
__global__ __launch_bounds__(256) void chunk_merge_kernel(PagedChunk a, PagedView c, int64_t max_tokens) {
    constexpr int PIECES = 4 / N;
    const int h = blockIdx.y, b = blockIdx.z;
    const int piece = blockIdx.x % PIECES, block = blockIdx.x / PIECES;
    const int j = block / S::WR, wr = block % S::WR;
    const int lane = threadIdx.x & (kWave - 1), col = lane & 31, half = lane >> 5;
    const int i = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int group = a.q_heads / c.kv_heads;
    const ChunkSizes z(a, c, max_tokens, b);
    const int64_t all = static_cast<int64_t>(z.rows) * group, row = static_cast<int64_t>(j) * S::ROWS + 32 * wr + col;
    if (row - col >= all) return;
    const int2 parts = a.parts[b * a.row_blocks + j];
    if (parts.y <= 1) return;
    auto state = [&](int s) {
        const int64_t place = 2 * static_cast<int64_t>(parts.x + s) + (s == 0 ? 1 : 0);
        return a.partials + (place * c.kv_heads + h) * S::STATE + wr * (4096 + 64);
    };
    float m = -INFINITY, l = 0.0f;
    float4 acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    // (parts on their way at once: four, where there are more eight of 16 dims or 16 of 4)
    auto fold = [&](auto ahead, int s0) {
        constexpr int AHEAD = decltype(ahead)::value;
        float4 y[AHEAD][N];
        float pm[AHEAD], pl[AHEAD], mx = m;
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) {
            const float* p = state(min(s0 + n, parts.y - 1));
            pm[n] = p[4096 + col];
            pl[n] = p[4096 + 32 + col];
#pragma unroll
            for (int k = 0; k < N; ++k)
                y[n][k] = *reinterpret_cast<const float4*>(p + ((4 * i + N * piece + k) * kWave + lane) * 4);
        }
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) mx = fmaxf(mx, pm[n]);
        const float g = m == -INFINITY ? 0.0f : exp2_fast(m - mx);
        l *= g;
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] = make_float4(acc[k].x * g, acc[k].y * g, acc[k].z * g, acc[k].w * g);
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) {
            if (s0 + n >= parts.y) break;
            const float f = exp2_fast(pm[n] - mx);
            l = fmaf(f, pl[n], l);
#pragma unroll
            for (int k = 0; k < N; ++k) {
                acc[k].x = fmaf(f, y[n][k].x, acc[k].x);
                acc[k].y = fmaf(f, y[n][k].y, acc[k].y);
                acc[k].z = fmaf(f, y[n][k].z, acc[k].z);
                acc[k].w = fmaf(f, y[n][k].w, acc[k].w);
            }
        }
        m = mx;
    };
    constexpr int MOST = N == 4 ? 8 : 16;
    if (parts.y <= 4)
        fold(std::integral_constant<int, 4>{}, 0);
    else
        for (int s0 = 0; s0 < parts.y; s0 += MOST) fold(std::integral_constant<int, MOST>{}, s0);
    if (row < all) {
        const int t_row = static_cast<int>(row / group);
        const int head = h * group + static_cast<int>(row - static_cast<int64_t>(t_row) * group);
        T* const out = static_cast<T*>(a.out) + b * a.o_bs + head * a.o_hs + static_cast<int64_t>(t_row) * a.o_ts;
        store4s<T, N>(out + 64 * half + 16 * i + 4 * N * piece, acc, 1.0f / l);
    }
    if (a.weights && i == 0 && half == 0 && piece == 0) {
        const int64_t row_tile = (static_cast<int64_t>(b) * c.kv_heads + h) * a.row_blocks * S::WR + j * S::WR + wr;
        a.sums[row_tile * 32 + col] = row_sums(m, l, row < all);
    }
}

// The attention weights of N times 32 tokens of a KV head a wave, from the logits once
// more and the rows' sums: keys stay in registers, as the first pass has them, and
// every row's operands pass once.  Rows stand in the products' rows, so that a token's
// weights lie in one lane's registers and that of the other half: no atomics, and equal
// bits from call to call.  Bound by the matrix instructions and the exponentials beside
// them: up to 4092 rows of each of two fp16 sequences up to 9023 tokens, 294 us (with sums
// not compensated 249, then 282 without the products of one part beside the weights of the
// other, and 328 with operands through LDS for four waves in the place of each wave's own
// reads); 16 decode steps up to 4200 tokens by the keys' dequantisation, 19 us.
template <typename T, int G, int N>
__global__ __launch_bounds__(256, (sizeof(T) == 4 ? 1 : 2)) void chunk_weights_kernel(PagedChunk a, PagedView c,
                                                                                     int64_t max_tokens) {
    using C = ChunkTypes<T, true>;
    constexpr int R = 128 / G, LOWS = R == 8 ? 2 : 1, SPAN = 32 * N;
    const int b = blockIdx.z, h = blockIdx.y;
    const int lane = threadIdx.x & (kWave - 1), col = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int group = div_nonneg(a.q_heads, c.kv_heads);
    const ChunkSizes z(a, c, max_tokens, b);
    const int rows = z.rows, count = z.count;
    const int cached_spans = (count + SPAN - 1) / SPAN, span = blockIdx.x * 4 + wave;
    const bool cached = span < cached_spans;
    const int t0 = SPAN * (cached ? span : span - cached_spans);
    if (rows == 0 || (!cached && t0 >= rows)) return;
    const int all = rows * group;
    const int64_t base = (static_cast<int64_t>(b) * c.kv_heads + h) * (a.row_blocks * a.row_waves);
    float sum[N], lost[N];  // (thousands of rows: what a tile's sum loses goes to the next)
    bool there[N];
#pragma unroll
    for (int n = 0; n < N; ++n) sum[n] = lost[n] = 0.0f;
    // a tile of 32 rows: its logits' products by `logits`, a row's weight added by `add_one`
    auto tile = [&](int r0, auto&& logits, auto&& add_one, bool scaled) {
        const float4* sums = reinterpret_cast<const float4*>(a.sums + (base * 32 + r0) + 4 * half);
        const float4* factors = reinterpret_cast<const float4*>(a.factors + (base * 32 + r0) + 4 * half);
        float4 f[4], x[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i][0] = sums[4 * i];
            x[i][1] = sums[4 * i + 1];
            f[i] = scaled ? factors[2 * i] : make_float4(kScaleHigh, kScaleHigh, kScaleHigh, kScaleHigh);
        }
        auto add = [&](int n, const f32x16_t& s) {
            float some = -lost[n];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = r0 + 8 * i + 4 * half;
                some = add_one(some, n, r, exp2_fast(fmaf(s[4 * i], f[i].x, -x[i][0].x)), x[i][0].y);
                some = add_one(some, n, r + 1, exp2_fast(fmaf(s[4 * i + 1], f[i].y, -x[i][0].z)), x[i][0].w);
                some = add_one(some, n, r + 2, exp2_fast(fmaf(s[4 * i + 2], f[i].z, -x[i][1].x)), x[i][1].y);
                some = add_one(some, n, r + 3, exp2_fast(fmaf(s[4 * i + 3], f[i].w, -x[i][1].z)), x[i][1].w);
            }
            const float all_of = sum[n] + some;
            lost[n] = (all_of - sum[n]) - some;
            sum[n] = all_of;
        };
        f32x16_t s = logits(0);
#pragma unroll
        for (int n = 1; n < N; ++n) {
            __builtin_amdgcn_sched_barrier(0);
            const f32x16_t next = logits(n);
            add(n - 1, s);
#pragma unroll
            for (int i = 0; i < 16; ++i) {  // (a product, and a weight beside it)
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
                __builtin_amdgcn_sched_group_barrier(0x400, 1, 0);
            }
            s = next;
        }
        add(N - 1, s);
    };
    const uint4* const queries = a.queries + base * (C::STORED * kWave) + lane;
    if (cached) {
        const CodeBits bits;
        uint4 k[N][2][8], low[N][LOWS];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int token = t0 + 32 * n + col;
            const int32_t e = token < count ? c.table[b * c.width + (token >> c.page_log2)] : -1;
            there[n] = static_cast<uint32_t>(e) < static_cast<uint32_t>(c.pages);
            const int64_t at = (there[n] ? e : 0) * (static_cast<int64_t>(c.kv_heads) << c.page_log2) +
                               (static_cast<int64_t>(h) << c.page_log2) + (token & ((1 << c.page_log2) - 1));
            const uint4* codes = reinterpret_cast<const uint4*>(c.codes + at * kCodeRow + 32 * half);
            const uint4 w0 = codes[0], w1 = codes[1];
            const uint32_t w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
            uint32_t sc[R];
#pragma unroll
            for (int g = 0; g < R; ++g) sc[g] = c.scales[at * (2 * R) + g];
            const uint32_t pick = half == 0 ? 0x01000100u : 0x03020302u;
#pragma unroll
            for (int m = 0; m < LOWS; ++m) {
                uint32_t x[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                for (int g = 0; g < 4 && g < R; ++g) x[g] = __builtin_amdgcn_perm(sc[4 * m + g], sc[4 * m + g], pick);
                low[n][m] = make_uint4(x[0], x[1], x[2], x[3]);
            }
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                const uint32_t own = half == 0 ? sc[8 * s / G] : sc[R / 2 + 8 * s / G];
                const half2_t delta = as_half2(high_halves(own, own));
                const half2_t top7 = as_half2(__builtin_bit_cast(uint32_t, delta) & 0xfff0fff0u), low4 = delta - top7;
                half2_t code[4];
                centred_pairs(bits, w[s], code);
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    hi[i] = __builtin_bit_cast(uint32_t, code[i] * top7);
                    lo[i] = __builtin_bit_cast(uint32_t, code[i] * low4);
                }
                k[n][0][s] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                k[n][1][s] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
        }
        for (int r0 = 0; r0 < all; r0 += 32) {
            const uint4* q = queries + r0 / 32 * static_cast<int64_t>(C::STORED * kWave);
            uint4 x[C::QT][8], ql[LOWS];
#pragma unroll
            for (int n = 0; n < LOWS; ++n) ql[n] = q[(8 * (C::QT + C::QPLANES) + n) * kWave];
#pragma unroll
            for (int n = 0; n < C::QT; ++n)
#pragma unroll
                for (int s = 0; s < 8; ++s) x[n][s] = q[(8 * n + s) * kWave];
            tile(
                r0,
                [&](int n) {
                    f32x16_t s;
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
                    for (int m = 0; m < LOWS; ++m) s = mfma_h(ql[m], low[n][m], s);
#pragma unroll
                    // (the small products first: the sums round less)
                    for (int kt = 1; kt >= 0; --kt)
#pragma unroll
                        for (int qt = C::QT - 1; qt >= 0; --qt)
#pragma unroll
                            for (int st = 0; st < 8; ++st) s = mfma_h(x[qt][st], k[n][kt][st], s);
                    return s;
                },
                [&](float some, int, int, float p, float g) { return fmaf(p, g, some); }, true);
        }
    } else {
        uint4 k[N][C::NT][8];
        bool odd[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int token = t0 + 32 * n + col;
            there[n] = token < rows;
            odd[n] = false;
            const T* k_row =
                static_cast<const T*>(a.k) + b * a.k_bs + h * a.k_hs + static_cast<int64_t>(min(token, rows - 1)) * a.k_ts;
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                Raw8<T> raw;
                raw.load(k_row + 64 * half + 8 * s);
                if constexpr (C::F32) {
                    odd[n] = odd[n] || odd_values<T>(raw);
                    uint4 t[3];
                    bf16_operand<3>([&](int i) { return raw.get(i); }, t);
#pragma unroll
                    for (int m = 0; m < 3; ++m) k[n][m][s] = t[m];
                } else {
                    k[n][0][s] = raw.u;
                }
            }
            // (the parts of an infinite fp32 key's products are no sum: its logit is minus
            // infinity or makes the row NaN)
            if constexpr (C::F32) odd[n] = odd[n] || lane_xor<32>(odd[n] ? 1.0f : 0.0f) != 0.0f;
        }
        for (int r0 = t0 * group / 32 * 32; r0 < all; r0 += 32) {
            const uint4* q = queries + r0 / 32 * static_cast<int64_t>(C::STORED * kWave) + 8 * C::QT * kWave;
            uint4 x[C::QPLANES][8];
#pragma unroll
            for (int n = 0; n < C::QPLANES; ++n)
#pragma unroll
                for (int s = 0; s < 8; ++s) x[n][s] = q[(8 * n + s) * kWave];
            tile(
                r0,
                [&](int n) {
                    f32x16_t s;
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
                    for (int m = C::NT - 1; m >= 0; --m)
#pragma unroll
                        for (int j = C::NT - 1 - m; j >= 0; --j)
#pragma unroll
                            for (int st = 0; st < 8; ++st) {
                                if constexpr (C::F16) s = mfma_h(x[j][st], k[n][m][st], s);
                                else s = mfma_b(x[j][st], k[n][m][st], s);
                            }
                    return s;
                },
                [&](float some, int n, int r, float p, float g) {
                    p *= g;
                    if (C::F32 && odd[n]) p = g == g ? 0.0f : g;
                    return some + (r >= (t0 + 32 * n + col) * group ? p : 0.0f);
                },
                false);
        }
    }
    // (new tokens stand behind all cached ones, those past max_tokens among them)
    const int64_t first = cached ? 0 : clamp_count(c.counts[b], c.width << c.page_log2);
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const float x = sum[n] + lane_xor<32>(sum[n]);
        const int64_t at = first + t0 + 32 * n + col;
        if (half == 0 && there[n] && at < a.weight_stride)
            a.weights[(static_cast<int64_t>(b) * c.kv_heads + h) * a.weight_stride + at] += x;
    }
}

template <typename T, int G, bool EXACT, typename S>
hipError_t launch_chunk_s(const PagedChunk& a, const PagedView& c, int64_t max_tokens, hipStream_t stream) {
    hipLaunchKernelGGL((paged_chunk_kernel<T, G, EXACT, S>), dim3(static_cast<unsigned>(a.groups * c.kv_heads)),
                       dim3(S::THREADS), 0, stream, a, c, max_tokens, a.groups);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && a.groups > 1) {
        const int64_t tiles = a.row_blocks * S::WR;
        auto launch = [&](auto kernel, int64_t pieces) {
            hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(tiles * pieces), c.kv_heads, c.batch), dim3(256), 0,
                               stream, a, c, max_tokens);
            return hipGetLastError();
        };
        e = tiles * c.kv_heads * c.batch <= kFewTiles ? launch(chunk_merge_kernel<T, S, 1>, 4)
                                                      : launch(chunk_merge_kernel<T, S, 4>, 1);
    }
    return e;
}

template <typename T, int G, bool EXACT>
hipError_t launch_chunk_e(const PagedChunk& a, const PagedView& c, int64_t max_tokens, hipStream_t stream) {
    switch (a.shape) {
        case 1:
            if constexpr (!std::is_same_v<T, float>)
                return launch_chunk_s<T, G, EXACT, ChunkShape<1, 4>>(a, c, max_tokens, stream);
        case 2: return launch_chunk_s<T, G, EXACT, ChunkShape<2, 2>>(a, c, max_tokens, stream);
        case 8:
            if constexpr (!std::is_same_v<T, float>)
                return launch_chunk_s<T, G, EXACT, ChunkShape<8, 1>>(a, c, max_tokens, stream);
        default: return launch_chunk_s<T, G, EXACT, ChunkShape<4, 1>>(a, c, max_tokens, stream);
    }
}

template <typename T, int G>
hipError_t launch_chunk_t(const PagedChunk& a, const PagedView& c, int64_t max_tokens, hipStream_t stream) {
    hipError_t e;
    if constexpr (std::is_same_v<T, bf16_t>) {
        e = a.weights ? launch_chunk_e<T, G, true>(a, c, max_tokens, stream)
                      : launch_chunk_e<T, G, false>(a, c, max_tokens, stream);
    } else {
        e = launch_chunk_e<T, G, true>(a, c, max_tokens, stream);
    }
    if (e != hipSuccess || !a.weights) return e;
    const int64_t most = min(max_tokens, c.width << c.page_log2);
    auto launch = [&](auto kernel, int64_t span) {
        const unsigned blocks = static_cast<unsigned>(((most + span - 1) / span + (a.rows + span - 1) / span + 3) / 4);
        hipLaunchKernelGGL(kernel, dim3(blocks, c.kv_heads, c.batch), dim3(256), 0, stream, a, c, max_tokens);
        return hipGetLastError();
    };
    // Two parts a wave where many rows pass, one where keys are most of the work (us of a
    // call with one and two: 132 rows behind 32703 tokens 120 and 113, 256 139 and 128, 512
    // 244 and 215; 16 sequences of 32 rows behind 4200 92.7 and 93.6, 32 rows behind 32703 64
    // both ways.  Two are ahead below 128 rows too: 64 rows 79.5 and 77.7, 128 99.5 and 94.3.)
    if constexpr (!std::is_same_v<T, float>)
        if (a.rows * (a.q_heads / c.kv_heads) > 128) return launch(chunk_weights_kernel<T, G, 2>, 64);
    return launch(chunk_weights_kernel<T, G, 1>, 32);
}

template <typename T>
hipError_t launch_chunk(const PagedChunk& a, const PagedView& c, int64_t max_tokens, int dim_group, hipStream_t stream) {
    switch (dim_group) {
        case 16: return launch_chunk_t<T, 16>(a, c, max_tokens, stream);
        case 32: return launch_chunk_t<T, 32>(a, c, max_tokens, stream);
        default: return launch_chunk_t<T, 64>(a, c, max_tokens, stream);
    }
}

}  // namespace
}  // namespace popkv
