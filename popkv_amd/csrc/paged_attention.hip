// Decode attention over the paged 4-bit K/V cache: every cached token
// (dense) or a selection of them (indexed), with the current token's K/V, not
// cached yet, folded into the merge at full precision.
//
// Both split a row's tokens among workgroups that each leave an online-softmax
// state (m, l, acc[128]), base-2 exponents; the last workgroup of a row merges
// them in the same launch (the hand-off rule stands in attention_common.h).
#include "attention_common.h"
#include "paged.h"

namespace popkv {
namespace {

constexpr int kState = 128 + 2;
// log2(e) / sqrt(128) as a float and what it leaves: logits reach tens, and
// one float's rounding of the factor would show in fp32 outputs
constexpr double kScale = 1.4426950408889634 * 0.08838834764831845;
constexpr float kScaleHigh = static_cast<float>(kScale);
constexpr float kScaleLow = static_cast<float>(kScale - static_cast<double>(kScaleHigh));
__device__ __forceinline__ float scaled_logit(float dot) { return fmaf(dot, kScaleHigh, dot * kScaleLow); }

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The factor that takes a state (m, l) to the maximum mx.  A state that folded
// nothing has l = 0; one whose logits were all NaN keeps its NaN.
__device__ __forceinline__ float state_weight(float m, float l, float mx) {
    return m == -INFINITY && l == 0.0f ? 0.0f : exp2_fast(m - mx);
}

// ---- codes as fp16 ----------------------------------------------------------

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ half2_t as_half2(uint32_t x) { return __builtin_bit_cast(half2_t, x); }
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
    return __builtin_bit_cast(uint32_t, half2_t{static_cast<_Float16>(a), static_cast<_Float16>(b)});
}
__device__ __forceinline__ uint32_t low_halves(uint32_t a, uint32_t b) {  // a.lo, b.lo
    return __builtin_amdgcn_perm(b, a, 0x05040100u);
}
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) {
    return __builtin_amdgcn_perm(b, a, 0x07060302u);
}

// Nibble pairs (0, 4), (1, 5), (2, 6), (3, 7) of w as fp16 1024 + c (first and
// third) and 1024 + 16 c.
// The constants sit in registers (an instruction takes one literal here, and
// with two the compiler makes an "and" and an "or" of it).
struct CodeBits {
    uint32_t even = 0x000f000fu, odd = 0x00f000f0u, bias = 0x64006400u;
    __device__ __forceinline__ CodeBits() {
        asm("" : "+s"(even));
        asm("" : "+s"(odd));
        asm("" : "+v"(bias));
    }
};
__device__ __forceinline__ void biased_pairs(const CodeBits& k, uint32_t w, uint32_t (&out)[4]) {
    const uint32_t x = w >> 8;
    out[0] = (w & k.even) | k.bias;
    out[1] = (w & k.odd) | k.bias;
    out[2] = (x & k.even) | k.bias;
    out[3] = (x & k.odd) | k.bias;
}

// ---- the VALU fold ----------------------------------------------------------

// Eight lanes a token, sixteen dims each (one scale group at G = 16, 32, 64).
struct Row4 {
    uint2 k, v;
    uint32_t ks, vs;
};

template <int QC>
struct FoldState {
    float m[QC], l[QC], acc[QC][16];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int j = 0; j < QC; ++j) {
            m[j] = -INFINITY;
            l[j] = 0.0f;
#pragma unroll
            for (int d = 0; d < 16; ++d) acc[j][d] = 0.0f;
        }
    }
};

// This lane's sixteen values low + c * delta, rounded once to fp32.  (Sums of
// codes with the scales applied after save an fma a value, but delta sum(q c)
// and low sum(q) cancel: fp32 results were twice as far off.)
__device__ __forceinline__ void values16(uint2 w, uint32_t scale, float (&x)[16]) {
    codes8(w.x, x);
    codes8(w.y, x + 8);
    const float low = f16_lo(scale), delta = f16_hi(scale);
#pragma unroll
    for (int d = 0; d < 16; ++d) x[d] = fmaf(x[d], delta, low);
}

// Folds four tokens into the lane octet's state, in fp32.  Dead tokens have
// zero scales (their values count with weight 0, so they must be finite).
template <int QC>
__device__ __forceinline__ void fold4(FoldState<QC>& st, const float (&q)[QC][16], const Row4 (&r)[4],
                                      const bool (&live)[4]) {
    float s[QC][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        float k[16];
        values16(r[t].k, r[t].ks, k);
#pragma unroll
        for (int j = 0; j < QC; ++j) {
            float dot = 0.0f;
#pragma unroll
            for (int d = 0; d < 16; ++d) dot = fmaf(q[j][d], k[d], dot);
            const float x = scaled_logit(row_sum<8>(dot));
            s[j][t] = live[t] ? x : -INFINITY;
        }
    }
    bool moved = false;
    float alpha[QC];
#pragma unroll
    for (int j = 0; j < QC; ++j) {
        const float mn = fmaxf(fmaxf(fmaxf(s[j][0], s[j][1]), fmaxf(s[j][2], s[j][3])), st.m[j]);
        alpha[j] = mn == -INFINITY ? 1.0f : exp2_fast(st.m[j] - mn);
        moved = moved || mn != st.m[j];
        st.m[j] = mn;
    }
    if (__ballot(moved) != 0) {
#pragma unroll
        for (int j = 0; j < QC; ++j) {
            st.l[j] *= alpha[j];
#pragma unroll
            for (int d = 0; d < 16; ++d) st.acc[j][d] *= alpha[j];
        }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        float v[16];
        values16(r[t].v, r[t].vs, v);
#pragma unroll
        for (int j = 0; j < QC; ++j) {
            const float p = s[j][t] == -INFINITY ? 0.0f : exp2_fast(s[j][t] - st.m[j]);
            st.l[j] += p;
#pragma unroll
            for (int d = 0; d < 16; ++d) st.acc[j][d] = fmaf(p, v[d], st.acc[j][d]);
        }
    }
}

// The eight octets' states of a wave become one, in every octet.
template <int QC>
__device__ __forceinline__ void join_octets(FoldState<QC>& st) {
#pragma unroll
    for (int j = 0; j < QC; ++j) {
        float mx = st.m[j];
        mx = fmaxf(mx, lane_xor<8>(mx));
        mx = fmaxf(mx, lane_xor<16>(mx));
        mx = fmaxf(mx, lane_xor<32>(mx));
        const float f = state_weight(st.m[j], st.l[j], mx);
        auto sum = [](float v) {
            v += lane_xor<8>(v);
            v += lane_xor<16>(v);
            return v + lane_xor<32>(v);
        };
        st.l[j] = sum(st.l[j] * f);
#pragma unroll
        for (int d = 0; d < 16; ++d) st.acc[j][d] = sum(st.acc[j][d] * f);
        st.m[j] = mx;
    }
}

// ---- the merge --------------------------------------------------------------

// Whether this workgroup is the last of `n` to come here (the states before it
// are acknowledged; the ticket goes back to zero).
__device__ __forceinline__ bool last_of(uint32_t* ticket, uint32_t n, uint32_t* s_last) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        const uint32_t old = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *s_last = old + 1u == n ? 1u : 0u;
        if (*s_last != 0u) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return *s_last != 0u;
}

// Adds `n` states, `stride` floats apart, to a wave's running (m, l, a0, a1);
// a lane owns dims lane and lane + 64.
__device__ __forceinline__ void fold_states(const float* ps, int64_t stride, int n, float& m, float& l, float& a0,
                                            float& a1) {
    constexpr int NF = 16;
    const int lane = threadIdx.x & (kWave - 1);
    for (int s0 = 0; s0 < n; s0 += NF) {
        float ms = -INFINITY, ls = 0.0f, x0[NF], x1[NF];
        const int k = min(NF, n - s0);
        if (lane < k) {
            ms = ld_f32<true>(ps + (s0 + lane) * stride);
            ls = ld_f32<true>(ps + (s0 + lane) * stride + 1);
        }
#pragma unroll
        for (int j = 0; j < NF; ++j) {
            const float* p = ps + (s0 + min(j, k - 1)) * stride + 2;
            x0[j] = ld_f32<true>(p + lane);
            x1[j] = ld_f32<true>(p + lane + 64);
        }
        const float mx = fmaxf(m, wave_max(ms));
        const float w = state_weight(ms, ls, mx);
        const float f = state_weight(m, l, mx);
        l = fmaf(l, f, wave_sum(ls * w));
        a0 *= f;
        a1 *= f;
#pragma unroll
        for (int j = 0; j < NF; ++j) {
            if (j < k) {
                const float wj = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), j));
                a0 = fmaf(wj, x0[j], a0);
                a1 = fmaf(wj, x1[j], a1);
            }
        }
        m = mx;
    }
}

// A row's output from its merged state and `hits` times the current token (NaN
// logits stay; nothing at all gives zeros).
template <typename T>
__device__ __forceinline__ void finish_row(float m, float l, float a0, float a1, float hits, const T* q, const T* ck,
                                           const T* cv, T* out) {
    const int lane = threadIdx.x & (kWave - 1);
    if (hits > 0.0f) {
        const float q0 = Elem<T>::load(q, lane), q1 = Elem<T>::load(q, lane + 64);
        const float k0 = Elem<T>::load(ck, lane), k1 = Elem<T>::load(ck, lane + 64);
        const float v0 = Elem<T>::load(cv, lane), v1 = Elem<T>::load(cv, lane + 64);
        const float s = scaled_logit(wave_sum(fmaf(q0, k0, q1 * k1)));
        const float mx = fmaxf(m, s);
        const float f = state_weight(m, l, mx), w = s == -INFINITY && mx != -INFINITY ? 0.0f : hits * exp2_fast(s - mx);
        l = fmaf(l, f, w);
        a0 = fmaf(a0, f, w * v0);
        a1 = fmaf(a1, f, w * v1);
    }
    const bool empty = l == 0.0f;
    Elem<T>::store(out, lane, empty ? 0.0f : a0 / l);
    Elem<T>::store(out, lane + 64, empty ? 0.0f : a1 / l);
}

// ---- dense ------------------------------------------------------------------

constexpr int kDenseWaves = 8;
constexpr int kDenseThreads = kDenseWaves * kWave;
// Tokens of a split: at least a tile for every wave.
constexpr int kDenseLeast = kDenseWaves * kPageTile;
constexpr int kDenseBlocks = 256;

int64_t dense_target(int64_t kv_heads) { return kDenseBlocks / kv_heads < 1 ? 1 : kDenseBlocks / kv_heads; }

// A wave-uniform 64-bit value as one the compiler knows to be uniform.
__device__ __forceinline__ int64_t uniform64(int64_t v, int src = 0) {
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(v), src);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(static_cast<uint64_t>(v) >> 32), src);
    return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}

// A workgroup's share: tokens [t0, t1) of sequence b, split `s` of `n`, the
// sequence's first item.
struct DenseShare {
    int b, s, n, first;
    int64_t t0, t1;
};

// The splits follow the real lengths, read on the device: every split holds at
// most total / target tokens (at least kDenseLeast), so a batch of short and
// long sequences is shared out evenly, in at most target + batch items.  Each
// wave works it out by itself from the counts.
__device__ __forceinline__ bool dense_share(const PagedView& c, int64_t max_tokens, int target, int item,
                                            DenseShare& out) {
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t most = min(c.width << c.page_log2, max_tokens);
    int64_t total = 0;
    for (int b0 = 0; b0 < c.batch; b0 += kWave) {
        int64_t n = b0 + lane < c.batch ? clamp_count(c.counts[b0 + lane], most) : 0;
        for (int o = 32; o; o >>= 1) n += __shfl_xor(n, o);
        total += n;
    }
    total = uniform64(total);
    int64_t per = ((total + target - 1) / target + kDenseLeast - 1) / kDenseLeast * kDenseLeast;
    if (per < kDenseLeast) per = kDenseLeast;
    int base = 0;
    for (int b0 = 0; b0 < c.batch; b0 += kWave) {
        const int64_t count = b0 + lane < c.batch ? clamp_count(c.counts[b0 + lane], most) : 0;
        const int splits = b0 + lane < c.batch ? max(1, static_cast<int>((count + per - 1) / per)) : 0;
        const int incl = static_cast<int>(wave_incl_scan(static_cast<uint32_t>(splits), lane));
        const int excl = base + incl - splits;
        const uint64_t mine = __ballot(item >= excl && item < excl + splits);
        if (mine) {
            const int src = __ffsll(static_cast<unsigned long long>(mine)) - 1;
            out.b = b0 + src;
            out.first = __builtin_amdgcn_readlane(excl, src);
            out.n = __builtin_amdgcn_readlane(splits, src);
            out.s = item - out.first;
            out.t0 = out.s * per;
            const int64_t n = uniform64(count, src);
            out.t1 = min(n, out.t0 + per);
            return true;
        }
        base += __builtin_amdgcn_readlane(incl, kWave - 1);
    }
    return false;
}

// The workgroup's waves hold `rows` states each in LDS (row-major: s_m, s_l
// [W][rows], s_acc [W][rows][128]); rows r0 .. of the item's group go to the
// partials as one state each.
template <int ROWS, int PITCH>
__device__ __forceinline__ void store_states(const float (*s_m)[ROWS], const float (*s_l)[ROWS],
                                             const float (*s_acc)[ROWS][PITCH], int rows, float* dst) {
    for (int i = threadIdx.x; i < rows * 128; i += kDenseThreads) {
        const int j = i / 128, d = i % 128;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < kDenseWaves; ++w) mx = fmaxf(mx, s_m[w][j]);
        float a = 0.0f, l = 0.0f;
#pragma unroll
        for (int w = 0; w < kDenseWaves; ++w) {
            const float f = state_weight(s_m[w][j], s_l[w][j], mx);
            a = fmaf(f, s_acc[w][j][d], a);
            l = fmaf(f, s_l[w][j], l);
        }
        float* p = dst + static_cast<int64_t>(j) * kState;
        st_f32<true>(p + 2 + d, a);
        if (d == 0) {
            st_f32<true>(p, mx);
            st_f32<true>(p + 1, l);
        }
    }
}

// The last workgroup of a (sequence, KV head) merges the group's rows: a row
// takes a wave, or up to eight waves' shares of its splits where the group has
// fewer rows than the workgroup waves.
template <typename T>
__device__ __forceinline__ void dense_merge(const PagedAttend& a, const PagedView& c, const DenseShare& sh, int h,
                                            int group) {
    __shared__ uint32_t s_last;
    __shared__ float s_part[kDenseWaves][kState];
    if (!last_of(a.tickets + sh.b * c.kv_heads + h, sh.n, &s_last)) return;
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    int share = 1;  // waves a row
    while (share * 2 * group <= kDenseWaves && share * 2 <= sh.n) share *= 2;
    const int at_once = kDenseWaves / share;
    const int64_t stride = static_cast<int64_t>(c.kv_heads) * group * kState;
    for (int r0 = 0; r0 < group; r0 += at_once) {
        const int r = r0 + wave / share, part = wave % share;
        float m = -INFINITY, l = 0.0f, a0 = 0.0f, a1 = 0.0f;
        if (r < group) {
            const int s0 = sh.n * part / share, s1 = sh.n * (part + 1) / share;
            const float* ps = a.partials + (static_cast<int64_t>(sh.first + s0) * c.kv_heads + h) * group * kState +
                              static_cast<int64_t>(r) * kState;
            fold_states(ps, stride, s1 - s0, m, l, a0, a1);
        }
        if (share > 1) {
            __syncthreads();
            if (lane == 0) {
                s_part[wave][0] = m;
                s_part[wave][1] = l;
            }
            s_part[wave][2 + lane] = a0;
            s_part[wave][66 + lane] = a1;
            __syncthreads();
            if (part == 0 && r < group) {
                for (int w = 1; w < share; ++w) {
                    const float m2 = s_part[wave + w][0], l2 = s_part[wave + w][1], mx = fmaxf(m, m2);
                    const float f = state_weight(m, l, mx), g = state_weight(m2, l2, mx);
                    l = fmaf(l, f, l2 * g);
                    a0 = fmaf(a0, f, s_part[wave + w][2 + lane] * g);
                    a1 = fmaf(a1, f, s_part[wave + w][66 + lane] * g);
                    m = mx;
                }
            }
        }
        if (part == 0 && r < group) {
            const int64_t row = static_cast<int64_t>(sh.b) * a.q_heads + static_cast<int64_t>(h) * group + r;
            const int64_t kv = (static_cast<int64_t>(sh.b) * c.kv_heads + h) * 128;
            finish_row<T>(m, l, a0, a1, 1.0f, static_cast<const T*>(a.q) + row * 128,
                          static_cast<const T*>(a.cur_k) + kv, static_cast<const T*>(a.cur_v) + kv,
                          static_cast<T*>(a.out) + row * 128);
        }
    }
}

// Matrix-core form (16-bit types), one workgroup a (share, KV head) for the
// whole group: its query heads are the 16 rows of the products (those past the
// group zero), so any group of 1 to 16 costs the same.  A wave takes tiles of
// 32 tokens, two of 16 for the logits:
//   dot_g[head, token] = q . c       one 16 x 16 x 32 step per 32 dims, codes as
//                                    they are, each scale group by itself
//   S = sum_g delta_g dot_g + sum_g low_g qsum_g   in fp32, the second sum by
//                                    one more product (qsum in two fp16 terms)
//   O[head, dim] += P . V            V as low + c delta in fp16
// so keys enter the logits exactly: with the outlier channels that keys have,
// their rounding to fp16 was four times fp16's own in the result.  (C layout:
// lane l holds rows 4 (l / 16) .. + 3 of column l % 16; A and B: lane l holds
// k-elements 8 (l / 16) .. + 7 of row / column l % 16.)
// A code becomes fp16 by its bits: 0x6400 | c is 1024 + c, and 0x6400 | 16 c
// is 1024 + 16 c.  For the keys the queries of odd dims are divided by 16, and
// what codes of zero would give, times delta, is taken off in that same extra
// product, so a dword of eight costs five instructions; for the values a packed
// subtraction and a packed fma follow (13).  A token's 16-byte quarters are exchanged among the four
// lane groups (lane swaps), so that a step's 32 dims are one group's.
// Queries are scaled by a power of two per head (bf16 reaches past fp16, and
// 1024 times a group's sum must not), and the weights are kept around 2^8, where fp16 keeps
// 11 bits; fp16 outputs take a second term for the rest of each weight.
// The same pairs as low + c * delta.
__device__ __forceinline__ void dequantise_pairs(const CodeBits& k, uint32_t w, half2_t delta, half2_t low, uint32_t (&out)[4]) {
    const half2_t k1024 = {1024.0f16, 1024.0f16}, k16th = {0.0625f16, 0.0625f16}, k64 = {-64.0f16, -64.0f16};
    uint32_t b[4];
    biased_pairs(k, w, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const half2_t c = i & 1 ? __builtin_elementwise_fma(as_half2(b[i]), k16th, k64) : as_half2(b[i]) - k1024;
        out[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(c, delta, low));
    }
}

__device__ __forceinline__ f32x4_t mfma_f16(const uint32_t (&a)[4], const uint32_t (&b)[4], f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, make_uint4(a[0], a[1], a[2], a[3])),
                                                  __builtin_bit_cast(half8_t, make_uint4(b[0], b[1], b[2], b[3])), c, 0, 0, 0);
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

template <typename T, int G>
__global__ __launch_bounds__(kDenseThreads) void paged_dense_mfma_kernel(PagedAttend a, PagedView c, int64_t max_tokens,
                                                                         int target) {
    constexpr int R = 128 / G;
    constexpr int HALVES = R == 8 ? 2 : 1;        // groups of a 32-dim step
    constexpr int LOWS = R == 8 ? 2 : 1;          // products for the low terms (four groups each)
    constexpr int TERMS = std::is_same_v<T, f16_t> ? 2 : 1;
    constexpr float kBase = 8.0f, kTop = 15.0f;   // weights start at 2^8 and may grow to 2^15
    constexpr float kNone = -3e38f;               // no weight yet
    const int h = blockIdx.x % c.kv_heads, item = blockIdx.x / c.kv_heads;
    DenseShare sh;
    if (!dense_share(c, max_tokens, target, item, sh)) return;
    const int group = a.q_heads / c.kv_heads;
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col = lane & 15, grp = lane >> 4;

    // the queries: row `col`, dims 32 s + 8 grp .. + 7 in step s, largest
    // magnitude of a head in [1/2, 1)
    uint32_t qa[HALVES][4][4], ql[LOWS][4];
    float factor[4];  // of rows 4 grp + i
    {
        float q[4][8], top = 0.0f;
        const int64_t row = static_cast<int64_t>(sh.b) * a.q_heads + static_cast<int64_t>(h) * group + min(col, group - 1);
        const T* src = static_cast<const T*>(a.q) + row * 128 + 8 * grp;
#pragma unroll
        for (int s = 0; s < 4; ++s) load8<T>(src + 32 * s, q[s]);
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (col >= group) q[s][i] = 0.0f;
                top = fmaxf(top, fabsf(q[s][i]));
            }
        top = fmaxf(top, lane_xor<16>(top));
        top = fmaxf(top, lane_xor<32>(top));
        const int e = static_cast<int>((__float_as_uint(top) >> 23) & 0xffu) - 127;
        const float mine = ldexpf(kScaleHigh, e + 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) factor[i] = __shfl(mine, 4 * grp + i);
        float sum[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            sum[s] = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                q[s][i] = ldexpf(q[s][i], -1 - e);
                sum[s] += q[s][i];
                if (i & 1) q[s][i] *= 0.0625f;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t x = pack_half2(q[s][j], q[s][j + 4]);
                if constexpr (HALVES == 2) {
                    qa[0][s][j] = grp < 2 ? x : 0u;
                    qa[1][s][j] = grp < 2 ? 0u : x;
                } else {
                    qa[0][s][j] = x;
                }
            }
            sum[s] += lane_xor<16>(sum[s]);
        }
        // the low terms' product: lane group 0 holds the groups' sums of queries
        // for low, lane group 1 minus their products with codes of zero for
        // delta, each as (high, rest)
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
        const uint32_t none[4] = {0x64006400u, 0x64006400u, 0x64006400u, 0x64006400u};
#pragma unroll
        for (int g = 0; g < 4 * LOWS; ++g) {
            uint32_t x = 0;
            if (g < R) {
                f32x4_t z = {0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (R == 2) z = mfma_f16(none, qa[0][2 * g % 4 + 1], mfma_f16(none, qa[0][2 * g % 4], z));
                else z = mfma_f16(none, qa[g % HALVES][g / HALVES % 4], z);
                // (rows of codes times columns of queries: every element of column `col` is head `col`'s)
                const float term = grp == 0 ? qs[g % R] : -z[0];
                const float high = static_cast<float>(static_cast<_Float16>(term));
                x = pack_half2(high, term - high);
            }
            ql[g / 4][g % 4] = grp < 2 ? x : 0u;
        }
    }
    const CodeBits bits;
    const uint32_t low_or_delta = grp == 1 ? 0x03020302u : 0x01000100u;  // byte picks of a scale pair

    struct Tile {
        uint4 k[2];
        uint32_t ks[2][R], v[8], vs[8];
        int left;  // live tokens
    };
    const int64_t per_page = static_cast<int64_t>(c.kv_heads) << c.page_log2, head_row = static_cast<int64_t>(h) << c.page_log2;
    const int in_page = (1 << c.page_log2) - 1;
    const int64_t first = sh.t0 + wave * kPageTile;
    const int tiles = first < sh.t1 ? static_cast<int>((sh.t1 - first + kDenseLeast - 1) / kDenseLeast) : 0;
    const uint32_t ko = col * kCodeRow + 16 * grp, vo = 4 * grp * kCodeRow + 64 + 4 * col;
    const uint32_t kso = col * (8 * R), vso = 4 * grp * (8 * R) + 4 * (R + 8 * col / G);
    int32_t entries = -1;  // lane i: the page of this wave's tile i of a block of 64
    auto load_entries = [&](int i0) {
        const int64_t t = first + static_cast<int64_t>(i0 + lane) * kDenseLeast;
        entries = t < sh.t1 ? c.table[sh.b * c.width + (t >> c.page_log2)] : -1;
    };
    auto load_tile = [&](int i, Tile& x) {
        const int64_t t = first + static_cast<int64_t>(i) * kDenseLeast;
        const int32_t e = __builtin_amdgcn_readlane(entries, i & (kWave - 1));
        const bool there = static_cast<uint32_t>(e) < static_cast<uint32_t>(c.pages);
        x.left = there ? static_cast<int>(min<int64_t>(kPageTile, sh.t1 - t)) : 0;
        const int64_t row = (there ? e : 0) * per_page + head_row + (t & in_page);
        const char* code = c.codes + row * kCodeRow;
        const char* sc = reinterpret_cast<const char*>(c.scales) + row * (8 * R);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            x.k[u] = *reinterpret_cast<const uint4*>(code + ko + 16 * u * kCodeRow);
            const char* p = sc + kso + 16 * u * (8 * R);
            if constexpr (R == 2) {
                const uint2 w = *reinterpret_cast<const uint2*>(p);
                x.ks[u][0] = w.x;
                x.ks[u][1] = w.y;
            } else {
#pragma unroll
                for (int g = 0; g < R; g += 4) {
                    const uint4 w = *reinterpret_cast<const uint4*>(p + 4 * g);
                    x.ks[u][g] = w.x;
                    x.ks[u][g + 1] = w.y;
                    x.ks[u][g + 2] = w.z;
                    x.ks[u][g + 3] = w.w;
                }
            }
        }
        // v[2 j], v[2 j + 1]: tokens 4 grp + j and 16 + 4 grp + j
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int tok = (j >> 1) + 16 * (j & 1);
            x.v[j] = *reinterpret_cast<const uint32_t*>(code + vo + tok * kCodeRow);
            x.vs[j] = *reinterpret_cast<const uint32_t*>(sc + vso + tok * (8 * R));
        }
    };

    // a wave's weights on their way from the logits' lanes to the product's:
    // [term][head][token pair (n, 16 + n)]
    __shared__ __align__(16) uint32_t s_p[kDenseWaves][TERMS][16][16];
    f32x4_t acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    float ref[4], l[4];  // rows 4 grp + i: weights are 2^(logit - ref)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        ref[i] = kNone;
        l[i] = 0.0f;
    }
    auto fold = [&](Tile& x) {
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
                biased_pairs(bits, w[st], cb);
                if constexpr (R == 2) {
                    dot[st / 2] = mfma_f16(qa[0][st], cb, st & 1 ? dot[st / 2] : f32x4_t{0.0f, 0.0f, 0.0f, 0.0f});
                } else {
#pragma unroll
                    for (int n = 0; n < HALVES; ++n)
                        dot[HALVES * st + n] = mfma_f16(qa[n][st], cb, f32x4_t{0.0f, 0.0f, 0.0f, 0.0f});
                }
            }
#pragma unroll
            for (int g = 0; g < R; ++g) {
                const float delta = static_cast<float>(as_half2(x.ks[u][g])[1]);
#pragma unroll
                for (int i = 0; i < 4; ++i) s[u][i] = fmaf(delta, dot[g][i], s[u][i]);
            }
        }
        const bool whole = x.left == kPageTile;  // uniform; the branches stay branches
        bool live[2] = {true, true};
        if (!whole) {
            asm volatile("");
#pragma unroll
            for (int u = 0; u < 2; ++u) live[u] = col + 16 * u < x.left;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (4 * grp + (j >> 1) + 16 * (j & 1) >= x.left) x.vs[j] = 0u;  // what lies behind the last token may be anything
        }
        float e[4][2], top = -INFINITY;
        auto exponents = [&] {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int u = 0; u < 2; ++u) e[i][u] = fmaf(s[u][i], factor[i], -ref[i]);
            if (!whole) {
                asm volatile("");
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int u = 0; u < 2; ++u) e[i][u] = live[u] ? e[i][u] : -INFINITY;
            }
        };
        exponents();
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(e[i][0], e[i][1]));
        if (__ballot(top > kTop) != 0) {  // some weight would pass 2^15
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float mx = fmaxf(live[0] ? s[0][i] * factor[i] : -INFINITY, live[1] ? s[1][i] * factor[i] : -INFINITY);
                mx = fmaxf(mx, dpp_mov<0xB1>(mx));
                mx = fmaxf(mx, dpp_mov<0x4E>(mx));
                mx = fmaxf(mx, dpp_mov<0x141>(mx));
                mx = fmaxf(mx, dpp_mov<0x140>(mx));
                const float to = fmaxf(mx - kBase, ref[i]);
                const float f = exp2_fast(ref[i] - to);
                l[i] *= f;
#pragma unroll
                for (int d = 0; d < 8; ++d) acc[d][i] *= f;
                ref[i] = to;
            }
            exponents();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float p0 = exp2_fast(e[i][0]), p1 = exp2_fast(e[i][1]);
            l[i] += p0 + p1;
            const uint32_t p = pack_half2(p0, p1);
            s_p[wave][0][4 * grp + i][col] = p;
            if constexpr (TERMS == 2)
                s_p[wave][1][4 * grp + i][col] = pack_half2(p0 - static_cast<float>(as_half2(p)[0]),
                                                            p1 - static_cast<float>(as_half2(p)[1]));
        }
        // the wave reads its own weights next: one wave's LDS operations complete in order
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        uint32_t pa[TERMS][4];
#pragma unroll
        for (int n = 0; n < TERMS; ++n) {
            const uint4 w = *reinterpret_cast<const uint4*>(&s_p[wave][n][col][4 * grp]);
            pa[n][0] = w.x;
            pa[n][1] = w.y;
            pa[n][2] = w.z;
            pa[n][3] = w.w;
        }
        // a lane's eight dims 8 col .. + 7 of V: the low halves of the tokens'
        // dwords hold dims 0 .. 3, the high ones 4 .. 7
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
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int n = 0; n < TERMS; ++n) acc[4 * half + i] = mfma_f16(pa[n], vf[i], acc[4 * half + i]);
        }
        // the next tile's weights overwrite s_p only after every lane has read
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };
    Tile x, y;
    for (int i0 = 0; i0 < tiles; i0 += kWave) {
        const int n = min(kWave, tiles - i0);
        load_entries(i0);
        load_tile(i0, x);
        for (int i = 0; i < n; i += 2) {
            if (i + 1 < n) load_tile(i0 + i + 1, y);
            fold(x);
            if (i + 1 >= n) break;
            if (i + 2 < n) load_tile(i0 + i + 2, x);
            fold(y);
        }
    }

    // the waves' states meet in LDS, eight heads at a time
    constexpr int ROWS = 8, PITCH = 132;
    __shared__ float s_m[kDenseWaves][ROWS], s_l[kDenseWaves][ROWS];
    __shared__ __align__(16) float s_acc[kDenseWaves][ROWS][PITCH];
#pragma unroll
    for (int i = 0; i < 4; ++i) l[i] = row_sum<16>(l[i]);
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
        store_states<ROWS, PITCH>(s_m, s_l, s_acc, min(ROWS, group - r0),
                                  a.partials + ((static_cast<int64_t>(item) * c.kv_heads + h) * group + r0) * kState);
        __syncthreads();
    }
    dense_merge<T>(a, c, sh, h, group);
}

// VALU form (fp32), QC query heads of the group at a time.  A tile of 32
// tokens lies in one page: its table entry is one scalar.
template <typename T, int G, int QC>
__global__ __launch_bounds__(kDenseThreads) void paged_dense_kernel(PagedAttend a, PagedView c, int64_t max_tokens,
                                                                    int target) {
    constexpr int R = 128 / G;
    const int h = blockIdx.x % c.kv_heads, item = blockIdx.x / c.kv_heads;
    DenseShare sh;
    if (!dense_share(c, max_tokens, target, item, sh)) return;
    const int group = a.q_heads / c.kv_heads;
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int oct = lane / 8, d0 = (lane % 8) * 16;
    __shared__ float s_m[kDenseWaves][QC], s_l[kDenseWaves][QC];
    __shared__ float s_acc[kDenseWaves][QC][128];
    const int64_t per_page = static_cast<int64_t>(c.kv_heads) << c.page_log2;
    const int64_t head_row = static_cast<int64_t>(h) << c.page_log2;
    for (int j0 = 0; j0 < group; j0 += QC) {
        const int rows = min(QC, group - j0);
        float q[QC][16];
#pragma unroll
        for (int j = 0; j < QC; ++j) {
            const int64_t row = static_cast<int64_t>(sh.b) * a.q_heads + static_cast<int64_t>(h) * group + j0 + min(j, rows - 1);
            load8<T>(static_cast<const T*>(a.q) + row * 128 + d0, q[j]);
            load8<T>(static_cast<const T*>(a.q) + row * 128 + d0 + 8, q[j] + 8);
        }
        FoldState<QC> st;
        st.clear();
        for (int64_t t = sh.t0 + wave * kPageTile; t < sh.t1; t += kDenseLeast) {
            const int32_t page = c.table[sh.b * c.width + (t >> c.page_log2)];
            if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(c.pages)) continue;  // uniform
            const int64_t row0 = page * per_page + head_row + (t & ((1 << c.page_log2) - 1));
            const int left = static_cast<int>(min<int64_t>(kPageTile, sh.t1 - t));
            Row4 r[4];
            bool live[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int tok = oct + 8 * i;
                live[i] = tok < left;
                const char* code = c.codes + (row0 + tok) * kCodeRow + d0 / 2;
                const uint32_t* sc = c.scales + (row0 + tok) * (2 * R) + d0 / G;
                r[i].k = *reinterpret_cast<const uint2*>(code);
                r[i].v = *reinterpret_cast<const uint2*>(code + 64);
                r[i].ks = sc[0];
                r[i].vs = live[i] ? sc[R] : 0u;  // what lies behind the last token may be anything
            }
            fold4<QC>(st, q, r, live);
        }
        join_octets<QC>(st);
        if (lane < 8) {
#pragma unroll
            for (int j = 0; j < QC; ++j) {
#pragma unroll
                for (int d = 0; d < 16; ++d) s_acc[wave][j][d0 + d] = st.acc[j][d];
                if (lane == 0) {
                    s_m[wave][j] = st.m[j];
                    s_l[wave][j] = st.l[j];
                }
            }
        }
        __syncthreads();
        store_states<QC, 128>(s_m, s_l, s_acc, rows,
                         a.partials + ((static_cast<int64_t>(item) * c.kv_heads + h) * group + j0) * kState);
        __syncthreads();
    }
    dense_merge<T>(a, c, sh, h, group);
}

// ---- indexed ----------------------------------------------------------------

// An octet's state for one query head, fp32 or 16-bit queries.  16-bit: codes
// as fp16 c - 8, dot products in packed pairs (v_dot2, fp32 sums),
//   s = delta sum(q (c - 8)) + mid sum(q),  mid = low + 8 delta
//   acc += (p delta) (c - 8),  the p mid apart
// 76 instructions a token against 115 for values dequantised to fp32; taking
// the middle of the codes keeps the two sums from cancelling.
template <typename T>
struct PickFold {
    FoldState<1> st;
    CodeBits bits;
    uint32_t qh[8];
    float qsum, factor, mid;
    __device__ __forceinline__ void start(const T* src) {
        st.clear();
        mid = 0.0f;
        float q[16], top = 0.0f;
        load8<T>(src, q);
        load8<T>(src + 8, q + 8);
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(q[i]));
        top = fmaxf(top, dpp_mov<0xB1>(top));
        top = fmaxf(top, dpp_mov<0x4E>(top));
        top = fmaxf(top, dpp_mov<0x141>(top));
        // fp16 to the queries' precision: the head's largest magnitude in [2^8, 2^9)
        const int e = static_cast<int>((__float_as_uint(top) >> 23) & 0xffu) - 127;
        factor = ldexpf(kScaleHigh, e - 8);
        qsum = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            q[i] = ldexpf(q[i], 8 - e);
            qsum += q[i];
        }
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int j = 0; j < 4; ++j) qh[4 * w + j] = pack_half2(q[8 * w + j], q[8 * w + j + 4]);
    }
    static __device__ __forceinline__ void centred(const CodeBits& k, uint32_t w, half2_t (&out)[4]) {
        const half2_t k1032 = {1032.0f16, 1032.0f16}, k16th = {0.0625f16, 0.0625f16}, k72 = {-72.0f16, -72.0f16};
        uint32_t b[4];
        biased_pairs(k, w, b);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            out[j] = j & 1 ? __builtin_elementwise_fma(as_half2(b[j]), k16th, k72) : as_half2(b[j]) - k1032;
    }
    __device__ __forceinline__ void fold(const Row4 (&r)[4], const bool (&live)[4]) {
        float s[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            float dot = 0.0f;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                half2_t c[4];
                centred(bits, w ? r[t].k.y : r[t].k.x, c);
#pragma unroll
                for (int j = 0; j < 4; ++j) dot = __builtin_amdgcn_fdot2(as_half2(qh[4 * w + j]), c[j], dot, false);
            }
            const float low = f16_lo(r[t].ks), delta = f16_hi(r[t].ks);
            const float x = row_sum<8>(fmaf(delta, dot, fmaf(8.0f, delta, low) * qsum)) * factor;
            s[t] = live[t] ? x : -INFINITY;
        }
        const float mn = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), st.m[0]);
        if (__ballot(mn != st.m[0]) != 0) {
            const float f = mn == -INFINITY ? 1.0f : exp2_fast(st.m[0] - mn);
            st.l[0] *= f;
            mid *= f;
#pragma unroll
            for (int d = 0; d < 16; ++d) st.acc[0][d] *= f;
            st.m[0] = mn;
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const float p = s[t] == -INFINITY ? 0.0f : exp2_fast(s[t] - mn);
            const float low = f16_lo(r[t].vs), delta = f16_hi(r[t].vs);
            st.l[0] += p;
            mid = fmaf(p, fmaf(8.0f, delta, low), mid);
            const float pd = p * delta;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                half2_t c[4];
                centred(bits, w ? r[t].v.y : r[t].v.x, c);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    st.acc[0][8 * w + j] = fmaf(static_cast<float>(c[j][0]), pd, st.acc[0][8 * w + j]);
                    st.acc[0][8 * w + j + 4] = fmaf(static_cast<float>(c[j][1]), pd, st.acc[0][8 * w + j + 4]);
                }
            }
        }
    }
    __device__ __forceinline__ void join() {
#pragma unroll
        for (int d = 0; d < 16; ++d) st.acc[0][d] += mid;
        join_octets<1>(st);
    }
};
template <>
struct PickFold<float> {
    FoldState<1> st;
    float q[1][16];
    __device__ __forceinline__ void start(const float* src) {
        st.clear();
        load8<float>(src, q[0]);
        load8<float>(src + 8, q[0] + 8);
    }
    __device__ __forceinline__ void fold(const Row4 (&r)[4], const bool (&live)[4]) { fold4<1>(st, q, r, live); }
    __device__ __forceinline__ void join() { join_octets<1>(st); }
};

constexpr int kPickWaves = 4;
constexpr int kPickThreads = kPickWaves * kWave;
constexpr int kPickRows = 8;                            // tokens an octet loads at once
constexpr int kPickTile = kPickRows * kWave / 8;        // tokens of a wave's pass
constexpr int kPickLeast = kPickWaves * kPickTile;
constexpr int kPickBlocks = 512;
constexpr int kPickState = kState + 1;                  // (m, l, acc[128], hits of the current token)

// Output dim threadIdx.x (of waves 0 and 1) from the row's state and `hits`
// times the current token; nothing at all gives zero.
template <typename T>
__device__ __forceinline__ void pick_finish(float m, float l, float x, float hits, const T* q, const T* ck, const T* cv,
                                            T* out) {
    const int lane = threadIdx.x & (kWave - 1), d = threadIdx.x;
    if (hits > 0.0f) {
        const float s = scaled_logit(wave_sum(fmaf(Elem<T>::load(q, lane), Elem<T>::load(ck, lane),
                                                   Elem<T>::load(q, lane + 64) * Elem<T>::load(ck, lane + 64))));
        const float mx = fmaxf(m, s);
        const float f = state_weight(m, l, mx);
        const float w = s == -INFINITY && mx != -INFINITY ? 0.0f : hits * exp2_fast(s - mx);
        l = fmaf(l, f, w);
        x = fmaf(x, f, w * Elem<T>::load(cv, d));
    }
    Elem<T>::store(out, d, l == 0.0f ? 0.0f : x / l);
}

// Merges a row's `n` states by the whole workgroup: the weights of 64 states at
// a time by every wave alike, the sums by threads (dim, half of the states).
template <typename T>
__device__ __forceinline__ void pick_merge(const float* ps, int n, const T* q, const T* ck, const T* cv, T* out) {
    constexpr int NF = 16;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int d = threadIdx.x & 127, half = threadIdx.x >> 7;
    float m = -INFINITY, l = 0.0f, hits = 0.0f, a = 0.0f;
    for (int s0 = 0; s0 < n; s0 += 2 * NF) {
        const int k = min(2 * NF, n - s0);
        const float* p = ps + static_cast<int64_t>(s0) * kPickState;
        float x[NF], ms = -INFINITY, ls = 0.0f, hs = 0.0f;
        if (lane < k) {
            ms = ld_f32<true>(p + lane * kPickState);
            ls = ld_f32<true>(p + lane * kPickState + 1);
            hs = ld_f32<true>(p + lane * kPickState + kState);
        }
#pragma unroll
        for (int j = 0; j < NF; ++j) x[j] = ld_f32<true>(p + min(2 * j + half, k - 1) * kPickState + 2 + d);
        const float mx = fmaxf(m, wave_max(ms));
        const float f = state_weight(m, l, mx), w = state_weight(ms, ls, mx);
        l = fmaf(l, f, wave_sum(ls * w));
        hits += wave_sum(hs);
        a *= f;
#pragma unroll
        for (int j = 0; j < NF; ++j)
            if (2 * j + half < k) a = fmaf(__shfl(w, 2 * j + half), x[j], a);
        m = mx;
    }
    __shared__ float s_sum[128];
    if (half == 1) s_sum[d] = a;
    __syncthreads();
    if (wave < 2) pick_finish<T>(m, l, a + s_sum[d], hits, q, ck, cv, out);
}

// One workgroup a (split of the selection, query head, sequence): every query
// head gathers its own tokens.  The current token is counted, not read: the
// merge folds it in as often as it was selected.
template <typename T, int G, typename I>
__global__ __launch_bounds__(kPickThreads) void paged_indexed_kernel(PagedAttend a, PagedIndexed ix, PagedView c,
                                                                     int splits, int per) {
    constexpr int R = 128 / G;
    const int s = blockIdx.x, qh = blockIdx.y, b = blockIdx.z;
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int oct = lane / 8, d0 = (lane % 8) * 16;
    const int64_t row = static_cast<int64_t>(b) * a.q_heads + qh;
    const int64_t kvh = ix.head_to_kv[qh];
    const int h = static_cast<int>(kvh < 0 ? 0 : kvh >= c.kv_heads ? c.kv_heads - 1 : kvh);
    const int64_t count = clamp_count(c.counts[b], c.width << c.page_log2);
    PickFold<T> f;
    f.start(static_cast<const T*>(a.q) + row * 128 + d0);
    const I* idx = static_cast<const I*>(ix.indices) + row * ix.selected;
    const uint8_t* valid = ix.valid ? ix.valid + row * ix.selected : nullptr;
    const int32_t* table = c.table + b * c.width;
    const int64_t e0 = static_cast<int64_t>(s) * per, e1 = min<int64_t>(e0 + per, ix.selected);
    int hits = 0;
    for (int64_t e = e0 + wave * kPickTile; e < e1; e += kPickLeast) {
        Row4 r[2][4];
        bool live[2][4];
        int64_t tok[kPickRows];
        int32_t page[kPickRows];
#pragma unroll
        for (int i = 0; i < kPickRows; ++i) {
            const int64_t at = e + oct + 8 * i;
            const bool in = at < e1 && (!valid || valid[at] != 0);
            tok[i] = in ? static_cast<int64_t>(idx[at]) : -1;
        }
#pragma unroll
        for (int i = 0; i < kPickRows; ++i) {
            hits += tok[i] == count ? 1 : 0;
            page[i] = tok[i] >= 0 && tok[i] < count ? table[tok[i] >> c.page_log2] : -1;
        }
#pragma unroll
        for (int i = 0; i < kPickRows; ++i) {
            Row4& x = r[i / 4][i % 4];
            const bool there = static_cast<uint32_t>(page[i]) < static_cast<uint32_t>(c.pages);
            live[i / 4][i % 4] = there;
            x.k = x.v = make_uint2(0u, 0u);
            x.ks = x.vs = 0u;
            if (there) {
                const int64_t at_row = ((static_cast<int64_t>(page[i]) * c.kv_heads + h) << c.page_log2) +
                                       (tok[i] & ((1 << c.page_log2) - 1));
                const char* code = c.codes + at_row * kCodeRow + d0 / 2;
                const uint32_t* sc = c.scales + at_row * (2 * R) + d0 / G;
                x.k = *reinterpret_cast<const uint2*>(code);
                x.v = *reinterpret_cast<const uint2*>(code + 64);
                x.ks = sc[0];
                x.vs = sc[R];
            }
        }
        f.fold(r[0], live[0]);
        f.fold(r[1], live[1]);
    }
    f.join();
    const float wave_hits = wave_sum(static_cast<float>(hits)) * 0.125f;  // the eight lanes of an octet count alike
    __shared__ float s_m[kPickWaves], s_l[kPickWaves], s_hits[kPickWaves], s_acc[kPickWaves][128];
    if (lane < 8) {
#pragma unroll
        for (int d = 0; d < 16; ++d) s_acc[wave][d0 + d] = f.st.acc[0][d];
        if (lane == 0) {
            s_m[wave] = f.st.m[0];
            s_l[wave] = f.st.l[0];
            s_hits[wave] = wave_hits;
        }
    }
    __syncthreads();
    float* mine = a.partials + (row * splits + s) * kPickState;
    const int64_t kv = (static_cast<int64_t>(b) * c.kv_heads + h) * 128;
    const T *q = static_cast<const T*>(a.q) + row * 128, *ck = static_cast<const T*>(a.cur_k) + kv,
            *cv = static_cast<const T*>(a.cur_v) + kv;
    T* out = static_cast<T*>(a.out) + row * 128;
    if (wave < 2) {
        float mx = -INFINITY, l = 0.0f, x = 0.0f, n = 0.0f;
#pragma unroll
        for (int w = 0; w < kPickWaves; ++w) mx = fmaxf(mx, s_m[w]);
#pragma unroll
        for (int w = 0; w < kPickWaves; ++w) {
            const float g = state_weight(s_m[w], s_l[w], mx);
            x = fmaf(g, s_acc[w][threadIdx.x], x);
            l = fmaf(g, s_l[w], l);
            n += s_hits[w];
        }
        if (splits == 1) {
            pick_finish<T>(mx, l, x, n, q, ck, cv, out);
        } else {
            st_f32<true>(mine + 2 + threadIdx.x, x);
            if (threadIdx.x == 0) {
                st_f32<true>(mine, mx);
                st_f32<true>(mine + 1, l);
                st_f32<true>(mine + kState, n);
            }
        }
    }
    if (splits == 1) return;
    __shared__ uint32_t s_last;
    if (!last_of(a.tickets + row, splits, &s_last)) return;
    pick_merge<T>(a.partials + row * splits * kPickState, splits, q, ck, cv, out);
}

struct PickPlan {
    int splits, per;
};
PickPlan pick_plan(int64_t rows, int64_t selected) {
    int64_t want = kPickBlocks / rows;
    const int64_t most = (selected + kPickLeast - 1) / kPickLeast;
    if (want > most) want = most;
    if (want < 1) want = 1;
    const int64_t per = ((selected + want - 1) / want + kPickLeast - 1) / kPickLeast * kPickLeast;
    return {static_cast<int>((selected + per - 1) / per), static_cast<int>(per)};
}

template <typename T, int G>
hipError_t launch_dense_t(const PagedAttend& a, const PagedView& c, int64_t max_tokens, hipStream_t stream) {
    const int group = a.q_heads / c.kv_heads;
    const dim3 grid(static_cast<unsigned>(paged_dense_items(c.batch, c.kv_heads, max_tokens) * c.kv_heads));
    const int target = static_cast<int>(dense_target(c.kv_heads));
#define POPKV_DENSE(QC)                                                                                            \
    hipLaunchKernelGGL((paged_dense_kernel<T, G, QC>), grid, dim3(kDenseThreads), 0, stream, a, c, max_tokens, target)
    if constexpr (sizeof(T) == 2) {
        hipLaunchKernelGGL((paged_dense_mfma_kernel<T, G>), grid, dim3(kDenseThreads), 0, stream, a, c, max_tokens, target);
    } else {
        if (group == 1) POPKV_DENSE(1);
        else if (group == 2) POPKV_DENSE(2);
        else POPKV_DENSE(4);
    }
#undef POPKV_DENSE
    return hipGetLastError();
}

template <typename T, int G>
hipError_t launch_indexed_t(const PagedAttend& a, const PagedIndexed& ix, const PagedView& c, hipStream_t stream) {
    const PickPlan p = pick_plan(static_cast<int64_t>(c.batch) * a.q_heads, ix.selected);
    const dim3 grid(static_cast<unsigned>(p.splits), static_cast<unsigned>(a.q_heads), static_cast<unsigned>(c.batch));
    if (ix.index_dtype == POPKV_INDEX_I32)
        hipLaunchKernelGGL((paged_indexed_kernel<T, G, int32_t>), grid, dim3(kPickThreads), 0, stream, a, ix, c, p.splits,
                           p.per);
    else
        hipLaunchKernelGGL((paged_indexed_kernel<T, G, int64_t>), grid, dim3(kPickThreads), 0, stream, a, ix, c, p.splits,
                           p.per);
    return hipGetLastError();
}

}  // namespace

int64_t paged_dense_items(int64_t batch, int64_t kv_heads, int64_t max_tokens) {
    const int64_t target = dense_target(kv_heads);
    const int64_t per_sequence = max_tokens < 1 ? 1 : (max_tokens + kDenseLeast - 1) / kDenseLeast;
    const int64_t all = batch * per_sequence;
    return all < target + batch ? all : target + batch;
}

int64_t paged_indexed_splits(int64_t rows, int64_t selected) { return pick_plan(rows, selected).splits; }

#define POPKV_PAGED_G(CALL, T)                  \
    switch (dim_group) {                        \
        case 16: return CALL(T, 16);            \
        case 32: return CALL(T, 32);            \
        default: return CALL(T, 64);            \
    }
#define POPKV_PAGED_T(CALL)                              \
    switch (dtype) {                                     \
        case POPKV_DTYPE_F32: POPKV_PAGED_G(CALL, float) \
        case POPKV_DTYPE_F16: POPKV_PAGED_G(CALL, f16_t) \
        default: POPKV_PAGED_G(CALL, bf16_t)             \
    }

hipError_t launch_paged_dense(const PagedAttend& a, const PagedView& c, int64_t max_tokens, int dtype, int dim_group,
                              hipStream_t stream) {
#define POPKV_CALL(T, G) launch_dense_t<T, G>(a, c, max_tokens, stream)
    POPKV_PAGED_T(POPKV_CALL)
#undef POPKV_CALL
}

hipError_t launch_paged_indexed(const PagedAttend& a, const PagedIndexed& ix, const PagedView& c, int dtype,
                                int dim_group, hipStream_t stream) {
#define POPKV_CALL(T, G) launch_indexed_t<T, G>(a, ix, c, stream)
    POPKV_PAGED_T(POPKV_CALL)
#undef POPKV_CALL
}

}  // namespace popkv
