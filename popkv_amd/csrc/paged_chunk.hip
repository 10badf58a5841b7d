// Attention of a chunk of new tokens a sequence over its paged 4-bit cache and,
// causally, over the chunk itself.
#include "paged_attention.h"

namespace popkv {
namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

constexpr int kChunkWaves = 4;
constexpr int kChunkThreads = kChunkWaves * kWave;
constexpr int kChunkRows = 32 * kChunkWaves;  // rows of a workgroup: (token, head of the group), heads innermost
constexpr int kChunkTile = 64;                // tokens of a tile
constexpr int kFrag = 1024;                   // bytes of one operand of a 32 x 32 x 16 product

__device__ __forceinline__ f32x16_t mfma_h(const uint4& a, const uint4& b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0,
                                                  0);
}
__device__ __forceinline__ f32x16_t mfma_b(const uint4& a, const uint4& b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0,
                                                   0, 0);
}

// x as bf16 terms: the first `n` of x = b0 + b1 + b2 (b1, b2 zero where x is not finite).
template <int N>
__device__ __forceinline__ void bf16_terms(float x, uint32_t (&t)[N]) {
    t[0] = bf16_rne(x);
    float rest = x - bits_bf16(t[0]);
    if ((t[0] & 0x7f80u) == 0x7f80u) rest = 0.0f;
#pragma unroll
    for (int i = 1; i < N; ++i) {
        t[i] = bf16_rne(rest);
        rest -= bits_bf16(t[i]);
    }
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

// What the kernel holds of each element type.
template <typename T>
struct ChunkTypes {
    static constexpr bool F32 = std::is_same_v<T, float>;
    static constexpr bool F16 = std::is_same_v<T, f16_t>;
    static constexpr int QT = F32 ? 2 : 1;      // fp16 terms of the queries
    static constexpr int KT = 2;                // of the cached keys
    static constexpr int VT = F32 || F16 ? 2 : 1;  // of the cached values and their weights
    static constexpr int NT = F32 ? 3 : 1;      // planes of the new tokens (fp32: bf16 terms)
    static constexpr int PT = F32 ? 3 : 2;      // terms of the weights on new tokens
    static constexpr int QPLANES = F32 ? 3 : 1;
    static constexpr int STORED = QT + QPLANES;  // query operands kept for the second pass
    static constexpr int PLANES = F32 ? 6 : F16 ? 4 : 3;  // 16 KB each
};

// Where lane l's sixteen bytes of value operand i of four lie in its KB: writers
// of one instruction (16 dwords of codes) meet different banks, readers too.
__device__ __forceinline__ int value_slot(int l, int i) { return (l ^ (i | ((l >> 4 & 1) << 3))) * 16; }

template <typename T, int G>
__global__ __launch_bounds__(kChunkThreads) void paged_chunk_kernel(PagedChunk a, PagedView c, int64_t max_tokens) {
    using C = ChunkTypes<T>;
    constexpr int R = 128 / G;
    constexpr int LOWS = R == 8 ? 2 : 1;
    constexpr int QTOP = 5;
    constexpr float kBase = 8.0f, kTop = 15.0f, kNone = -3e38f;
    constexpr int PLANE = kChunkTile / 32 * 8 * kFrag;
    __shared__ __align__(16) unsigned char s_mem[C::PLANES * PLANE];
    __shared__ __align__(16) uint32_t s_scale[kChunkTile][R];
    __shared__ __align__(16) float s_bias[kChunkTile];
    __shared__ int s_ragged[kChunkWaves], s_odd_keys[kChunkWaves];
    unsigned char* const s_k = s_mem;
    unsigned char* const s_v = s_mem + C::KT * PLANE;   // cached tokens
    unsigned char* const s_nv = s_mem + C::NT * PLANE;  // new tokens

    const int b = blockIdx.z, h = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int col = lane & 31, half = lane >> 5;
    const int group = a.q_heads / c.kv_heads;
    const int rows = static_cast<int>(a.tokens ? clamp_count(a.tokens[b], a.rows) : a.rows);
    const int count = static_cast<int>(clamp_count(c.counts[b], min(c.width << c.page_log2, max_tokens)));
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kChunkRows;
    const int64_t all = static_cast<int64_t>(rows) * group;
    if (row0 >= all) return;
    const int64_t row = min<int64_t>(row0 + 32 * wave + col, all - 1);
    const bool live_row = row0 + 32 * wave + col < all;
    const int t_row = static_cast<int>(row / group), head = h * group + static_cast<int>(row - static_cast<int64_t>(t_row) * group);
    const int seen = static_cast<int>(min<int64_t>((row0 + kChunkRows - 1) / group + 1, rows));  // new tokens of the tile

    const T* const q_row = static_cast<const T*>(a.q) + b * a.q_bs + head * a.q_hs + static_cast<int64_t>(t_row) * a.q_ts;
    Raw8<T> raw[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) raw[s].load(q_row + 64 * half + 8 * s);

    f32x16_t acc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[i][j] = 0.0f;
    float ref = kNone, l = 0.0f;

    uint4 q[C::QPLANES][8], ql[LOWS];
    float factor;
    {
        float top = 0.0f;
#pragma unroll
        for (int s = 0; s < 8; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(raw[s].get(i)));
        top = fmaxf(top, lane_xor<32>(top));
        const int e = static_cast<int>((__float_as_uint(top) >> 23) & 0xffu) - 127;
        factor = ldexpf(kScaleHigh, e + 1 - QTOP);
        float sum[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            float x[8];
            sum[s] = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = ldexpf(raw[s].get(i), QTOP - 1 - e);
                sum[s] += x[i];
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
        float qs[8], part[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // sums of every scale group, of this half's
#pragma unroll
        for (int g = 0; g < 8; ++g) qs[g] = 0.0f;
#pragma unroll
        for (int s = 0; s < 8; ++s) part[8 * s / G] += sum[s];
#pragma unroll
        for (int g = 0; g < R / 2; ++g) {
            const float other = lane_xor<32>(part[g]);
            qs[g] = half == 0 ? part[g] : other;
            qs[R / 2 + g] = half == 0 ? other : part[g];
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

    // what the second pass reads of these rows: the query operands of both kinds of tokens, their factors
    const int64_t row_tile = a.weights ? ((static_cast<int64_t>(b) * c.kv_heads + h) * a.row_tiles + blockIdx.x * kChunkWaves + wave) : 0;
    const bool store_rows = a.weights && row0 + 32 * wave < all;
    if (store_rows) {
        if (half == 0) a.factors[row_tile * 32 + col] = factor;
#pragma unroll
        for (int n = 0; n < C::QT; ++n)
#pragma unroll
            for (int s = 0; s < 8; ++s) a.queries[((row_tile * C::STORED + n) * 8 + s) * kWave + lane] = q[n][s];
    }

    // a thread's part of a tile: quarter tid % 4 of token tid / 4's key, dword tid
    // % 16 of the values of tokens 4 (tid / 16) .. + 3, which share a page
    const int my_quad = 4 * (tid / 16), my_token = tid / 4, quarter = tid % 4, dw = tid % 16;
    const int64_t per_page = static_cast<int64_t>(c.kv_heads) << c.page_log2;
    const int64_t head_row = static_cast<int64_t>(h) << c.page_log2;
    const int in_page = (1 << c.page_log2) - 1;
    struct Cached {
        uint4 k;
        uint32_t ks[2], v[4], vs[4];
        bool there;
    } x;
    auto load_cached = [&](int tile) {
        const int t = tile * kChunkTile + my_quad;
        int32_t e = -1;
        if (t < count) e = c.table[b * c.width + (t >> c.page_log2)];
        x.there = static_cast<uint32_t>(e) < static_cast<uint32_t>(c.pages);
        const int64_t at = (x.there ? e : 0) * per_page + head_row + (t & in_page);
        const int64_t key = at + (my_token & 3);
        x.there = x.there && t < count;
        x.k = *reinterpret_cast<const uint4*>(c.codes + key * kCodeRow + 16 * quarter);
        const uint32_t* sc = c.scales + key * (2 * R);
        if constexpr (R == 8) {
            x.ks[0] = sc[2 * quarter];
            x.ks[1] = sc[2 * quarter + 1];
        } else {
            x.ks[0] = sc[R == 4 ? quarter : quarter / 2];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x.v[j] = *reinterpret_cast<const uint32_t*>(c.codes + (at + j) * kCodeRow + 64 + 4 * dw);
            x.vs[j] = c.scales[(at + j) * (2 * R) + R + 8 * dw / G];
        }
        const int left = count - t;
        if (!x.there || (my_token & 3) >= left) x.ks[0] = x.ks[1] = 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (!x.there || j >= left) x.vs[j] = 0u;
        x.there = x.there && (my_token & 3) < left;
    };
    const CodeBits bits;
    const int v_hh = dw / 8, v_i = dw % 8 / 2, v_a = 2 * (dw % 2);
    auto value_at = [&](unsigned char* base, int e) {  // dim e of the dword, the quad's eight bytes
        const int quad = my_quad / 4, u = quad / 8, s = quad % 8 / 4, r = quad % 4;
        const int m = 8 * (v_a + e / 4) + 4 * v_hh + e % 4;
        return reinterpret_cast<uint2*>(base + ((u * 2 + s) * 4 + v_i) * kFrag + value_slot((r & 1) * 32 + m, v_i) +
                                        8 * (r >> 1));
    };
    auto key_at = [&](unsigned char* base, int e) {  // eight dims 32 quarter + 8 e
        const int st = 4 * (quarter & 1) + e;
        return reinterpret_cast<uint4*>(base + (my_token / 32 * 8 + st) * kFrag + (quarter / 2 * 32 + my_token % 32) * 16);
    };
    auto stage_cached = [&](int tile) {
        const uint32_t w[4] = {x.k.x, x.k.y, x.k.z, x.k.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t sc = x.ks[R == 8 ? e / 2 : 0];
            const half2_t delta = as_half2(high_halves(sc, sc));
            const half2_t top7 = as_half2(__builtin_bit_cast(uint32_t, delta) & 0xfff0fff0u);
            half2_t code[4];
            centred_pairs(bits, w[e], code);
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                hi[i] = __builtin_bit_cast(uint32_t, code[i] * top7);
                lo[i] = __builtin_bit_cast(uint32_t, code[i] * (delta - top7));
            }
            *key_at(s_k, e) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *key_at(s_k + PLANE, e) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        if constexpr (R == 8) {
            s_scale[my_token][2 * quarter] = x.ks[0];
            s_scale[my_token][2 * quarter + 1] = x.ks[1];
        } else if (R == 4 || quarter % 2 == 0) {
            s_scale[my_token][R == 4 ? quarter : quarter / 2] = x.ks[0];
        }
        if (quarter == 0) s_bias[my_token] = x.there ? 0.0f : -INFINITY;
        const bool some = __ballot(!x.there) != 0;
        if (lane == 0) s_ragged[wave] = some ? 1 : 0;
        uint32_t out[8][2], low[8][2];  // [dim][token pair]
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const uint32_t v0 = x.v[2 * p], v1 = x.v[2 * p + 1];
            const half2_t delta = as_half2(high_halves(x.vs[2 * p], x.vs[2 * p + 1]));
            const half2_t base = as_half2(low_halves(x.vs[2 * p], x.vs[2 * p + 1]));
#pragma unroll
            for (int hw = 0; hw < 2; ++hw) {
                half2_t code[4];
                centred_pairs(bits, hw ? high_halves(v0, v1) : low_halves(v0, v1), code);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const half2_t c8 = code[i] + half2_t{8.0f16, 8.0f16};
                    if constexpr (C::VT == 1) {
                        out[4 * hw + i][p] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(c8, delta, base));
                    } else {
                        // low + code * delta to 22 bits
                        float y[2], z[2];
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            y[k] = fmaf(static_cast<float>(c8[k]), static_cast<float>(delta[k]), static_cast<float>(base[k]));
                            z[k] = y[k] - static_cast<float>(static_cast<_Float16>(y[k]));
                        }
                        out[4 * hw + i][p] = pack_half2(y[0], y[1]);
                        low[4 * hw + i][p] = pack_half2(z[0], z[1]);
                    }
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            *value_at(s_v, e) = make_uint2(out[e][0], out[e][1]);
            if constexpr (C::VT == 2) *value_at(s_v + PLANE, e) = make_uint2(low[e][0], low[e][1]);
        }
    };

    // weights of a tile's 32 tokens from its logits: lane col's own row, tokens 8
    // (i / 4) + 4 half + i % 4
    auto weights = [&](const f32x16_t& s, float f, float (&p)[16]) {
        float e[16], top = -INFINITY;
        auto exponents = [&] {
#pragma unroll
            for (int i = 0; i < 16; ++i) e[i] = fmaf(s[i], f, -ref);
        };
        exponents();
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, e[i]);
        if (__ballot(top > kTop) != 0) {
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[i] * f);
            mx = fmaxf(mx, lane_xor<32>(mx));
            const float to = fmaxf(mx - kBase, ref), g = exp2_fast(ref - to);
            l *= g;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[i][j] *= g;
            ref = to;
            exponents();
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            p[i] = exp2_fast(e[i]);
            l += p[i];
        }
    };
    auto ld16 = [&](const unsigned char* p) { return *reinterpret_cast<const uint4*>(p); };

    auto fold_cached = [&] {
        const bool ragged = __builtin_amdgcn_readfirstlane(s_ragged[0] | s_ragged[1] | s_ragged[2] | s_ragged[3]) != 0;
#pragma unroll
        for (int u = 0; u < kChunkTile / 32; ++u) {
            f32x16_t s;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = 0.0f;
            const uint32_t pick = half == 0 ? 0x01000100u : 0x03020302u;
#pragma unroll
            for (int n = 0; n < LOWS; ++n) {
                uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                for (int g = 0; g < 4 && g < R; ++g) {
                    const uint32_t sc = s_scale[32 * u + col][4 * n + g];
                    w[g] = __builtin_amdgcn_perm(sc, sc, pick);
                }
                s = mfma_h(make_uint4(w[0], w[1], w[2], w[3]), ql[n], s);
            }
#pragma unroll
            for (int st = 0; st < 8; ++st)
#pragma unroll
                for (int kt = 0; kt < C::KT; ++kt) {
                    const uint4 k = ld16(s_k + kt * PLANE + (u * 8 + st) * kFrag + lane * 16);
#pragma unroll
                    for (int qt = C::QT - 1; qt >= 0; --qt) s = mfma_h(k, q[qt][st], s);
                }
            if (ragged) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const bool out = s_bias[32 * u + 8 * (i / 4) + 4 * half + i % 4] != 0.0f;
                    s[i] = out ? -INFINITY : s[i];
                }
            }
            float p[16];
            weights(s, factor, p);
            // (factor is finite and positive: a token left out keeps -inf)
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                uint32_t w[4], rest[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float p0 = p[8 * st + 2 * j], p1 = p[8 * st + 2 * j + 1];
                    w[j] = pack_half2(p0, p1);
                    rest[j] = pack_half2(p0 - static_cast<float>(as_half2(w[j])[0]), p1 - static_cast<float>(as_half2(w[j])[1]));
                }
                const uint4 ph = make_uint4(w[0], w[1], w[2], w[3]), pl = make_uint4(rest[0], rest[1], rest[2], rest[3]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const unsigned char* at = s_v + ((u * 2 + st) * 4 + i) * kFrag + value_slot(lane, i);
                    const uint4 v = ld16(at);
                    acc[i] = mfma_h(v, ph, acc[i]);
                    if constexpr (C::VT == 2) {
                        acc[i] = mfma_h(v, pl, acc[i]);
                        acc[i] = mfma_h(ld16(at + PLANE), ph, acc[i]);
                    }
                }
            }
        }
    };

    const int cached_tiles = (count + kChunkTile - 1) / kChunkTile;
    if (cached_tiles > 0) load_cached(0);
    for (int tile = 0; tile < cached_tiles; ++tile) {
        __syncthreads();
        stage_cached(tile);
        if (tile + 1 < cached_tiles) load_cached(tile + 1);
        __syncthreads();
        fold_cached();
    }

    // ---- the new tokens, in their own type (fp32: three bf16 terms)
#pragma unroll
    for (int s = 0; s < 8; ++s) {
        if constexpr (C::F32) {
            uint32_t t[8][3];
#pragma unroll
            for (int i = 0; i < 8; ++i) bf16_terms<3>(raw[s].get(i), t[i]);
#pragma unroll
            for (int n = 0; n < 3; ++n)
                q[n][s] = make_uint4(t[0][n] | t[1][n] << 16, t[2][n] | t[3][n] << 16, t[4][n] | t[5][n] << 16,
                                     t[6][n] | t[7][n] << 16);
        } else {
            q[0][s] = raw[s].u;
        }
    }
    if (store_rows) {
#pragma unroll
        for (int n = 0; n < C::QPLANES; ++n)
#pragma unroll
            for (int s = 0; s < 8; ++s) a.queries[((row_tile * C::STORED + C::QT + n) * 8 + s) * kWave + lane] = q[n][s];
    }
    auto mfma_t = [&](const uint4& x, const uint4& y, f32x16_t z) {
        if constexpr (C::F16) return mfma_h(x, y, z);
        else return mfma_b(x, y, z);
    };
    Raw8<T> nk[4], nv[4];
    auto load_new = [&](int tile) {
        const int t0 = tile * kChunkTile, tk = t0 + my_token, tv = t0 + my_quad;
        const T* k_row = static_cast<const T*>(a.k) + b * a.k_bs + h * a.k_hs + static_cast<int64_t>(min(tk, rows - 1)) * a.k_ts;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            nk[e].load(k_row + 32 * quarter + 8 * e);
            if (tk >= rows) nk[e].zero();
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const T* v_row =
                static_cast<const T*>(a.v) + b * a.v_bs + h * a.v_hs + static_cast<int64_t>(min(tv + j, rows - 1)) * a.v_ts;
            nv[j].load(v_row + 8 * dw);
            if (tv + j >= rows) nv[j].zero();
        }
    };
    auto stage_new = [&] {
        bool odd = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) odd = odd || odd_values<T>(nv[j]);
        const bool some = __ballot(odd) != 0;
        if (lane == 0) s_ragged[wave] = some ? 1 : 0;
        if constexpr (C::F32) {
            bool odd_key = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) odd_key = odd_key || odd_values<T>(nk[e]);
            const bool any = __ballot(odd_key) != 0;
            if (lane == 0) s_odd_keys[wave] = any ? 1 : 0;
        }
        if (some) {
#pragma unroll
            for (int j = 0; j < 4; ++j) clear_odd<T>(nv[j]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (C::F32) {
                uint32_t t[8][3];
#pragma unroll
                for (int i = 0; i < 8; ++i) bf16_terms<3>(nk[e].get(i), t[i]);
#pragma unroll
                for (int n = 0; n < 3; ++n)
                    *key_at(s_k + n * PLANE, e) = make_uint4(t[0][n] | t[1][n] << 16, t[2][n] | t[3][n] << 16,
                                                             t[4][n] | t[5][n] << 16, t[6][n] | t[7][n] << 16);
            } else {
                *key_at(s_k, e) = nk[e].u;
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (C::F32) {
                uint32_t t[4][3];
#pragma unroll
                for (int j = 0; j < 4; ++j) bf16_terms<3>(nv[j].get(e), t[j]);
#pragma unroll
                for (int n = 0; n < 3; ++n)
                    *value_at(s_nv + n * PLANE, e) = make_uint2(t[0][n] | t[1][n] << 16, t[2][n] | t[3][n] << 16);
            } else {
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint4& u = nv[j].u;
                    w[j] = e < 2 ? u.x : e < 4 ? u.y : e < 6 ? u.z : u.w;
                }
                *value_at(s_nv, e) = e & 1 ? make_uint2(high_halves(w[0], w[1]), high_halves(w[2], w[3]))
                                           : make_uint2(low_halves(w[0], w[1]), low_halves(w[2], w[3]));
            }
        }
    };
    // Infinite and NaN values: times a weight of zero they would reach rows that do
    // not see their token, so the products take them as zero, and their dims of the
    // rows that do see it get them here.
    auto add_odd = [&](int tile) {
        const int first = tile * kChunkTile;
#pragma unroll 1
        for (int t = first; t < min(first + kChunkTile, rows); ++t) {
            const T* v_row = static_cast<const T*>(a.v) + b * a.v_bs + h * a.v_hs + static_cast<int64_t>(t) * a.v_ts + 64 * half;
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
            const T* k_row = static_cast<const T*>(a.k) + b * a.k_bs + h * a.k_hs + static_cast<int64_t>(first + t) * a.k_ts + 64 * half;
            float dot = 0.0f;
            bool odd = false;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                Raw8<T> k;
                k.load(k_row + 8 * i);
                odd = odd || odd_values<T>(k);
#pragma unroll
                for (int j = 0; j < 8; ++j) dot = fmaf(raw[i].get(j), k.get(j), dot);
            }
            if (__ballot(odd) == 0) continue;
            dot += lane_xor<32>(dot);
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = 8 * (i / 4) + 4 * half + i % 4 == t ? dot : s[i];
        }
    };
    auto fold_new = [&](int tile) {
#pragma unroll
        for (int u = 0; u < kChunkTile / 32; ++u) {
            f32x16_t s;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
            for (int st = 0; st < 8; ++st) {
                uint4 k[C::NT];
#pragma unroll
                for (int n = 0; n < C::NT; ++n) k[n] = ld16(s_k + n * PLANE + (u * 8 + st) * kFrag + lane * 16);
                // terms of at most 2^-16 of the largest first
#pragma unroll
                for (int n = C::NT - 1; n >= 0; --n)
#pragma unroll
                    for (int m = n; m >= 0; --m) s = mfma_t(k[m], q[n - m][st], s);
            }
            if constexpr (C::F32)
                if (__builtin_amdgcn_readfirstlane(s_odd_keys[0] | s_odd_keys[1] | s_odd_keys[2] | s_odd_keys[3]) != 0)
                    odd_logits(tile * kChunkTile + 32 * u, s);
            const int t0 = tile * kChunkTile + 32 * u + 4 * half;
            // (tokens behind the chunk's last are ahead of every row)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = t0 + 8 * (i / 4) + i % 4 <= t_row ? s[i] : -INFINITY;
            float p[16];
            weights(s, kScaleHigh, p);
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                uint4 pw[C::PT];
                uint32_t t[8][C::PT];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float y = p[8 * st + j];
                    if constexpr (C::F16) {
                        const _Float16 high = static_cast<_Float16>(y), low = static_cast<_Float16>(y - static_cast<float>(high));
                        t[j][0] = __builtin_bit_cast(uint16_t, high);
                        t[j][1] = __builtin_bit_cast(uint16_t, low);
                    } else {
                        bf16_terms<C::PT>(y, t[j]);
                    }
                }
#pragma unroll
                for (int n = 0; n < C::PT; ++n)
                    pw[n] = make_uint4(t[0][n] | t[1][n] << 16, t[2][n] | t[3][n] << 16, t[4][n] | t[5][n] << 16,
                                       t[6][n] | t[7][n] << 16);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const unsigned char* at = s_nv + ((u * 2 + st) * 4 + i) * kFrag + value_slot(lane, i);
#pragma unroll
                    for (int n = 0; n < C::NT; ++n) {
                        const uint4 v = ld16(at + n * PLANE);
#pragma unroll
                        for (int m = 0; m < C::PT; ++m)
                            if (n + m < 3) acc[i] = mfma_t(v, pw[m], acc[i]);
                    }
                }
            }
        }
    };
    const int new_tiles = (seen + kChunkTile - 1) / kChunkTile;
    if (new_tiles > 0) load_new(0);
    for (int tile = 0; tile < new_tiles; ++tile) {
        __syncthreads();
        stage_new();
        if (tile + 1 < new_tiles) load_new(tile + 1);
        __syncthreads();
        fold_new(tile);
        if (__builtin_amdgcn_readfirstlane(s_ragged[0] | s_ragged[1] | s_ragged[2] | s_ragged[3]) != 0) add_odd(tile);
    }

    l += lane_xor<32>(l);
    if (live_row) {
        // dims 64 half + 16 i + j
        T* const out = static_cast<T*>(a.out) + b * a.o_bs + head * a.o_hs + static_cast<int64_t>(t_row) * a.o_ts + 64 * half;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 16; j += 2) store2<T>(out + 16 * i + j, acc[i][j] / l, acc[i][j + 1] / l);
    }
    // (rows past the last one weigh nothing)
    if (store_rows && half == 0) a.lse[row_tile * 32 + col] = live_row ? ref + __log2f(l) : INFINITY;
}

// The attention weights of 32 tokens of a KV head a wave, from the logits once
// more and the rows' sums: keys stay in registers as two fp16 terms (fp32's 22
// bits), every row's operands pass once.
template <typename T, int G>
__global__ __launch_bounds__(256) void chunk_weights_kernel(PagedChunk a, PagedView c, int64_t max_tokens) {
    using C = ChunkTypes<T>;
    constexpr int R = 128 / G;
    const int b = blockIdx.z, h = blockIdx.y;
    const int lane = threadIdx.x & (kWave - 1), col = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int group = a.q_heads / c.kv_heads;
    const int rows = static_cast<int>(a.tokens ? clamp_count(a.tokens[b], a.rows) : a.rows);
    const int count = static_cast<int>(clamp_count(c.counts[b], min(c.width << c.page_log2, max_tokens)));
    const int cached_tiles = (count + 31) / 32, tile = blockIdx.x * 4 + wave;
    const bool cached = tile < cached_tiles;
    const int t0 = 32 * (cached ? tile : tile - cached_tiles);
    if (rows == 0 || (!cached && t0 >= rows)) return;
    const int64_t all = static_cast<int64_t>(rows) * group;
    const int64_t base = (static_cast<int64_t>(b) * c.kv_heads + h) * a.row_tiles;
    const int token = t0 + col;
    uint4 k[C::F32 ? 3 : 2][8];
    bool there = true, odd = false;
    if (cached) {
        const int32_t e = token < count ? c.table[b * c.width + (token >> c.page_log2)] : -1;
        there = static_cast<uint32_t>(e) < static_cast<uint32_t>(c.pages);
        const int64_t at = (there ? e : 0) * (static_cast<int64_t>(c.kv_heads) << c.page_log2) +
                           (static_cast<int64_t>(h) << c.page_log2) + (token & ((1 << c.page_log2) - 1));
        const uint4* codes = reinterpret_cast<const uint4*>(c.codes + at * kCodeRow + 32 * half);
        const uint4 w0 = codes[0], w1 = codes[1];
        const uint32_t w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            const uint32_t sc = c.scales[at * (2 * R) + (64 * half + 8 * s) / G];
            float code[8], x[8], y[8];
            codes8(w[s], code);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = fmaf(code[i], f16_hi(sc), f16_lo(sc));
                y[i] = x[i] - static_cast<float>(static_cast<_Float16>(x[i]));
            }
            k[0][s] = make_uint4(pack_half2(x[0], x[4]), pack_half2(x[1], x[5]), pack_half2(x[2], x[6]), pack_half2(x[3], x[7]));
            k[1][s] = make_uint4(pack_half2(y[0], y[4]), pack_half2(y[1], y[5]), pack_half2(y[2], y[6]), pack_half2(y[3], y[7]));
        }
    } else {
        const T* k_row = static_cast<const T*>(a.k) + b * a.k_bs + h * a.k_hs + static_cast<int64_t>(min(token, rows - 1)) * a.k_ts;
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            Raw8<T> raw;
            raw.load(k_row + 64 * half + 8 * s);
            if constexpr (C::F32) {
                odd = odd || odd_values<T>(raw);
                uint32_t t[8][3];
#pragma unroll
                for (int i = 0; i < 8; ++i) bf16_terms<3>(raw.get(i), t[i]);
#pragma unroll
                for (int n = 0; n < 3; ++n)
                    k[n][s] = make_uint4(t[0][n] | t[1][n] << 16, t[2][n] | t[3][n] << 16, t[4][n] | t[5][n] << 16,
                                         t[6][n] | t[7][n] << 16);
            } else {
                k[0][s] = raw.u;
            }
        }
    }
    // (the parts of an infinite fp32 key's products are no sum: its logit is minus
    // infinity or makes the row NaN)
    if constexpr (C::F32) odd = odd || lane_xor<32>(odd ? 1.0f : 0.0f) != 0.0f;
    float sum = 0.0f;
    const int64_t first_row = cached ? 0 : static_cast<int64_t>(t0) * group;
    const int64_t own_first = cached ? 0 : static_cast<int64_t>(token) * group;  // the first row that sees the token
    for (int64_t r0 = first_row / 32 * 32; r0 < all; r0 += 32) {
        const uint4* q = a.queries + (base + r0 / 32) * (C::STORED * 8 * kWave) + lane;
        f32x16_t s;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.0f;
        if (cached) {
#pragma unroll
            for (int st = 0; st < 8; ++st)
#pragma unroll
                for (int qt = C::QT - 1; qt >= 0; --qt) {
                    const uint4 x = q[(qt * 8 + st) * kWave];
                    s = mfma_h(x, k[1][st], s);
                    s = mfma_h(x, k[0][st], s);
                }
        } else {
#pragma unroll
            for (int st = 0; st < 8; ++st) {
                uint4 x[C::QPLANES];
#pragma unroll
                for (int n = 0; n < C::QPLANES; ++n) x[n] = q[((C::QT + n) * 8 + st) * kWave];
#pragma unroll
                for (int n = C::QPLANES - 1; n >= 0; --n)
#pragma unroll
                    for (int m = n; m >= 0; --m) {
                        if constexpr (C::F16) s = mfma_h(x[m], k[n - m][st], s);
                        else s = mfma_b(x[m], k[n - m][st], s);
                    }
            }
        }
        const float4* lse = reinterpret_cast<const float4*>(a.lse + (base * 32 + r0) + 4 * half);
        const float4* factors = reinterpret_cast<const float4*>(a.factors + (base * 32 + r0) + 4 * half);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 off = lse[2 * i];
            float4 f = make_float4(kScaleHigh, kScaleHigh, kScaleHigh, kScaleHigh);
            if (cached) f = factors[2 * i];
            const int64_t r = r0 + 8 * i + 4 * half;
            if constexpr (C::F32)
                if (odd)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[4 * i + j] = -INFINITY;
            sum += r >= own_first ? exp2_fast(fmaf(s[4 * i], f.x, -off.x)) : 0.0f;
            sum += r + 1 >= own_first ? exp2_fast(fmaf(s[4 * i + 1], f.y, -off.y)) : 0.0f;
            sum += r + 2 >= own_first ? exp2_fast(fmaf(s[4 * i + 2], f.z, -off.z)) : 0.0f;
            sum += r + 3 >= own_first ? exp2_fast(fmaf(s[4 * i + 3], f.w, -off.w)) : 0.0f;
        }
    }
    sum += lane_xor<32>(sum);
    const int64_t at = cached ? token : static_cast<int64_t>(count) + token;
    if (half == 0 && there && (cached || token < rows) && at < a.weight_stride)
        a.weights[(static_cast<int64_t>(b) * c.kv_heads + h) * a.weight_stride + at] += sum;
}

// Rows behind a sequence's last one, cleared.
template <typename T>
__global__ __launch_bounds__(256) void chunk_clear_kernel(PagedChunk a) {
    const int b = blockIdx.y, head = blockIdx.x;
    const int64_t rows = clamp_count(a.tokens[b], a.rows);
    for (int64_t i = rows * 16 + threadIdx.x; i < a.rows * 16; i += 256) {
        T* p = static_cast<T*>(a.out) + b * a.o_bs + head * a.o_hs + (i / 16) * a.o_ts + 8 * (i % 16);
        for (int j = 0; j < static_cast<int>(sizeof(T)) / 2; ++j)
            reinterpret_cast<uint4*>(p)[j] = make_uint4(0u, 0u, 0u, 0u);
    }
}

template <typename T, int G>
hipError_t launch_chunk_t(const PagedChunk& a, const PagedView& c, int64_t max_tokens, hipStream_t stream) {
    const int64_t tiles = (a.rows * (a.q_heads / c.kv_heads) + kChunkRows - 1) / kChunkRows;
    hipLaunchKernelGGL((paged_chunk_kernel<T, G>), dim3(static_cast<unsigned>(tiles), c.kv_heads, c.batch), dim3(kChunkThreads), 0, stream, a, c,
                       max_tokens);
    if (a.weights) {
        const int64_t most = min(max_tokens, c.width << c.page_log2);
        const unsigned blocks = static_cast<unsigned>(((most + 31) / 32 + (a.rows + 31) / 32 + 3) / 4);
        hipLaunchKernelGGL((chunk_weights_kernel<T, G>), dim3(blocks, c.kv_heads, c.batch), dim3(256), 0, stream, a, c,
                           max_tokens);
    }
    if (a.fill && a.tokens)
        hipLaunchKernelGGL(chunk_clear_kernel<T>, dim3(a.q_heads, c.batch), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace

// (whole workgroups of the first pass)
int64_t paged_chunk_row_tiles(int64_t rows, int64_t group) {
    return (rows * group + kChunkRows - 1) / kChunkRows * kChunkWaves;
}

int64_t paged_chunk_stored(int dtype) {
    return dtype == POPKV_DTYPE_F32 ? ChunkTypes<float>::STORED
           : dtype == POPKV_DTYPE_F16 ? ChunkTypes<f16_t>::STORED : ChunkTypes<bf16_t>::STORED;
}

hipError_t launch_paged_chunk(const PagedChunk& a, const PagedView& c, int64_t max_tokens, int dtype, int dim_group,
                              hipStream_t stream) {
#define POPKV_CALL(T, G) launch_chunk_t<T, G>(a, c, max_tokens, stream)
    POPKV_PAGED_T(POPKV_CALL)
#undef POPKV_CALL
}

}  // namespace popkv
