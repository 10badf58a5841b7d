// Device pieces shared by the attention kernels of the paged 4-bit K/V cache
// (paged_dense.hip, paged_indexed.hip).  Both split a row's tokens among
// workgroups that each leave an online-softmax state (m, l, acc[128]), base-2
// exponents; the last workgroup of a row merges them in the same launch (the
// hand-off rule stands in attention_common.h).  The current token's K/V, not
// cached yet, enter the merge at full precision.
#pragma once

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

}  // namespace
}  // namespace popkv

// Calls CALL(T, G) of an element type and a group size, in a function that returns its result.
#define POPKV_PAGED_G(CALL, T)       \
    switch (dim_group) {             \
        case 16: return CALL(T, 16); \
        case 32: return CALL(T, 32); \
        default: return CALL(T, 64); \
    }
#define POPKV_PAGED_T(CALL)                              \
    switch (dtype) {                                     \
        case POPKV_DTYPE_F32: POPKV_PAGED_G(CALL, float) \
        case POPKV_DTYPE_F16: POPKV_PAGED_G(CALL, f16_t) \
        default: POPKV_PAGED_G(CALL, bf16_t)             \
    }
