// Device pieces shared by the attention kernels of the paged 4-bit K/V cache
// (paged_dense.hip, paged_indexed.hip; paged_chunk.h takes the scale and the
// codes).  The first two split a row's tokens among
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

// The pairs of biased_pairs as c - 8.
__device__ __forceinline__ void centred_pairs(const CodeBits& k, uint32_t w, half2_t (&out)[4]) {
    const half2_t k1032 = {1032.0f16, 1032.0f16}, k16th = {0.0625f16, 0.0625f16}, k72 = {-72.0f16, -72.0f16};
    uint32_t b[4];
    biased_pairs(k, w, b);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        out[i] = i & 1 ? __builtin_elementwise_fma(as_half2(b[i]), k16th, k72) : as_half2(b[i]) - k1032;
}

// The pairs of biased_pairs as c, and as low + c * delta.
__device__ __forceinline__ void code_pairs(const CodeBits& k, uint32_t w, half2_t (&out)[4]) {
    const half2_t k1024 = {1024.0f16, 1024.0f16}, k16th = {0.0625f16, 0.0625f16}, k64 = {-64.0f16, -64.0f16};
    uint32_t b[4];
    biased_pairs(k, w, b);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        out[i] = i & 1 ? __builtin_elementwise_fma(as_half2(b[i]), k16th, k64) : as_half2(b[i]) - k1024;
}
__device__ __forceinline__ void dequantise_pairs(const CodeBits& k, uint32_t w, half2_t delta, half2_t low,
                                                 uint32_t (&out)[4]) {
    half2_t code[4];
    code_pairs(k, w, code);
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(code[i], delta, low));
}

// ---- the merge --------------------------------------------------------------

// Two neighbouring floats of a state (8-byte aligned), as ld_f32<true> and
// st_f32<true>.
__device__ __forceinline__ float2 ld_pair(const float* p) {
    uint64_t* at = reinterpret_cast<uint64_t*>(const_cast<float*>(p));
    return __builtin_bit_cast(float2, __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}
__device__ __forceinline__ void st_pair(float* p, float x, float y) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), __builtin_bit_cast(uint64_t, make_float2(x, y)),
                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Two neighbouring elements.
template <typename T>
__device__ __forceinline__ float2 load2(const T* p) {
    if constexpr (sizeof(T) == 4) {
        return *reinterpret_cast<const float2*>(p);
    } else {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
        if constexpr (Elem<T>::kDtype == POPKV_DTYPE_F16) return make_float2(f16_lo(w), f16_hi(w));
        else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
}
template <typename T>
__device__ __forceinline__ void store2(T* p, float x, float y) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(p) = make_float2(x, y);
    else *reinterpret_cast<uint32_t*>(p) = pack2<T>(x, y);
}

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
