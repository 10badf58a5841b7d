// Device pieces shared by the kernels of the paged 4-bit K/V cache
// (pages.hip, paged_dense.hip, paged_indexed.hip): where a token's codes and scales lie.
//
// One layer's pool: codes [pages, KVH, P, 2, 64] bytes -- a token's K row and
// V row side by side, 128 bytes, one L2 line, so a gathered token costs one
// line and a streamed page is contiguous per head -- and scales [pages, KVH,
// P, 2, R] dwords, (low, delta) as two fp16 in each, R = 128 / G.  Dword j of
// a row holds dims 8j .. 8j + 7, nibble i dim 8j + i.  A value is
// low + code * delta.
#pragma once

#include "device_common.h"
#include "kernels.h"

namespace popkv {
namespace {

constexpr int kCodeRow = 128;   // bytes of a token's codes, K then V
constexpr int kPageTile = 32;   // every page holds a whole number of 32-token tiles

__device__ __forceinline__ int64_t clamp_count(int64_t n, int64_t most) {
    return n < 0 ? 0 : n > most ? most : n;
}

__device__ __forceinline__ float f16_lo(uint32_t w) { return bits_f16(w & 0xffffu); }
__device__ __forceinline__ float f16_hi(uint32_t w) { return bits_f16(w >> 16); }

// Two neighbouring elements of a 16-bit type.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    if constexpr (Elem<T>::kDtype == POPKV_DTYPE_F16) return f16_rne(x) | static_cast<uint32_t>(f16_rne(y)) << 16;
    else return bf16_rne(x) | static_cast<uint32_t>(bf16_rne(y)) << 16;
}

// Sixteen bytes that pass once and need no place in the caches behind the
// streams of a large cache.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x4 load_once(const void* p) {
    return __builtin_nontemporal_load(static_cast<const u32x4*>(p));
}
__device__ __forceinline__ void store_once(void* p, u32x4 x) {
    __builtin_nontemporal_store(x, static_cast<u32x4*>(p));
}

// The eight codes of a dword as floats (v_cvt_f32_ubyte of each nibble pair).
__device__ __forceinline__ void codes8(uint32_t w, float* c) {
    const uint32_t e = w & 0x0f0f0f0fu, o = (w >> 4) & 0x0f0f0f0fu;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        c[2 * i] = static_cast<float>((e >> (8 * i)) & 0xffu);
        c[2 * i + 1] = static_cast<float>((o >> (8 * i)) & 0xffu);
    }
}

}  // namespace
}  // namespace popkv
