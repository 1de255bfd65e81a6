// matrix_tile.h -- the matrix-core building blocks of the feature decoder:
// element types, fragments and their products.
//
// A fragment is what one lane gives one operand of a 16 x 16 product: 16
// consecutive bytes of a row, VEC elements of the summed index.  Lane l holds
// row l % 16 and the VEC elements that begin at VEC (l / 16), so a fragment
// spans KB = 4 VEC of the summed index (16 in float32, 32 in 16 bits).  Both
// operands name the summed index in the same order, so its order inside a
// fragment is free: float32 takes its four products of depth four one element
// at a time.  The product's lane l holds column l % 16 (the second operand's
// row) and rows 4 (l / 16) .. + 3 (the first's).
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace gsx {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;

// The three element types of the decoder's tensors (gsx_dtype).  Sums are
// float32 in all of them.
struct F32 {
    using T = float;
    static constexpr int VEC = 4;
    static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
        const f32x4 fa = __builtin_bit_cast(f32x4, a), fb = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[i], fb[i], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ float up(T v) { return v; }
    static __device__ __forceinline__ T down(float v) { return v; }
    // a small whole number in an element's place, told apart by its bits
    static __device__ __forceinline__ T tag(int k) { return __uint_as_float((uint32_t)k); }
    static __device__ __forceinline__ bool is_tag(T v, int k) {
        return __float_as_uint(v) == (uint32_t)k;
    }
};
using f32x2 = __attribute__((ext_vector_type(2))) float;
using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;

struct BF16 {
    using T = uint16_t;
    static constexpr int VEC = 8;
    static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ float up(T v) { return __uint_as_float((uint32_t)v << 16); }
    static __device__ __forceinline__ T down(float v) {
        return __builtin_bit_cast(uint16_t, (__bf16)v);
    }
    static __device__ __forceinline__ uint32_t pair(float lo, float hi) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
    }
    static __device__ __forceinline__ T tag(int k) { return (T)k; }
    static __device__ __forceinline__ bool is_tag(T v, int k) { return v == (T)k; }
};
struct F16 {
    using T = uint16_t;
    static constexpr int VEC = 8;
    static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                      __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ float up(T v) {
        return (float)__builtin_bit_cast(_Float16, v);
    }
    static __device__ __forceinline__ T down(float v) {
        return __builtin_bit_cast(uint16_t, (_Float16)v);
    }
    static __device__ __forceinline__ uint32_t pair(float lo, float hi) {
        return (uint32_t)down(lo) | (uint32_t)down(hi) << 16;
    }
    static __device__ __forceinline__ T tag(int k) { return (T)k; }
    static __device__ __forceinline__ bool is_tag(T v, int k) { return v == (T)k; }
};

}  // namespace gsx
