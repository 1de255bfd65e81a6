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

#include <type_traits>

namespace gsx {

// Keeps the compiler from computing what depends on v ahead of this place (and
// holding it in registers through a loop).
__device__ __forceinline__ int here(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

using f32x4 = __attribute__((ext_vector_type(4))) float;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
__device__ __forceinline__ u32x4 here(u32x4 v) {
    asm volatile("" : "+v"(v));
    return v;
}

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

// What the narrow kernels multiply: a float32 operand as three bf16 pieces (the
// first cut off, the others rounded to nearest: 8 + 8 + 8 bits hold the 24
// exactly) and six of their nine products; the rest is below 2^-22 of a product.
// 16-bit operands are taken as they are.  The matrix units take 16 bits at eight
// times the float32 rate (1248 against 154 TFLOP/s in large products), so six
// products cost less than half of one in float32.
//
// Cutting holds every finite number, where rounding would make infinities of those
// next to the largest; it takes as many instructions.  Pieces end at bf16's
// smallest number, so of an operand below 2^-110 up to 2^-126 is lost.  An
// infinity has no second piece: it gives NaN.
struct Split3 {
    u32x4 p[3];
};
__device__ __forceinline__ void split_pair(float a, float b, uint32_t* p0, uint32_t* p1,
                                           uint32_t* p2) {
    const uint32_t ha = __float_as_uint(a) & 0xffff0000u, hb = __float_as_uint(b) & 0xffff0000u;
    *p0 = ha >> 16 | hb;
    a -= __uint_as_float(ha);
    b -= __uint_as_float(hb);
    *p1 = BF16::pair(a, b);
    a -= __uint_as_float(*p1 << 16);
    b -= __uint_as_float(*p1 & 0xffff0000u);
    *p2 = BF16::pair(a, b);
}
__device__ __forceinline__ Split3 split(const float* x) {
    Split3 s;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t w[3];
        split_pair(x[2 * i], x[2 * i + 1], &w[0], &w[1], &w[2]);
#pragma unroll
        for (int k = 0; k < 3; ++k) s.p[k][i] = w[k];
    }
    return s;
}

// An element type with its operand form: eight elements of a row on a lane.
template <class E>
struct Wide {
    static constexpr int PIECES = 1;
    using Raw = u32x4;
    struct Frag {
        u32x4 p[1];
    };
    static __device__ __forceinline__ Frag frag(const Raw& r) { return Frag{{r}}; }
    static __device__ __forceinline__ f32x4 mma(const Frag& a, const Frag& b, f32x4 c) {
        return E::mma(a.p[0], b.p[0], c);
    }
    // zero elements from number n on
    static __device__ __forceinline__ void cut(Raw& r, int n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (2 * i + 1 >= n) r[i] &= 0xffffu;
            if (2 * i >= n) r[i] = 0;
        }
    }
};
template <>
struct Wide<F32> {
    static constexpr int PIECES = 3;
    struct Raw {
        float v[8];
    };
    using Frag = Split3;
    static __device__ __forceinline__ Frag frag(const Raw& r) { return split(r.v); }
    static __device__ __forceinline__ void four(const float* x, uint2* w) {
        split_pair(x[0], x[1], &w[0].x, &w[1].x, &w[2].x);
        split_pair(x[2], x[3], &w[0].y, &w[1].y, &w[2].y);
    }
    static __device__ __forceinline__ f32x4 mma(const Frag& a, const Frag& b, f32x4 c) {
        c = BF16::mma(a.p[2], b.p[0], c);
        c = BF16::mma(a.p[0], b.p[2], c);
        c = BF16::mma(a.p[1], b.p[1], c);
        c = BF16::mma(a.p[1], b.p[0], c);
        c = BF16::mma(a.p[0], b.p[1], c);
        return BF16::mma(a.p[0], b.p[0], c);
    }
    static __device__ __forceinline__ void cut(Raw& r, int n) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i >= n) r.v[i] = 0.f;
    }
};

// The second products, whose one operand is formed on the chip in float32 (`Mid`:
// hidden channels and their gradients) and whose other one (`Other`) is the
// tensors': float32 as above.  In 16 bits Mid is two bf16 pieces, sixteen bits or
// more in float32's range, so that nothing is rounded to the tensors' type but the
// outputs; the other operand is itself in bf16, and two bf16 pieces (11 = 8 + 3
// bits, exact) in float16, where the product of the second pieces, below 2^-16 of
// one, is left out.  That takes two products for one in bf16 and three in float16.
// An infinity has no second piece here either: it gives NaN.
struct Split2 {
    u32x4 p[2];
};
// CUT: the first piece is cut off, which no finite number survives as an infinity;
// else it is rounded, for a smaller second one (float16 products end far below)
template <bool CUT>
__device__ __forceinline__ void split_two(float a, float b, uint32_t* p0, uint32_t* p1) {
    uint32_t ha, hb;
    if constexpr (CUT) {
        ha = __float_as_uint(a) & 0xffff0000u;
        hb = __float_as_uint(b) & 0xffff0000u;
        *p0 = ha >> 16 | hb;
    } else {
        *p0 = BF16::pair(a, b);
        ha = *p0 << 16;
        hb = *p0 & 0xffff0000u;
    }
    *p1 = BF16::pair(a - __uint_as_float(ha), b - __uint_as_float(hb));
}

template <class E>
struct Second {  // BF16, F16
    static constexpr bool HALF = std::is_same_v<E, F16>;
    static constexpr int MID = 2, OTHER = HALF ? 2 : 1;
    using M = BF16;  // the products' type
    using Mid = Split2;
    struct Other {
        u32x4 p[OTHER];
    };
    static __device__ __forceinline__ Mid mid(const float* x) {
        Mid m;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t w[2];
            split_two<!HALF>(x[2 * i], x[2 * i + 1], &w[0], &w[1]);
            m.p[0][i] = w[0];
            m.p[1][i] = w[1];
        }
        return m;
    }
    // four elements of each piece
    static __device__ __forceinline__ void four(const float* x, uint2* w) {
        split_two<!HALF>(x[0], x[1], &w[0].x, &w[1].x);
        split_two<!HALF>(x[2], x[3], &w[0].y, &w[1].y);
    }
    static __device__ __forceinline__ Other other(const u32x4& r) {
        Other o;
        if constexpr (HALF) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t w[2];
                split_two<false>(E::up((uint16_t)r[i]), E::up((uint16_t)(r[i] >> 16)), &w[0],
                                 &w[1]);
                o.p[0][i] = w[0];
                o.p[1][i] = w[1];
            }
        } else {
            o.p[0] = r;
        }
        return o;
    }
    static __device__ __forceinline__ f32x4 mma(const Other& o, const Mid& m, f32x4 c) {
        if constexpr (HALF) c = BF16::mma(o.p[1], m.p[0], c);
        c = BF16::mma(o.p[0], m.p[1], c);
        return BF16::mma(o.p[0], m.p[0], c);
    }
};
template <>
struct Second<F32> {
    static constexpr int MID = 3, OTHER = 3;
    using M = F32;  // of the tiled products
    using Mid = Split3;
    using Other = Split3;
    static __device__ __forceinline__ Mid mid(const float* x) { return split(x); }
    static __device__ __forceinline__ void four(const float* x, uint2* w) {
        Wide<F32>::four(x, w);
    }
    static __device__ __forceinline__ Other other(const Wide<F32>::Raw& r) { return split(r.v); }
    static __device__ __forceinline__ f32x4 mma(const Other& o, const Mid& m, f32x4 c) {
        return Wide<F32>::mma(o, m, c);
    }
};

// Eight elements from p on, of which the first n (at least one) belong to the
// row; zeros for the others.  With `after` rows behind this one, eight or more,
// what follows the row's end is the tensor's too (a row takes an element at
// least) and may be read and dropped.
template <class E>
__device__ __forceinline__ typename Wide<E>::Raw load8(const typename E::T* p, int n, int after) {
    using T = typename E::T;
    typename Wide<E>::Raw r;
    if (n >= 8 || after >= 8) {
        __builtin_memcpy(&r, p, sizeof(r));
        if (n < 8) Wide<E>::cut(r, n);
    } else {
        T v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : (T)0;
        __builtin_memcpy(&r, v, sizeof(r));
    }
    return r;
}

}  // namespace gsx
