// row_pieces.h -- rows of any width and alignment in pieces of 16 bytes.
//
// A row of at least VEC elements is cut into ceil(width / VEC) pieces; the last one
// ends with the row and so overlaps the one before it where VEC does not divide the
// width.  Pieces are loaded and stored whole from any element's address (the
// hardware takes unaligned vectors); what two pieces share is read twice, and written
// twice with the same value.  Shorter rows go element by element.
#pragma once

#include <hip/hip_runtime.h>

#include "matrix_tile.h"

namespace gsx {

// 16 bytes at an element's address
using u32x4_at2 = __attribute__((ext_vector_type(4), aligned(2))) uint32_t;
using u32x4_at4 = __attribute__((ext_vector_type(4), aligned(4))) uint32_t;

// V consecutive elements of a row on a lane: VEC (16 bytes) or 1.
template <class E, int V>
struct Piece {
    static_assert(V == E::VEC, "16 bytes, or one element");
    using T = typename E::T;
    using Raw = u32x4;
    static __device__ __forceinline__ Raw load(const T* p) {
        if constexpr (sizeof(T) == 4) return *(const u32x4_at4*)p;
        else return *(const u32x4_at2*)p;
    }
    static __device__ __forceinline__ void store(T* p, Raw r) {
        if constexpr (sizeof(T) == 4) *(u32x4_at4*)p = r;
        else *(u32x4_at2*)p = r;
    }
    static __device__ __forceinline__ void up(Raw r, float* v) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                v[i] = __uint_as_float(r[i]);
            } else {
                v[2 * i] = E::up((T)(r[i] & 0xffffu));
                v[2 * i + 1] = E::up((T)(r[i] >> 16));
            }
        }
    }
    static __device__ __forceinline__ Raw down(const float* v) {
        Raw r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) r[i] = __float_as_uint(v[i]);
            else r[i] = E::pair(v[2 * i], v[2 * i + 1]);
        }
        return r;
    }
};
template <class E>
struct Piece<E, 1> {
    using T = typename E::T;
    using Raw = T;
    static __device__ __forceinline__ Raw load(const T* p) { return *p; }
    static __device__ __forceinline__ void store(T* p, Raw r) { *p = r; }
    static __device__ __forceinline__ void up(Raw r, float* v) { v[0] = E::up(r); }
    static __device__ __forceinline__ Raw down(const float* v) { return E::down(v[0]); }
};

// V floats at any float's address.
template <int V>
__device__ __forceinline__ void load_floats(const float* p, float* v) {
    if constexpr (V == 1) {
        v[0] = *p;
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            const u32x4 r = *(const u32x4_at4*)(p + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[i + k] = __uint_as_float(r[k]);
        }
    }
}
template <int V>
__device__ __forceinline__ void store_floats(float* p, const float* v) {
    if constexpr (V == 1) {
        *p = v[0];
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            u32x4 r;
#pragma unroll
            for (int k = 0; k < 4; ++k) r[k] = __float_as_uint(v[i + k]);
            *(u32x4_at4*)(p + i) = r;
        }
    }
}

}  // namespace gsx
