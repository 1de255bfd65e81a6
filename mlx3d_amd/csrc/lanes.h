// lanes.h -- reductions over groups of a wave's lanes, and their order in shared memory.
#pragma once

#include <hip/hip_runtime.h>

namespace gsx {

// Sum or maximum over the G lanes of a group (a power of two, aligned): cross-lane
// moves inside rows of 16, then swaps of rows and halves.
template <int CTRL>
__device__ __forceinline__ float lane_move(float v) {
    return __uint_as_float(
        __builtin_amdgcn_update_dpp(0u, __float_as_uint(v), CTRL, 0xF, 0xF, true));
}
struct Add {
    static __device__ __forceinline__ float of(float a, float b) { return a + b; }
};
struct Max {
    static __device__ __forceinline__ float of(float a, float b) { return fmaxf(a, b); }
};
template <int G, class Op>
__device__ __forceinline__ float group_reduce(float v) {
    if constexpr (G >= 2) v = Op::of(v, lane_move<0xB1>(v));   // quad_perm 1 0 3 2
    if constexpr (G >= 4) v = Op::of(v, lane_move<0x4E>(v));   // quad_perm 2 3 0 1
    if constexpr (G >= 8) v = Op::of(v, lane_move<0x141>(v));  // row_half_mirror
    if constexpr (G >= 16) v = Op::of(v, lane_move<0x140>(v)); // row_mirror
    if constexpr (G >= 32) {
        const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v),
                                                        false, false);
        v = Op::of(__uint_as_float(p[0]), __uint_as_float(p[1]));
    }
    if constexpr (G >= 64) {
        const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v),
                                                        false, false);
        v = Op::of(__uint_as_float(p[0]), __uint_as_float(p[1]));
    }
    return v;
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
    return group_reduce<G, Add>(v);
}
template <int G>
__device__ __forceinline__ float group_max(float v) {
    return group_reduce<G, Max>(v);
}

// Orders a wave's own accesses to shared memory (they are executed in order).
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

}  // namespace gsx
