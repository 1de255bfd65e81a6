// dropout.hip -- y = residual + [kept] x / (1 - p), the kept elements told by a
// counter-based generator, so that no mask is stored: the gradient is the same
// call on the incoming gradient.
//
// Element i (in row-major order) has a 32-bit number u_i and is kept where
// u_i >= round(p 2^32).  The numbers come from Philox4x32 with ten rounds (Salmon,
// Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) with
// the key `seed` and the counter (block, offset): the eight half-words of the block
// i / 8 are the upper halves of eight elements' numbers, those of the block
// 2^63 + i / 8 the lower ones.  A lower half matters only where the upper one equals
// the threshold's, once in 65 536 elements: a block's ten rounds serve eight elements
// and not four.
//
// Bound by memory: 118 million bfloat16 79 us (6.0 TB/s, 4 bytes an element), 59 million
// float32 80 us, 124 on top of a residual (5.7).  Beside it the rounds keep the vector
// units busy for 61 % of the first; with both blocks formed for all elements, and
// elements loaded one by one, it took 238.
#include <hip/hip_runtime.h>

#include <cmath>

#include "gsx.h"
#include "gsx_device.h"
#include "matrix_tile.h"
#include "row_pieces.h"

using namespace gsx;

namespace {

constexpr int kThreads = 256;
constexpr int kBlock = 8;  // elements of a generator block, of a thread

struct Drop {
    const void *x, *residual;
    void* y;
    int64_t n;
    uint32_t key0, key1;
    int64_t offset;
    const int64_t* offset_at;  // on the device, in place of offset; or NULL
    uint32_t upper, lower;     // the threshold's halves; upper may be 2^16: none is kept
    uint32_t limit;            // what a half-word has to reach
    float scale;
};

__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
    return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);
}
__device__ __forceinline__ void philox(uint32_t* c, uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p = (uint64_t)c[0] * 0xD2511F53u, q = (uint64_t)c[2] * 0xCD9E8D57u;
        c[0] = xor3((uint32_t)(q >> 32), c[1], k0);
        c[1] = (uint32_t)q;
        c[2] = xor3((uint32_t)(p >> 32), c[3], k1);
        c[3] = (uint32_t)p;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
}

// The block's eight half-words, two a word, of which element e is kept where its own is
// at least q.limit.  Half-words equal to the threshold's upper half, if a lower half
// matters, are replaced by what the lower one decides; a wave gets there once in 128
// times.
__device__ __forceinline__ void halves(const Drop& q, uint64_t block, int64_t offset,
                                       uint32_t* hi) {
    const uint32_t c[4] = {(uint32_t)block, (uint32_t)(block >> 32), (uint32_t)offset,
                           (uint32_t)((uint64_t)offset >> 32)};
#pragma unroll
    for (int i = 0; i < 4; ++i) hi[i] = c[i];
    philox(hi, q.key0, q.key1);
    if (q.lower == 0) return;
    // a half of t that is zero sets its top bit in `equal` (and so may halves above it)
    uint32_t equal = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t t = hi[i] ^ (q.upper | q.upper << 16);
        equal |= (t - 0x00010001u) & ~t & 0x80008000u;
    }
    if (equal) {
        uint32_t lo[4] = {c[0], c[1] | 0x80000000u, c[2], c[3]};
        philox(lo, q.key0, q.key1);
#pragma unroll
        for (int e = 0; e < kBlock; ++e) {
            const int shift = 16 * (e % 2);
            const uint32_t part = 0xffffu << shift;
            if ((hi[e / 2] & part) == q.upper << shift)
                hi[e / 2] = (lo[e / 2] >> shift & 0xffffu) >= q.lower ? hi[e / 2] | part
                                                                      : hi[e / 2] & ~part;
        }
    }
}
__device__ __forceinline__ bool kept(const Drop& q, const uint32_t* hi, int e) {
    return (e % 2 ? hi[e / 2] >> 16 : hi[e / 2] & 0xffffu) >= q.limit;
}

// One generator block a thread: eight elements.
template <class E, bool RES>
__global__ __launch_bounds__(kThreads) void k_dropout(const Drop q) {
    using T = typename E::T;
    using P = Piece<E, E::VEC>;
    constexpr int N = kBlock / E::VEC;  // vectors of a block
    const int64_t block = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const int64_t first = block * kBlock;
    if (first >= q.n) return;
    const T* x = (const T*)q.x + first;
    const T* r = (const T*)q.residual + first;
    T* y = (T*)q.y + first;
    const bool whole = first + kBlock <= q.n;
    typename P::Raw rx[N], rr[N];
    if (whole) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            rx[k] = P::load(x + k * E::VEC);
            if (RES) rr[k] = P::load(r + k * E::VEC);
        }
    }
    uint32_t hi[4];
    halves(q, (uint64_t)block, q.offset_at ? *q.offset_at : q.offset, hi);
    if (whole) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            float v[E::VEC], base[E::VEC] = {};
            P::up(rx[k], v);
            if (RES) P::up(rr[k], base);
#pragma unroll
            for (int e = 0; e < E::VEC; ++e)
                v[e] = kept(q, hi, k * E::VEC + e) ? fmaf(v[e], q.scale, base[e]) : base[e];
            P::store(y + k * E::VEC, P::down(v));
        }
    } else {
        const int left = (int)(q.n - first);
#pragma unroll
        for (int e = 0; e < kBlock - 1; ++e)
            if (e < left) {
                const float base = RES ? E::up(r[e]) : 0.f;
                y[e] = E::down(kept(q, hi, e) ? fmaf(E::up(x[e]), q.scale, base) : base);
            }
    }
}

template <class E>
int run(const Drop& q, hipStream_t st) {
    // below 2^23 workgroups for the 2^34 elements that are taken at most
    const int64_t blocks = (q.n + kBlock * kThreads - 1) / (kBlock * kThreads);
    if (q.residual)
        hipLaunchKernelGGL((k_dropout<E, true>), dim3((unsigned)blocks), dim3(kThreads), 0, st, q);
    else
        hipLaunchKernelGGL((k_dropout<E, false>), dim3((unsigned)blocks), dim3(kThreads), 0, st, q);
    GSX_LAUNCH_CHECK();
    return GSX_OK;
}

}  // namespace

extern "C" int gsx_dropout(int32_t dtype, int64_t n, double p, uint64_t seed, int64_t offset,
                           const int64_t* offset_at, const void* x, const void* residual, void* y,
                           void* stream) {
    if (dtype != GSX_F32 && dtype != GSX_BF16 && dtype != GSX_F16) return GSX_ERR_INVALID;
    if (n < 0 || !(p >= 0.0 && p <= 1.0) || offset < 0) return GSX_ERR_INVALID;
    if (n > (int64_t)1 << 34) return GSX_ERR_TOO_LARGE;
    const uintptr_t size = dtype == GSX_F32 ? 4 : 2;
    if ((uintptr_t)x % size || (uintptr_t)residual % size || (uintptr_t)y % size ||
        (uintptr_t)offset_at % 8)
        return GSX_ERR_INVALID;
    if (n == 0) return GSX_OK;
    if (!x || !y) return GSX_ERR_INVALID;
    // p 2^32 to the nearest, ties to even, as Python's round
    const uint64_t threshold = (uint64_t)std::nearbyint(p * 4294967296.0);
    Drop q{};
    q.x = x;
    q.residual = residual;
    q.y = y;
    q.n = n;
    q.key0 = (uint32_t)seed;
    q.key1 = (uint32_t)(seed >> 32);
    q.offset = offset;
    q.offset_at = offset_at;
    q.upper = (uint32_t)(threshold >> 16);
    q.lower = (uint32_t)(threshold & 0xffffu);
    // kept: above the upper half, and at it where nothing is below; replaced half-words
    // are 0 or 2^16 - 1, so the limit lies between them
    q.limit = q.lower == 0 ? q.upper : q.upper > 1 ? q.upper : 1;
    q.scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.f;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == GSX_F32) return run<F32>(q, st);
    if (dtype == GSX_BF16) return run<BF16>(q, st);
    return run<F16>(q, st);
}
