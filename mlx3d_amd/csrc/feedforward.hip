// feedforward.hip -- the gated feed-forward block that decodes rows of
// features, and its gradient.
//
//   g = x Wg^T,  u = x Wu^T,  h = act(g) u,  y = h Wd^T
//   dh = dy Wd,  du = dh act(g),  dg = dh u act'(g)
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dWd = dy^T h
//
// x (rows, d_in), Wg and Wu (hidden, d_in), Wd (d_out, hidden), row-major.
// Products and their sums are float32 on the matrix units.  What they multiply is
// held to float32 where the tensors are float32 (three bf16 pieces in the narrow
// kernels, the float32 instructions in the tiled ones) and to sixteen bits, two bf16
// pieces, for h, dg and du of 16-bit tensors (matrix_tile.h), so that 16-bit outputs
// are rounded once, at the end, and h may be what float16 cannot hold.
//
// Two paths.  Narrow widths (a decoder over pixels) run the whole block in one
// kernel, forward and backward: h, dg and du never leave the chip.  Any other
// sizes run tiled products with the elementwise work in their epilogue: g and u
// share one pass over x, so only h leaves the first kernel.  Neither keeps g and
// u for the backward: forming them again costs a pass over x against writing and
// reading two arrays of hidden width.  Weight gradients sum over the rows in
// splits or workgroups, whose float32 sums are added up in a fixed order, so the
// same inputs give the same bits.
#include <hip/hip_runtime.h>

#include <cmath>
#include <type_traits>

#include "gsx.h"
#include "gsx_device.h"
#include "matrix_tile.h"

using namespace gsx;

namespace {

constexpr int kThreads = 256;
constexpr int kBM = 128;  // rows of the first operand in a tile
constexpr int kBN = 64;   // rows of the second

// ---------------------------------------------------------- activations --

// act(g) and act'(g); NaN and infinities as the formulas give them.
//
// sigmoid from the hardware's power of two and reciprocal: exp(-g)'s relative
// error, |g| 2^-24 and one unit, comes into s times 1 - s, so act(g) is within
// two units of max(|g|, 1) 2^-24 for every g.  Phi(g): in 16 bits Phi(-a) is
// exp(-a^2 / 2) t P(t) with t = 1 / (1 + 0.3 a), P of degree seven fitted to the
// scaled complementary error function for the least relative error (2^-21 as
// evaluated), so the far tail keeps the type's bits, and the power serves the slope
// too; in float32, where that is too coarse for a slope near zero, from erff.
template <class E>
constexpr bool kExact = sizeof(typename E::T) == 4;

template <bool GELU, bool EXACT>
__device__ __forceinline__ float activate(bool silu, float g, float& slope) {
    if constexpr (GELU) {
        const float e = __builtin_amdgcn_exp2f(g * g * -0.72134752044448170f);
        float cdf;
        if constexpr (EXACT) {
            cdf = 0.5f * (1.0f + erff(g * 0.70710678118654752f));
        } else {
            const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(g), 0.3f, 1.0f));
            float p = fmaf(t, 0.03567432f, -0.15720116f);
            p = fmaf(t, p, 0.20635013f);
            p = fmaf(t, p, -0.05368054f);
            p = fmaf(t, p, 0.12855998f);
            p = fmaf(t, p, 0.099914f);
            p = fmaf(t, p, 0.12075388f);
            p = fmaf(t, p, 0.11962931f);
            const float tail = p * t * e;  // Phi(-|g|)
            cdf = g < 0.f ? tail : 1.0f - tail;
        }
        slope = fmaf(g * 0.39894228040143268f, e, cdf);
        return g * cdf;
    } else {
        const float e = __builtin_amdgcn_exp2f(g * -1.4426950408889634f);
        const float s = __builtin_amdgcn_rcpf(1.0f + e);
        const float a = s * (silu ? g : 1.0f);
        slope = fmaf(a, 1.0f - s, silu ? s : 0.0f);
        return a;
    }
}
template <bool EXACT>
__device__ __forceinline__ float activate_any(int act, float g, float& slope) {
    return act == GSX_ACT_GELU ? activate<true, EXACT>(false, g, slope)
                               : activate<false, EXACT>(act == GSX_ACT_SILU, g, slope);
}

// ---------------------------------------------------------------- tiles --

// One operand: element (row, k) is p[row * ld + k] where KC (the summed index
// is contiguous), else p[k * ld + row].
struct Operand {
    const void* p;
    int64_t ld;
    int rows;
    const void* lo = nullptr;  // a second piece of every element, where there is one
};

// Rows in shared memory, SLOTS 16-byte slots a row, the slots turned
// by the row so that no access meets a bank twice.  What the accesses ask for
// (measured with a counter of conflicts): a 16-byte read serves lanes 0-3, 12-15,
// 20-27 of a half wave in one clock, then the others, so rows 0-3 and 12-15 of
// one slot with rows 4-11 of the next; a transposing read 32 lanes, rows r .. r + 3
// and r + 8 .. r + 11 of two slots; a 16-byte write eight lanes, over half the
// banks.
template <int SLOTS>
__device__ __forceinline__ int tile_slot(int row, int slot) {
    const int b0 = row & 1, b1 = row >> 1 & 1, b2 = row >> 2 & 1, b3 = row >> 3 & 1;
    if constexpr (SLOTS == 4) return row * 4 + (slot ^ ((b2 ^ b3) << 1 | (b3 ^ b1)));
    if constexpr (SLOTS == 8) return row * 8 + (slot ^ (b1 << 1 | b3 << 2));
    return row * SLOTS + (slot ^ (b0 << 1 | b1 << 2 | b3 << 3));
}
// The operand whose rows are 16 of a tile's columns, block `block` of them, and whose
// summed index are 32 of the tile's rows (16-bit elements).  A lane's two places
// differ from the ones that turned_base() gives for block 0 by what the turned slots
// change: bits of the address, flipped.
template <int SLOTS>
__device__ __forceinline__ int turned_base(int lane) {
    const int s = lane & 15, row = 8 * (lane >> 4) + (s >> 2), col = 4 * (s & 3);
    return tile_slot<SLOTS>(row, col >> 3) * 16 + 8 * ((col >> 2) & 1);
}
template <int SLOTS>
__device__ __forceinline__ u32x4 read_turned(const u32x4* tile, int block, int base) {
    using v4 = __attribute__((ext_vector_type(4))) short;
    typedef __attribute__((address_space(3))) v4* lds_v4;
    union {
        v4 h[2];
        u32x4 v;
    } r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {  // four rows on: with four slots a row they turn by two
        const int flip = SLOTS == 4 ? (block ^ i) * 32 : block * 32;
        char* at = (char*)tile + (base ^ flip) + i * 64 * SLOTS;
        r.h[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)at);
    }
    return r.v;
}

// ROWS rows times two fragments' depth of one operand, kept in fragment order
// (row block, fragment, lane), a lane's 16 bytes at a time.  Rows of odd length
// are read unaligned, which global memory allows at the price of a sector.
//
// Where the rows are contiguous instead, 16-bit operands are staged as they lie
// and turned by the reads; float32 ones are turned in registers by patches.
//
// The lanes of a fragment lie so that what a wave reads, and eight lanes of what
// it stores, meet each bank once: where the summed index is contiguous eight lanes
// load and store one row's 128 bytes, and the row's low bits are turned by the
// piece; else its lanes are a few rows apart, and the four low bits of the row
// change places (bits 2, 3, 0, 1), odd row blocks half a turn on.
template <class E, int ROWS, bool KC>
struct Stage {
    static constexpr bool TURNED = !KC && E::VEC == 8;
    static constexpr int SLOTS = ROWS / 8;  // of one summed index, TURNED
    using T = typename E::T;
    static constexpr int VEC = E::VEC;
    static constexpr int STEP = 8 * VEC;  // depth of a stage
    static constexpr int N = ROWS / 32;   // 16-byte pieces of a thread
    u32x4 r[N];

    static __device__ __forceinline__ int slot(int row, int piece) {
        const int in = row & 15;
        const int turned = KC ? in ^ piece : ((in & 3) << 2 | in >> 2) ^ (row >> 4 & 1) << 2;
        return ((row >> 4) * 2 + (piece >> 2)) * 64 + (piece & 3) * 16 + turned;
    }
    // the fragment f of row block b, on this lane
    static __device__ __forceinline__ u32x4 read(const u32x4* lds, int b, int f, int lane) {
        if constexpr (TURNED)
            return read_turned<SLOTS>(lds + f * 32 * SLOTS, b, turned_base<SLOTS>(lane));
        return lds[slot(b * 16 + (lane & 15), f * 4 + (lane >> 4))];
    }

    // A stage of the summed index [k0, k1).  Not the last one: no bounds, so that
    // the loads of several stages can be in flight and each waited for alone.
    // Rows past the operand's then repeat its last one, or hold what follows it:
    // they only reach outputs that are not stored.
    __device__ __forceinline__ void load_inner(const Operand& o, int row0, int64_t k0) {
        const T* p = (const T*)o.p;
        const int t = threadIdx.x;
        if constexpr (KC) {
            const int64_t k = k0 + (t & 7) * VEC;
#pragma unroll
            for (int n = 0; n < N; ++n) {
                int row = row0 + (t >> 3) + 32 * n;
                row = row < o.rows ? row : o.rows - 1;
                __builtin_memcpy(&r[n], p + (int64_t)row * o.ld + k, 16);
            }
        } else if constexpr (TURNED) {
            int row = row0 + t % SLOTS * 8;
            row = row < o.rows ? row : o.rows - 1;
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int64_t k = k0 + t / SLOTS + n * (kThreads / SLOTS);
                __builtin_memcpy(&r[n], p + k * o.ld + row, 16);
            }
        } else {
            load(o, row0, k0, k0 + STEP);
        }
    }

    __device__ __forceinline__ void load(const Operand& o, int row0, int64_t k0, int64_t k1) {
        const T* p = (const T*)o.p;
        const int t = threadIdx.x;
        if constexpr (KC) {
            const int64_t k = k0 + (t & 7) * VEC;
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int row = row0 + (t >> 3) + 32 * n;
                const T* at = p + (int64_t)row * o.ld + k;
                if (row < o.rows && k + VEC <= k1) {
                    __builtin_memcpy(&r[n], at, 16);
                } else {
                    T v[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; ++i)
                        v[i] = (row < o.rows && k + i < k1) ? at[i] : (T)0;
                    __builtin_memcpy(&r[n], v, 16);
                }
            }
        } else if constexpr (TURNED) {
            const int row = row0 + t % SLOTS * 8;
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int64_t k = k0 + t / SLOTS + n * (kThreads / SLOTS);
                const T* at = p + k * o.ld + row;
                if (k < k1 && row + 8 <= o.rows) {
                    __builtin_memcpy(&r[n], at, 16);
                } else {
                    T v[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = (k < k1 && row + i < o.rows) ? at[i] : (T)0;
                    __builtin_memcpy(&r[n], v, 16);
                }
            }
        } else {
            // a patch of N rows times VEC of the summed index, turned in registers
            const int row = row0 + (t & 31) * N;
            const int64_t k = k0 + (int64_t)(t >> 5) * VEC;
            T v[VEC][N];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const T* at = p + (k + i) * o.ld + row;
                if (k + i < k1 && row + N <= o.rows) {
                    __builtin_memcpy(v[i], at, N * sizeof(T));
                } else {
#pragma unroll
                    for (int n = 0; n < N; ++n)
                        v[i][n] = (k + i < k1 && row + n < o.rows) ? at[n] : (T)0;
                }
            }
#pragma unroll
            for (int n = 0; n < N; ++n) {
                T w[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) w[i] = v[i][n];
                __builtin_memcpy(&r[n], w, 16);
            }
        }
    }

    __device__ __forceinline__ void store(u32x4* lds) const {
        const int t = threadIdx.x;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if constexpr (KC)
                lds[slot((t >> 3) + 32 * n, t & 7)] = r[n];
            else if constexpr (TURNED)
                lds[tile_slot<SLOTS>(t / SLOTS + n * (kThreads / SLOTS), t % SLOTS)] = r[n];
            else
                lds[slot((t & 31) * N + n, t >> 5)] = r[n];
        }
    }
};

// What a wave keeps of a product: 64 x 32 of the tile, as 4 x 2 blocks; lane l
// of block (a, b) holds row 16 a + l % 16 and columns 16 b + 4 (l / 16) .. + 3.
using Acc = f32x4[4][2];

__device__ __forceinline__ void clear(Acc& c) {
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b) c[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
}

// 16-byte slots of shared memory for a workgroup: half of a unit's, so that two
// run on it (y of 8205 x 1365 x 512 f16 81 us, with two stages for one 107), but all
// of it where the registers of two second operands of pieces fill a SIMD with one
// wave (the pair of weight gradients 123, with two workgroups' registers 165).
template <int NB, int PA, int PB>
constexpr bool kAlone = NB == 2 && PA + PB > 2;
template <int NB, int PA, int PB>
constexpr int kTileSlots = (kAlone<NB, PA, PB> ? 160 : 80) * 1024 / 16;

// c0 += A B0^T and (NB == 2) c1 += A B1^T over the summed index [k0, k1), of
// operands of PA and PB pieces whose product of second pieces is left out.  The
// next two stages' loads are in flight while one is multiplied, and shared memory
// holds two stages where two workgroups a unit leave room for them, so one barrier
// each, else one.  What bounds it is the time that a stage's
// loads take to arrive (8205 x 512 x 1365 f16: 420 to 500 TFLOP/s, its second
// products' three counted, against 1200 of an 8192-wide square product): one stage
// ahead and two barriers took 473 us for the training step of one piece instead of
// 343.  Tiles of 128 columns were no faster.
//
// Every stage but the last runs without bounds.  A transposed operand's may read
// up to seven elements past its rows, which the next of the summed index holds if
// the pitch is eight or more; below, every stage is bounded.
template <class E, bool AKC, bool BKC, int NB, int PA = 1, int PB = 1>
__device__ __forceinline__ void multiply(u32x4* lds, const Operand& A, const Operand& B0,
                                         const Operand& B1, int m0, int n0, int64_t k0, int64_t k1,
                                         Acc& c0, Acc& c1) {
    using SA = Stage<E, kBM, AKC>;
    using SB = Stage<E, kBN, BKC>;
    constexpr int STAGE = (PA * kBM + NB * PB * kBN) * 8;
    constexpr bool BOTH = 2 * STAGE <= kTileSlots<NB, PA, PB>;  // stages in shared memory
    SA a[2][PA];
    SB b0[2][PB], b1[2][PB];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int wm = (wave >> 1) * 4, wn = (wave & 1) * 2;  // in blocks of 16
    const int steps = (int)((k1 - k0 + SA::STEP - 1) / SA::STEP);
    const bool inner = (AKC || A.ld >= 8) && (BKC || (B0.ld >= 8 && B1.ld >= 8));
    auto piece = [](const Operand& o, int p) { return p ? Operand{o.lo, o.ld, o.rows} : o; };
    auto load_inner = [&](int step, int i) {
        const int64_t k = k0 + (int64_t)step * SA::STEP;
#pragma unroll
        for (int p = 0; p < PA; ++p) a[i][p].load_inner(piece(A, p), m0, k);
#pragma unroll
        for (int p = 0; p < PB; ++p) {
            b0[i][p].load_inner(piece(B0, p), n0, k);
            if constexpr (NB == 2) b1[i][p].load_inner(piece(B1, p), n0, k);
        }
    };
    auto load = [&](int step, int i) {
        if (step >= steps) return;
        const int64_t k = k0 + (int64_t)step * SA::STEP;
        const int64_t stop = k + SA::STEP < k1 ? k + SA::STEP : k1;
#pragma unroll
        for (int p = 0; p < PA; ++p) a[i][p].load(piece(A, p), m0, k, stop);
#pragma unroll
        for (int p = 0; p < PB; ++p) {
            b0[i][p].load(piece(B0, p), n0, k, stop);
            if constexpr (NB == 2) b1[i][p].load(piece(B1, p), n0, k, stop);
        }
    };
    auto step = [&](int s, int i, auto is_inner) {
        u32x4* la = lds + (BOTH ? i * STAGE : 0);
        u32x4* lb0 = la + PA * kBM * 8;
        if constexpr (!BOTH) __syncthreads();  // the last stage's reads
        u32x4* lb1 = lb0 + PB * kBN * 8;
#pragma unroll
        for (int p = 0; p < PA; ++p) a[i][p].store(la + p * kBM * 8);
#pragma unroll
        for (int p = 0; p < PB; ++p) {
            b0[i][p].store(lb0 + p * kBN * 8);
            if constexpr (NB == 2) b1[i][p].store(lb1 + p * kBN * 8);
        }
        __syncthreads();
        if constexpr (is_inner)
            load_inner(s + 2, i);
        else
            load(s + 2, i);
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            u32x4 fa[PA][4];
#pragma unroll
            for (int p = 0; p < PA; ++p)
#pragma unroll
                for (int i = 0; i < 4; ++i) fa[p][i] = SA::read(la + p * kBM * 8, wm + i, f, lane);
            auto with = [&](const u32x4* lb, Acc& c) {
#pragma unroll
                for (int p = PB - 1; p >= 0; --p) {
                    u32x4 fb[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) fb[j] = SB::read(lb + p * kBN * 8, wn + j, f, lane);
#pragma unroll
                    for (int pa = p ? 0 : PA - 1; pa >= 0; --pa)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int j = 0; j < 2; ++j)
                                c[i][j] = E::mma(fb[j], fa[pa][i], c[i][j]);
                }
            };
            with(lb0, c0);
            if constexpr (NB == 2) with(lb1, c1);
        }
    };
    __syncthreads();  // an earlier product's reads
    int s = 0;
    if (inner && steps > 4) {
        // a loop of its own, so that its waits count on every load being there
        load_inner(0, 0);
        load_inner(1, 1);
        for (; s + 4 < steps; s += 2) {
            step(s, 0, std::true_type{});
            step(s + 1, 1, std::true_type{});
        }
    } else {
        load(0, 0);
        load(1, 1);
    }
    for (; s < steps; s += 2) {
        step(s, 0, std::false_type{});
        if (s + 1 < steps) step(s + 1, 1, std::false_type{});
    }
}

// Four consecutive columns of one row; the row's end cuts them short.
template <class E>
__device__ __forceinline__ void put(typename E::T* p, int64_t ld, int row, int col, int rows,
                                    int cols, f32x4 v) {
    using T = typename E::T;
    if (row >= rows || col >= cols) return;
    T w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = E::down(v[i]);
    T* at = p + (int64_t)row * ld + col;
    if (col + 4 <= cols) {
        __builtin_memcpy(at, w, 4 * sizeof(T));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (col + i < cols) at[i] = w[i];
    }
}

// Four values that are an operand later on: float32 as they are, else two bf16
// pieces, the second `plane` elements behind the first.
template <class E>
__device__ __forceinline__ void put_mid(void* p, int64_t plane, int64_t ld, int row, int col,
                                        int rows, int cols, f32x4 v) {
    if constexpr (std::is_same_v<E, F32>) {
        put<F32>((float*)p, ld, row, col, rows, cols, v);
    } else {
        if (row >= rows || col >= cols) return;
        const float x[4] = {v[0], v[1], v[2], v[3]};
        uint2 w[2];
        Second<E>::four(x, w);
        // whole 16-byte rows: the columns up to the pitch belong to nobody else
#pragma unroll
        for (int i = 0; i < 2; ++i)
            *(uint2*)((uint16_t*)p + i * plane + (int64_t)row * ld + col) = w[i];
    }
}

enum Mode {
    HIDDEN,      // out0 = act(A B0^T) (A B1^T)
    PLAIN,       // out0 = A B0^T
    BWD_HIDDEN,  // g, u as in HIDDEN, dh = A2 B2^T: out0 = dg, out1 = du, out2 = h
    SUM2,        // out0 = A B0^T + A2 B2^T
    WGRAD2,      // out0^T = A B0^T, out1^T = A B1^T over a split of the summed index
    WGRAD        // out0 = A B0^T over a split
};

struct Tile {
    Operand a, b0, b1, a2, b2;
    int64_t k, k2;        // depths
    int m, n;             // rows of A, rows of B
    void* out[3];
    int64_t ldo, plane;   // plane: from a first piece of out to its second
    int act;
    int64_t split_k;      // depth of a split (WGRAD*)
    int64_t split_out;    // floats of a split's partial sums; 0: out itself, in E
    bool add;             // to the partial sums that an earlier stretch of rows left
};

// Pieces of a tiled product's operands: of what was formed on the chip, and of the
// tensors that it meets (float32 takes the float32 instructions, one piece each).
template <class E>
constexpr int kMid = std::is_same_v<E, F32> ? 1 : 2;
template <class E>
constexpr int kOther = std::is_same_v<E, F16> ? 2 : 1;

// A product's pieces, and its shared memory: one stage or two.
template <class E, Mode MODE>
struct TileShape {
    static constexpr bool SECOND = MODE != HIDDEN && MODE != BWD_HIDDEN;
    static constexpr bool GRAD = MODE == WGRAD || MODE == WGRAD2;
    static constexpr int PA = !SECOND ? 1 : GRAD ? kOther<E> : kMid<E>;
    static constexpr int PB = !SECOND ? 1 : GRAD ? kMid<E> : kOther<E>;
    static constexpr int NB = !SECOND || MODE == WGRAD2 ? 2 : 1;
    static constexpr int STAGE = (PA * kBM + NB * PB * kBN) * 8;
    static constexpr int BYTES = (2 * STAGE <= kTileSlots<NB, PA, PB> ? 2 : 1) * STAGE * 16;
    static constexpr int WAVES = kExact<E> || kAlone<NB, PA, PB> ? 1 : 2;  // of a SIMD
};

template <class E, Mode MODE>
__global__ __launch_bounds__(kThreads, (TileShape<E, MODE>::WAVES)) void k_tile(const Tile q) {
    using T = typename E::T;
    using M = typename Second<E>::M;
    using S = TileShape<E, MODE>;
    extern __shared__ u32x4 lds[];
    const int tiles_n = (q.n + kBN - 1) / kBN;
    const uint32_t id = xcd_remap(blockIdx.x, gridDim.x);
    const int m0 = (int)(id / tiles_n) * kBM, n0 = (int)(id % tiles_n) * kBN;
    Acc c0, c1, c2;
    clear(c0);
    if constexpr (MODE == HIDDEN || MODE == BWD_HIDDEN) {
        clear(c1);
        multiply<E, true, true, 2>(lds, q.a, q.b0, q.b1, m0, n0, 0, q.k, c0, c1);
        if constexpr (MODE == BWD_HIDDEN) {
            clear(c2);
            multiply<E, true, false, 1>(lds, q.a2, q.b2, q.b2, m0, n0, 0, q.k2, c2, c2);
        }
    } else if constexpr (MODE == PLAIN) {
        multiply<M, true, true, 1, S::PA, S::PB>(lds, q.a, q.b0, q.b0, m0, n0, 0, q.k, c0, c0);
    } else if constexpr (MODE == SUM2) {
        multiply<M, true, false, 1, S::PA, S::PB>(lds, q.a, q.b0, q.b0, m0, n0, 0, q.k, c0, c0);
        multiply<M, true, false, 1, S::PA, S::PB>(lds, q.a2, q.b2, q.b2, m0, n0, 0, q.k, c0, c0);
    } else {
        const int64_t k0 = blockIdx.y * q.split_k;
        const int64_t k1 = k0 + q.split_k < q.k ? k0 + q.split_k : q.k;
        if constexpr (MODE == WGRAD2) clear(c1);
        multiply<M, false, false, S::NB, S::PA, S::PB>(lds, q.a, q.b0, q.b1, m0, n0, k0, k1, c0,
                                                       c1);
    }
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int row0 = m0 + (wave >> 1) * 64 + (lane & 15);
    const int col0 = n0 + (wave & 1) * 32 + (lane >> 4) * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int row = row0 + 16 * i, col = col0 + 16 * j;
            if constexpr (MODE == WGRAD2) {
                // these gradients lie (B row, A row): lanes run along A's
                if (row >= q.m) continue;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (col + e >= q.n) continue;
                    const int64_t at = (int64_t)(col + e) * q.ldo + row;
                    if (q.split_out) {
                        const int64_t s = blockIdx.y * q.split_out;
                        float* o0 = (float*)q.out[0] + s + at;
                        float* o1 = (float*)q.out[1] + s + at;
                        *o0 = q.add ? *o0 + c0[i][j][e] : c0[i][j][e];
                        *o1 = q.add ? *o1 + c1[i][j][e] : c1[i][j][e];
                    } else {
                        ((T*)q.out[0])[at] = E::down(c0[i][j][e]);
                        ((T*)q.out[1])[at] = E::down(c1[i][j][e]);
                    }
                }
            } else if constexpr (MODE == WGRAD) {
                if (q.split_out) {
                    float* parts = (float*)q.out[0] + blockIdx.y * q.split_out;
                    f32x4 v = c0[i][j];
                    if (q.add && row < q.m) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (col + e < q.n) v[e] += parts[(int64_t)row * q.ldo + col + e];
                    }
                    put<F32>(parts, q.ldo, row, col, q.m, q.n, v);
                } else
                    put<E>((T*)q.out[0], q.ldo, row, col, q.m, q.n, c0[i][j]);
            } else if constexpr (MODE == HIDDEN) {
                f32x4 h;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float slope;
                    h[e] = activate_any<kExact<E>>(q.act, c0[i][j][e], slope) * c1[i][j][e];
                }
                put_mid<E>(q.out[0], q.plane, q.ldo, row, col, q.m, q.n, h);
            } else if constexpr (MODE == BWD_HIDDEN) {
                f32x4 dg, du, h;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float slope;
                    const float a = activate_any<kExact<E>>(q.act, c0[i][j][e], slope);
                    const float u = c1[i][j][e], dh = c2[i][j][e];
                    h[e] = a * u;
                    du[e] = dh * a;
                    dg[e] = dh * u * slope;
                }
                put_mid<E>(q.out[0], q.plane, q.ldo, row, col, q.m, q.n, dg);
                put_mid<E>(q.out[1], q.plane, q.ldo, row, col, q.m, q.n, du);
                put_mid<E>(q.out[2], q.plane, q.ldo, row, col, q.m, q.n, h);
            } else {
                put<E>((T*)q.out[0], q.ldo, row, col, q.m, q.n, c0[i][j]);
            }
        }
}

// The two bf16 pieces of float16 rows, in planes of `pitch` elements a row.  A few
// us beside the products that read them: splitting in their stages would be done
// again by every tile.
__global__ __launch_bounds__(kThreads) void k_pieces(const uint16_t* x, int64_t ld, int64_t rows,
                                                     int cols, int pitch, uint16_t* out) {
    const int pairs = (cols + 1) / 2;
    const int64_t n = rows * pairs, step = (int64_t)gridDim.x * kThreads, plane = rows * pitch;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += step) {
        const int64_t row = i / pairs;
        const int col = (int)(i % pairs) * 2;
        const uint16_t* at = x + row * ld + col;
        uint32_t w[2];
        split_two<false>(F16::up(at[0]), col + 1 < cols ? F16::up(at[1]) : 0.f, &w[0], &w[1]);
        uint32_t* to = (uint32_t*)(out + row * pitch + col);
        to[0] = w[0];
        to[plane / 2] = w[1];
    }
}

// Adds up the splits' partial sums in their order.  5 us for 512 x 1365 f16.
template <class E>
__global__ __launch_bounds__(kThreads) void k_join(const float* parts, int64_t n, int splits,
                                                   typename E::T* out) {
    const int64_t step = (int64_t)gridDim.x * kThreads;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += step) {
        float s = 0.f;
        for (int k = 0; k < splits; ++k) s += parts[k * n + i];
        out[i] = E::down(s);
    }
}

__global__ __launch_bounds__(kThreads) void k_zero_bytes(uint8_t* p, int64_t n) {
    const int64_t step = (int64_t)gridDim.x * kThreads;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += step) p[i] = 0;
}

// --------------------------------------------------------------- narrow --

// The whole block in one kernel, for narrow widths and many rows: h stays in
// registers, so x is read and y written once and nothing else moves.  Each wave
// takes 32 rows through all of it.
//
// 921 600 rows of 32 -> 128 -> 64 float32: 177 to 190 us, 1.9 TB/s; bound by the matrix
// units, whose six bf16 products for one float32 run at 1.02 PFLOP/s, 82 % of what
// a large product reaches (the float32 instructions would take 196 us at best).
// 2 073 600 rows of 32 -> 96 -> 48 bf16: 122 us, 2.7 TB/s; bound by the vector
// units (activations, h's two pieces), the copy of its bytes would take 69; with h
// rounded to bf16 it took 104.
//
// Products run with the weights first, so that a lane holds one row (its column
// of the product) and consecutive channels: g^T and u^T come out with channels
// 4 (l / 16) .. + 3 of 16 on a lane, and two such blocks are the eight channels
// that the next product's operand wants there, if the blocks' rows are taken in
// the order 8 (r / 4) + r % 4 (+ 4 in the second).  h never crosses lanes.
//
// The weights lie in shared memory in operand order, cut into chunks of 32
// hidden channels; as many chunks at a time as fit (all of them: staged once).
constexpr int kNarrowThreads = 512;
constexpr int kNarrowRows = 32;                   // rows of a wave
constexpr int64_t kNarrowLds = 144 * 1024;

template <class E>
struct Narrow {
    const typename E::T *x, *wg, *wu, *wd;
    typename E::T* y;
    int64_t ldx, rows;
    int d_in, hidden, d_out, act;
    int chunks, resident;  // chunks of 32 hidden channels, how many are staged at a time
};

// A chunk in shared memory: the fragments of Wg and Wu with their pieces, then those
// of Wd, 64 lanes' 16 bytes each.
template <class E, int KD, int OB>
struct FwdShape {
    static constexpr int PC = Wide<E>::PIECES, PO = Second<E>::OTHER;
    static constexpr int CHUNK = 4 * KD * PC + OB * PO;
    static __device__ __forceinline__ int in(int c, int frag, int p) {
        return (c * CHUNK + frag * PC + p) * 64;
    }
    static __device__ __forceinline__ int out(int c, int o, int p) {
        return (c * CHUNK + 4 * KD * PC + o * PO + p) * 64;
    }
};

// Stages `count` chunks from number c0 on: for each chunk, fragments of Wg (two
// blocks of 16 channels times KD), of Wu, then OB of Wd, each with its pieces.
template <class E, int KD, int OB>
__device__ __forceinline__ void stage_weights(const Narrow<E>& q, u32x4* lds, int c0, int count) {
    using Wd = Wide<E>;
    using S2 = Second<E>;
    using L = FwdShape<E, KD, OB>;
    constexpr int FRAGS = 4 * KD + OB;
    for (int i = threadIdx.x; i < count * FRAGS * 64; i += kNarrowThreads) {
        const int lane = i & 63, frag = (i >> 6) % FRAGS, c = (i >> 6) / FRAGS;
        const int r = lane & 15, k8 = (lane >> 4) * 8;
        typename Wd::Raw raw{};
        if (frag < 4 * KD) {
            const int kd = frag % KD, which = frag / KD;  // Wg a, Wg b, Wu a, Wu b
            const int f = (c0 + c) * 32 + 8 * (r >> 2) + (r & 3) + 4 * (which & 1);
            const int k = kd * 32 + k8;
            if (f < q.hidden && k < q.d_in)
                raw = load8<E>((which < 2 ? q.wg : q.wu) + (int64_t)f * q.d_in + k, q.d_in - k,
                               q.hidden - 1 - f);
            const typename Wd::Frag w = Wd::frag(raw);
#pragma unroll
            for (int p = 0; p < Wd::PIECES; ++p) lds[L::in(c, frag, p) + lane] = w.p[p];
        } else {
            const int o = (frag - 4 * KD) * 16 + r, k = (c0 + c) * 32 + k8;
            if (o < q.d_out && k < q.hidden)
                raw = load8<E>(q.wd + (int64_t)o * q.hidden + k, q.hidden - k, q.d_out - 1 - o);
            const typename S2::Other w = S2::other(raw);
#pragma unroll
            for (int p = 0; p < S2::OTHER; ++p)
                lds[L::out(c, frag - 4 * KD, p) + lane] = w.p[p];
        }
    }
}

template <class E, int KD, int OB, bool GELU>
__global__ __launch_bounds__(kNarrowThreads) void k_narrow_fwd(const Narrow<E> q) {
    using T = typename E::T;
    using W = Wide<E>;
    using S2 = Second<E>;
    using L = FwdShape<E, KD, OB>;
    constexpr int kWaves = kNarrowThreads / 64, R = kNarrowRows / 16;
    extern __shared__ u32x4 smem[];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int col = lane & 15, k8 = (lane >> 4) * 8;
    const bool once = q.resident >= q.chunks, silu = q.act == GSX_ACT_SILU;
    auto weights = [&](int c, int frag) {
        typename W::Frag w;
#pragma unroll
        for (int p = 0; p < W::PIECES; ++p) w.p[p] = smem[L::in(c, frag, p) + lane];
        return w;
    };
    if (once) {
        stage_weights<E, KD, OB>(q, smem, 0, q.chunks);
        __syncthreads();
    }
    const int64_t tile_rows = kWaves * kNarrowRows;
    for (int64_t base = blockIdx.x * tile_rows; base < q.rows; base += gridDim.x * tile_rows) {
        const int64_t row0 = base + wave * kNarrowRows + col;
        typename W::Frag x[R][KD];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int kd = 0; kd < KD; ++kd) {
                const int64_t row = row0 + 16 * r;
                const int k = kd * 32 + k8;
                typename W::Raw raw{};
                if (row < q.rows && k < q.d_in)
                    raw = load8<E>(q.x + row * q.ldx + k, q.d_in - k, (int)(q.rows - 1 - row));
                x[r][kd] = W::frag(raw);
            }
        f32x4 y[OB][R];
#pragma unroll
        for (int o = 0; o < OB; ++o)
#pragma unroll
            for (int r = 0; r < R; ++r) y[o][r] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int c0 = 0; c0 < q.chunks; c0 += q.resident) {
            const int count = q.chunks - c0 < q.resident ? q.chunks - c0 : q.resident;
            if (!once) {
                __syncthreads();  // the last chunks are read
                stage_weights<E, KD, OB>(q, smem, c0, count);
                __syncthreads();
            }
            for (int c = 0; c < count; ++c) {
                f32x4 g[2][R], u[2][R];
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int r = 0; r < R; ++r) g[b][r] = u[b][r] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kd = 0; kd < KD; ++kd)
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const auto wg = weights(c, b * KD + kd), wu = weights(c, (2 + b) * KD + kd);
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            g[b][r] = W::mma(wg, x[r][kd], g[b][r]);
                            u[b][r] = W::mma(wu, x[r][kd], u[b][r]);
                        }
                    }
                typename S2::Mid h[R];
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    float v[8], slope;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        v[i] = activate<GELU, kExact<E>>(silu, g[i >> 2][r][i & 3], slope) *
                               u[i >> 2][r][i & 3];
                    h[r] = S2::mid(v);
                }
#pragma unroll
                for (int o = 0; o < OB; ++o)
                    if (o * 16 < q.d_out) {
                        typename S2::Other wd;
#pragma unroll
                        for (int p = 0; p < S2::OTHER; ++p) wd.p[p] = smem[L::out(c, o, p) + lane];
#pragma unroll
                        for (int r = 0; r < R; ++r) y[o][r] = S2::mma(wd, h[r], y[o][r]);
                    }
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t row = row0 + 16 * r;
            if (row >= q.rows) continue;
#pragma unroll
            for (int o = 0; o < OB; ++o) {
                const int at = o * 16 + (lane >> 4) * 4;
                T w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = E::down(y[o][r][i]);
                T* out = q.y + row * q.d_out + at;
                if (at + 4 <= q.d_out) {
                    __builtin_memcpy(out, w, sizeof(w));
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (at + i < q.d_out) out[i] = w[i];
                }
            }
        }
    }
}

// The whole backward pass in one kernel for narrow widths and many rows.  A pair
// of waves owns 32 hidden channels, 16 each: their rows of Wg and Wu, their
// columns of Wd and the running sums of their weight gradients stay in its
// registers while the workgroup walks tiles of 32 rows.  x and dy are staged
// once for all pairs, g, u and dh are formed again, and dg, du and h go through
// shared memory once: read as they lie they are dx's operand (the pair shares
// dx's channels), read along the rows (a transposing read: 16 lanes turn 4 x 16
// elements) the weight gradients'.  The pairs' parts of dx are added up there
// too.  Two barriers a tile; the next tile's loads are in flight meanwhile.
//
// 921 600 rows of 32 -> 128 -> 64: bf16 213 us, 1.3 TB/s (shared memory, which dg, du
// and h pass in two pieces, and the vector units, 60 % busy; 150 with one
// piece); float32 487 to 546 us (matrix units, the pieces' conversions and shared
// memory; the mean as clocks rise).
// One wave for the 32 channels instead of a pair needs twice the registers; with half
// the waves a SIMD the training step took 414 us instead of 225 (in one piece),
// float32 870 instead of 656.
//
// More than 4 x 32 hidden channels run as groups, each with its part of dx;
// the workgroups' weight gradients and the groups' dx are added up in a fixed
// order afterwards.
constexpr int kBwdPairs = 4;
constexpr int kBwdRows = 32;

template <class E>
struct NarrowBwd {
    using T = typename E::T;
    const T *x, *wg, *wu, *wd, *dy;
    T* dx;            // one group's result, or NULL
    float* dx_parts;  // (groups, rows, d_in), or NULL
    float* parts;     // (workgroups, groups, pairs, halves, sums, 64)
    int64_t ldx, lddy, rows;
    int d_in, hidden, d_out, act;
    bool add;         // to the parts that an earlier stretch of rows left
};

// Rows of float32 sums, written and read along the slots only.
template <int SLOTS>
__device__ __forceinline__ int sum_slot(int row, int slot) {
    return row * SLOTS + (slot ^ (row & (SLOTS - 1)));
}

// A staged tile's planes: the pieces of the first products' operands, and those of
// the second ones where they are others (float16, whose bf16 pieces are formed once
// for all waves).  LATE: of 128 float16 inputs neither shared memory nor registers
// hold the pieces; each wave forms them where it uses them.
template <class E, int KD, int KO>
struct BwdShape {
    static constexpr int PC = Wide<E>::PIECES, PM = Second<E>::MID, PO = Second<E>::OTHER;
    static constexpr bool HALF = std::is_same_v<E, F16>, LATE = HALF && KD == 4;
    static constexpr int AT = HALF && !LATE ? 1 : 0, PLANES = AT ? 3 : PC;
    static constexpr int XS = 4 * KD, YS = 4 * KO;              // slots of a row of x, of dy
    static constexpr int TILE = kBwdRows * (XS + YS) * PLANES;  // 16-byte slots of a staged tile
    static constexpr int GATE = kBwdRows * 4 * PM;              // of a pair's dg, du or h
    static constexpr int SUM = kBwdRows * 8 * KD;               // of a pair's part of dx
    static constexpr int SUMS = 16 * KD + 8 * KO;               // weight gradient registers
    static int64_t lds(int pairs) { return 16 * (2 * TILE + (int64_t)pairs * (3 * GATE + SUM)); }
};

// Waves for a SIMD that the registers leave room for: one workgroup or two.
template <class E, int KD, int KO>
constexpr int bwd_waves() {
    return std::is_same_v<E, BF16> && KD == 1 && KO <= 2 ? 4 : 2;
}

template <class E, int KD, int KO, bool GELU>
__global__ __launch_bounds__(128 * kBwdPairs, (bwd_waves<E, KD, KO>()))
void k_narrow_bwd(const NarrowBwd<E> q) {
    using T = typename E::T;
    using W = Wide<E>;
    using S = BwdShape<E, KD, KO>;
    using S2 = Second<E>;
    using Frag = typename W::Frag;
    using Mid = typename S2::Mid;
    using Other = typename S2::Other;
    constexpr int PC = S::PC, PM = S::PM, R = kBwdRows / 16;
    extern __shared__ u32x4 smem[];
    const int threads = blockDim.x, pairs = threads >> 7;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int pair = wave >> 1, half = wave & 1;
    const bool silu = q.act == GSX_ACT_SILU;
    const int col = lane & 15, quad = lane >> 4, k8 = quad * 8;
    u32x4* tiles = smem;
    u32x4* gates = smem + 2 * S::TILE + pair * 3 * S::GATE;
    u32x4* sums = smem + 2 * S::TILE + pairs * 3 * S::GATE;
    const int f0 = (blockIdx.y * kBwdPairs + pair) * 32;

    // the wave's weights: its 16 channels' rows (operands of x and of dy), and the
    // pair's 32 channels for every other 16 of dx's
    Frag wg[KD], wu[KD], wd[KO];
    using Kept = std::conditional_t<S::LATE, typename W::Raw, Other>;
    Kept wgt[KD], wut[KD];
    {
        auto gather = [&](const T* w, int64_t first, int64_t step, int n) {
            typename W::Raw raw;
            T v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = i < n ? w[first + i * step] : (T)0;
            __builtin_memcpy(&raw, v, sizeof(raw));
            return raw;
        };
        const int f = f0 + 16 * half + col;
        const bool there = f < q.hidden;
#pragma unroll
        for (int kd = 0; kd < KD; ++kd) {
            const int k = kd * 32 + k8;
            typename W::Raw a{}, c{};
            if (there && k < q.d_in) {
                const int64_t at = (int64_t)f * q.d_in + k;
                a = load8<E>(q.wg + at, q.d_in - k, q.hidden - 1 - f);
                c = load8<E>(q.wu + at, q.d_in - k, q.hidden - 1 - f);
            }
            wg[kd] = W::frag(a);
            wu[kd] = W::frag(c);
        }
#pragma unroll
        for (int ko = 0; ko < KO; ++ko) {
            const int o = ko * 32 + k8;
            wd[ko] = W::frag(gather(q.wd, (int64_t)o * q.hidden + f, q.hidden,
                                    there ? q.d_out - o : 0));
        }
#pragma unroll
        for (int j = 0; j < KD; ++j) {
            const int d = 16 * (2 * j + half) + col, f8 = f0 + k8;
            const int n = d < q.d_in ? q.hidden - f8 : 0;
            const auto a = gather(q.wg, (int64_t)f8 * q.d_in + d, q.d_in, n);
            const auto c = gather(q.wu, (int64_t)f8 * q.d_in + d, q.d_in, n);
            if constexpr (S::LATE) {
                wgt[j] = a;
                wut[j] = c;
            } else {
                wgt[j] = S2::other(a);
                wut[j] = S2::other(c);
            }
        }
    }

    // no work is moved over these places where the registers hold what is asked for
    constexpr bool EARLY = PC == 3 && KD == 1;
    auto asked = [] {
        if constexpr (EARLY) __builtin_amdgcn_sched_barrier(0);
    };
    // elsewhere over these: what is in flight would take too many (or, in 16 bits,
    // the registers of the second workgroup that hides the waits)
    auto pause = [] {
        if constexpr (!EARLY) __builtin_amdgcn_sched_barrier(0);
    };

    // staging: pieces of eight elements of x's and dy's rows, HELD of them in a
    // thread's registers one tile ahead
    constexpr int PIECES = kBwdRows * (S::XS + S::YS);
    constexpr int HELD = (PIECES + 128 * kBwdPairs - 1) / (128 * kBwdPairs);
    const int rows = (int)q.rows, step = (int)gridDim.x * kBwdRows;
    struct Piece {
        const T* p;    // in the next tile to be read
        int row, n;    // its row; how many elements the row has from here on
        int slot;      // its place in the staged tile
    };
    const int64_t hop_x = step * q.ldx, hop_y = step * q.lddy;  // from a tile to the next
    auto of_x = [&](int n) { return n < kBwdRows * S::XS; };
    auto piece_of = [&](int n, int row0) {
        const bool x = of_x(n);
        const int i = x ? n : n - kBwdRows * S::XS;
        const int slots = x ? S::XS : S::YS, row = i / slots, k = i % slots * 8;
        Piece m;
        m.row = row0 + row;
        m.p = (x ? q.x : q.dy) + (int64_t)m.row * (x ? q.ldx : q.lddy) + k;
        m.n = (x ? q.d_in : q.d_out) - k;
        m.slot = x ? tile_slot<S::XS>(row, k / 8)
                   : S::PLANES * kBwdRows * S::XS + tile_slot<S::YS>(row, k / 8);
        return m;
    };
    auto fetch = [&](const Piece& m) {
        typename W::Raw raw{};
        if (m.row < rows && m.n > 0) raw = load8<E>(m.p, m.n, rows - 1 - m.row);
        return raw;
    };
    auto settle = [&](u32x4* tile, const Piece& m, bool x, const typename W::Raw& raw) {
        const Frag f = W::frag(raw);
        const int pitch = kBwdRows * (x ? S::XS : S::YS);
#pragma unroll
        for (int p = 0; p < PC; ++p) tile[m.slot + p * pitch] = f.p[p];
        if constexpr (S::AT > 0) {
            const Other o = S2::other(raw);
#pragma unroll
            for (int p = 0; p < S::PO; ++p) tile[m.slot + (S::AT + p) * pitch] = o.p[p];
        }
    };
    Piece mine[HELD];
    typename W::Raw next[HELD];
    auto fetch_all = [&] {
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            const int n = threadIdx.x + i * threads;
            if (n < PIECES) {
                next[i] = fetch(mine[i]);
                mine[i].p += of_x(n) ? hop_x : hop_y;
                mine[i].row += step;
            }
        }
    };
    auto settle_all = [&](u32x4* tile, int row0) {
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            const int n = threadIdx.x + i * threads;
            if (n < PIECES) settle(tile, mine[i], of_x(n), next[i]);
        }
        for (int n = threadIdx.x + HELD * threads; n < PIECES; n += threads) {  // fewer pairs
            const Piece m = piece_of(n, row0);
            settle(tile, m, of_x(n), fetch(m));
        }
    };

    f32x4 sg[2 * KD], su[2 * KD], sd[2 * KO];  // the weight gradients' sums
#pragma unroll
    for (int d = 0; d < 2 * KD; ++d) sg[d] = su[d] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int o = 0; o < 2 * KO; ++o) sd[o] = f32x4{0.f, 0.f, 0.f, 0.f};

    // a lane's places in a tile: the row of the first products' operand (its next four
    // slots: bits flipped), the columns of the second ones'
    const int x_at = tile_slot<S::XS>(col, quad), y_at = tile_slot<S::YS>(col, quad);
    const int turned4 = turned_base<4>(lane);
    const int turned_xs = turned_base<S::XS>(lane), turned_ys = turned_base<S::YS>(lane);
    int row0 = (int)blockIdx.x * kBwdRows;
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (threadIdx.x + i * threads < PIECES) mine[i] = piece_of(threadIdx.x + i * threads, row0);
    fetch_all();
    settle_all(tiles, row0);
    fetch_all();
    __syncthreads();
    for (int turn = 0; row0 < rows; row0 += step, turn ^= 1) {
        const u32x4* xt = tiles + turn * S::TILE;
        const u32x4* yt = xt + S::PLANES * kBwdRows * S::XS;
        // where the registers allow it, a phase asks shared memory for all that it
        // needs first, and its products begin with the first answer
        Frag fx[R][KD], fy[R][KO];
        auto ask = [&](int r) {
            const int x0 = EARLY ? x_at : here(x_at), y0 = EARLY ? y_at : here(y_at);
#pragma unroll
            for (int kd = 0; kd < KD; ++kd)
#pragma unroll
                for (int p = 0; p < PC; ++p)
                    fx[r][kd].p[p] = xt[(p * kBwdRows + 16 * r) * S::XS + (x0 ^ 4 * kd)];
#pragma unroll
            for (int ko = 0; ko < KO; ++ko)
#pragma unroll
                for (int p = 0; p < PC; ++p)
                    fy[r][ko].p[p] = yt[(p * kBwdRows + 16 * r) * S::YS + (y0 ^ 4 * ko)];
        };
        if constexpr (EARLY) {
#pragma unroll
            for (int r = 0; r < R; ++r) ask(r);
            asked();
        }
        uint2 gate[R][3][PM];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if constexpr (!EARLY) ask(r);
            f32x4 g{0.f, 0.f, 0.f, 0.f}, u = g, dh = g;
#pragma unroll
            for (int kd = 0; kd < KD; ++kd) {
                g = W::mma(wg[kd], fx[r][kd], g);
                u = W::mma(wu[kd], fx[r][kd], u);
            }
#pragma unroll
            for (int ko = 0; ko < KO; ++ko) dh = W::mma(wd[ko], fy[r][ko], dh);
            float v[3][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float slope;
                const float a = activate<GELU, kExact<E>>(silu, g[i], slope);
                v[0][i] = dh[i] * u[i] * slope;
                v[1][i] = dh[i] * a;
                v[2][i] = a * u[i];
            }
#pragma unroll
            for (int j = 0; j < 3; ++j) S2::four(v[j], gate[r][j]);
            pause();
        }
        // lanes of neighbouring quads hold channels 0-3 and 4-7 of the same two
        // rows: they swap, and each stores eight of one row
#pragma unroll
        for (int j = 0; j < 3; ++j)
#pragma unroll
            for (int p = 0; p < PM; ++p) {
                const auto lo = __builtin_amdgcn_permlane16_swap(gate[0][j][p].x, gate[1][j][p].x,
                                                                 false, false);
                const auto hi = __builtin_amdgcn_permlane16_swap(gate[0][j][p].y, gate[1][j][p].y,
                                                                 false, false);
                gates[j * S::GATE + p * kBwdRows * 4 +
                      tile_slot<4>(16 * (quad & 1) + col, 2 * half + (quad >> 1))] =
                    u32x4{lo[0], hi[0], lo[1], hi[1]};
            }
        __syncthreads();
        // the pair's part of dx, every other 16 of its channels, and the weight
        // gradients, whose operands lie along the rows
        Mid fg[R], fu[R], t[3];
        auto ask_gates = [&](int r) {
            const int row = 16 * r + col;
#pragma unroll
            for (int p = 0; p < PM; ++p) {
                fg[r].p[p] = gates[p * kBwdRows * 4 + tile_slot<4>(row, quad)];
                fu[r].p[p] = gates[S::GATE + p * kBwdRows * 4 + tile_slot<4>(row, quad)];
            }
        };
        auto turn_gate = [&](int j) {
#pragma unroll
            for (int p = 0; p < PM; ++p)
                t[j].p[p] = read_turned<4>(gates + j * S::GATE + p * kBwdRows * 4, half, turned4);
        };
        if constexpr (EARLY) {
#pragma unroll
            for (int r = 0; r < R; ++r) ask_gates(r);
            turn_gate(0);
            turn_gate(1);
            turn_gate(2);
        }
        asked();
        auto dx_part = [&](int r, int j, const Other& g, const Other& u) {
            f32x4 d{0.f, 0.f, 0.f, 0.f};
            d = S2::mma(g, fg[r], d);
            d = S2::mma(u, fu[r], d);
            sums[pair * S::SUM + sum_slot<8 * KD>(16 * r + col, (2 * j + half) * 4 + quad)] =
                __builtin_bit_cast(u32x4, d);
        };
        if constexpr (S::LATE) {
#pragma unroll
            for (int r = 0; r < R; ++r) ask_gates(r);
#pragma unroll
            for (int j = 0; j < KD; ++j) {
                const Other g = S2::other(here(wgt[j])), u = S2::other(here(wut[j]));
#pragma unroll
                for (int r = 0; r < R; ++r) dx_part(r, j, g, u);
                pause();
            }
        } else {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if constexpr (!EARLY) ask_gates(r);
#pragma unroll
                for (int j = 0; j < KD; ++j) dx_part(r, j, wgt[j], wut[j]);
                pause();
            }
        }
        // 16 channels of x or dy along the rows; where registers are short the
        // places are formed again for every tile, too
        const int at_x = EARLY ? turned_xs : here(turned_xs);
        const int at_y = EARLY ? turned_ys : here(turned_ys);
        auto turned = [&](const u32x4* tile, auto slots, int block, int base) {
            constexpr int SLOTS = decltype(slots)::value;
            if constexpr (S::LATE) return S2::other(read_turned<SLOTS>(tile, block, base));
            Other o;
#pragma unroll
            for (int p = 0; p < S::PO; ++p)
                o.p[p] = read_turned<SLOTS>(tile + (S::AT + p) * kBwdRows * SLOTS, block, base);
            return o;
        };
        auto turned_x = [&](int db) {
            return turned(xt, std::integral_constant<int, S::XS>{}, db, at_x);
        };
        auto turned_y = [&](int ob) {
            return turned(yt, std::integral_constant<int, S::YS>{}, ob, at_y);
        };
        Other ahead;  // the next block's operand
        if constexpr (EARLY) {
            ahead = turned_x(0);
        } else {
            turn_gate(0);
            turn_gate(1);
        }
        asked();
#pragma unroll
        for (int db = 0; db < 2 * KD; ++db) {
            Other x;
            if constexpr (EARLY) {
                x = ahead;
                ahead = db + 1 < 2 * KD ? turned_x(db + 1) : turned_y(0);
                asked();
            } else {
                x = turned_x(db);
            }
            sg[db] = S2::mma(x, t[0], sg[db]);
            su[db] = S2::mma(x, t[1], su[db]);
        }
        pause();
        if constexpr (!EARLY) turn_gate(2);
#pragma unroll
        for (int ob = 0; ob < 2 * KO; ++ob) {
            Other y;
            if constexpr (EARLY) {
                y = ahead;
                if (ob + 1 < 2 * KO) ahead = turned_y(ob + 1);
                asked();
            } else {
                y = turned_y(ob);
            }
            sd[ob] = S2::mma(y, t[2], sd[ob]);
        }
        // the next tile into the other place, then the pairs' parts of dx
        settle_all(tiles + (turn ^ 1) * S::TILE, row0 + step);
        fetch_all();
        __syncthreads();
        if (q.dx || q.dx_parts)
            for (int n = threadIdx.x; n < kBwdRows * 8 * KD; n += threads) {
                const int row = n / (8 * KD), slot = n % (8 * KD), d = 4 * slot;
                const int64_t at = row0 + row;
                if (at >= rows || d >= q.d_in) continue;
                f32x4 v{0.f, 0.f, 0.f, 0.f};
                const u32x4* part = sums + sum_slot<8 * KD>(row, slot);
#pragma unroll
                for (int w = 0; w < kBwdPairs; ++w)
                    if (w < pairs) v += __builtin_bit_cast(f32x4, part[w * S::SUM]);
                if (q.dx_parts) {
                    float* out = q.dx_parts + ((int64_t)blockIdx.y * q.rows + at) * q.d_in + d;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (d + i < q.d_in) out[i] = v[i];
                } else {
                    T w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = E::down(v[i]);
                    T* out = q.dx + at * q.d_in + d;
                    if (d + 4 <= q.d_in) {
                        __builtin_memcpy(out, w, sizeof(w));
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (d + i < q.d_in) out[i] = w[i];
                    }
                }
            }
    }
    float* out = q.parts +
                 (((int64_t)blockIdx.x * gridDim.y + blockIdx.y) * 2 * kBwdPairs + wave) * S::SUMS *
                     64 + lane;
    auto leave = [&](float v) {
        *out = q.add ? *out + v : v;
        out += 64;
    };
#pragma unroll
    for (int d = 0; d < 2 * KD; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            leave(sg[d][i]);
            leave(su[d][i]);
        }
#pragma unroll
    for (int o = 0; o < 2 * KO; ++o)
#pragma unroll
        for (int i = 0; i < 4; ++i) leave(sd[o][i]);
}

// Adds up the workgroups' weight gradients in their order: 64 sums of one wave
// on the lanes, a quarter of the workgroups on each of four waves.
template <class E, int KD, int KO>
__global__ __launch_bounds__(kThreads) void k_narrow_join(const float* parts, int blocks,
                                                          int groups, int d_in, int hidden,
                                                          int d_out, typename E::T* dwg,
                                                          typename E::T* dwu, typename E::T* dwd) {
    constexpr int SUMS = 16 * KD + 8 * KO;
    __shared__ float red[kThreads];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int unit = blockIdx.x;  // (group, pair, half, sum)
    const int in = unit % SUMS, chunk = unit / SUMS;
    const int64_t pitch = (int64_t)groups * 2 * kBwdPairs * SUMS * 64;
    const float* p = parts + (int64_t)unit * 64 + lane;
    const int per = (blocks + 3) / 4, b0 = wave * per, b1 = b0 + per < blocks ? b0 + per : blocks;
    float s = 0.f;
    int b = b0;
    for (; b + 8 <= b1; b += 8) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = p[(b + i) * pitch];
#pragma unroll
        for (int i = 0; i < 8; ++i) s += v[i];
    }
    for (; b < b1; ++b) s += p[b * pitch];
    red[threadIdx.x] = s;
    __syncthreads();
    if (wave) return;
    s = red[lane] + red[lane + 64] + red[lane + 128] + red[lane + 192];
    const int f = chunk * 16 + (lane & 15), quad = lane >> 4;
    if (f >= hidden) return;
    if (in < 16 * KD) {
        const int d = 16 * (in / 8) + 4 * quad + in % 8 / 2;
        typename E::T* out = in & 1 ? dwu : dwg;
        if (d < d_in && out) out[(int64_t)f * d_in + d] = E::down(s);
    } else {
        const int o = 16 * ((in - 16 * KD) / 4) + 4 * quad + in % 4;
        if (o < d_out && dwd) dwd[(int64_t)o * hidden + f] = E::down(s);
    }
}

// ----------------------------------------------------------------- host --

struct Shape {
    int dtype, act;
    int64_t rows;
    int d_in, hidden, d_out;
    int size() const { return dtype == GSX_F32 ? 4 : 2; }
};

int64_t up_to(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

int check_shape(const Shape& s) {
    if (s.dtype != GSX_F32 && s.dtype != GSX_BF16 && s.dtype != GSX_F16) return GSX_ERR_INVALID;
    if (s.act != GSX_ACT_SILU && s.act != GSX_ACT_GELU && s.act != GSX_ACT_SIGMOID)
        return GSX_ERR_INVALID;
    if (s.rows < 0 || s.d_in <= 0 || s.hidden <= 0 || s.d_out <= 0) return GSX_ERR_INVALID;
    constexpr int64_t most = 1 << 30, wide = 1 << 20;
    if (s.rows > most || s.d_in > wide || s.hidden > wide || s.d_out > wide)
        return GSX_ERR_TOO_LARGE;
    return GSX_OK;
}

// A launch holds fewer than 2^32 threads in all, workgroups times their size.
constexpr int64_t kMostGroups = (1LL << 32) / kThreads - 1;
// Workgroups for n elements that threads walk by the grid's size.
dim3 groups_for(int64_t n) {
    const int64_t groups = (n + kThreads - 1) / kThreads;
    return dim3((unsigned)(groups < kMostGroups ? groups : kMostGroups));
}

// Workgroups of one product; the grid's x holds all of them.
int64_t tiles(int64_t m, int64_t n) { return up_to(m, kBM) / kBM * (up_to(n, kBN) / kBN); }

// Splits of the rows for a weight gradient of m x n: workgroups for twice the 256
// compute units, which hold two each (a few more would run as a second round),
// no split under eight stages of 64 rows.
struct Splits {
    int count;
    int64_t depth;
};
Splits splits_of(int64_t rows, int64_t m, int64_t n) {
    int64_t want = 512 / tiles(m, n);
    const int64_t most = (rows + 511) / 512;
    if (want > most) want = most;
    if (want < 1) want = 1;
    const int64_t depth = up_to((rows + want - 1) / want, 64);
    return Splits{(int)((rows + depth - 1) / depth), depth};
}

template <class E, Mode MODE>
int launch_tile(const Tile& q, int splits, hipStream_t st) {
    const int64_t n = tiles(q.m, q.n);
    if (n * splits > kMostGroups) return GSX_ERR_TOO_LARGE;
    constexpr int lds = TileShape<E, MODE>::BYTES;
    if (hipFuncSetAttribute((const void*)k_tile<E, MODE>,
                            hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
        return GSX_ERR_HIP;
    hipLaunchKernelGGL((k_tile<E, MODE>), dim3((unsigned)n, (unsigned)splits), dim3(kThreads), lds,
                       st, q);
    GSX_LAUNCH_CHECK();
    return GSX_OK;
}

// The rows are walked in stretches, so that what stands between two kernels
// (arrays of hidden width, the groups' parts of dx) is bounded: kStretchBytes an
// array, and no more workgroups than a launch holds.  Stretches of equal length:
// a power of two (131 072 rows of 512 float32) cost 8 %, its splits begin on the
// same memory channels.  Gradient, us in one stretch / in stretches of 1 GB / of
// 256 MB, 921 600 rows: 64 -> 512 -> 64 float32 11 470 / 11 670 / 12 430; 128 ->
// 1024 -> 32 bf16, whose workgroups take up 100 MB of sums in each, 4220 / 4520 / 5370.
constexpr int64_t kStretchBytes = 1 << 30;

// Rows of a stretch that holds at most `most`, in whole tiles.
int64_t even_stretch(int64_t rows, int64_t most, int tile) {
    most = most / tile * tile;
    if (most < tile) most = tile;
    if (rows <= most) return rows;
    const int64_t count = (rows + most - 1) / most;
    return up_to((rows + count - 1) / count, tile);
}

// A row's pitch in the workspace: whole 16-byte pieces.  Four bytes an element,
// float32 or two bf16 pieces.
int64_t pitch(int width) { return up_to(width, 8); }
int64_t pitch(const Shape& s) { return pitch(s.hidden); }
int64_t held_bytes(int64_t rows, int width) { return up_to(rows * pitch(width) * 4, 256); }
int64_t tiled_stretch(const Shape& s) {
    const int wide = s.hidden > s.d_out ? (s.hidden > s.d_in ? s.hidden : s.d_in)
                                        : (s.d_out > s.d_in ? s.d_out : s.d_in);
    // (float16 rows' pieces stand beside the hidden channels)
    const int64_t fit = kStretchBytes / (4 * (s.dtype == GSX_F16 ? pitch(wide) : pitch(s)));
    const int64_t most = kMostGroups / (up_to(wide, kBN) / kBN) * kBM;
    return even_stretch(s.rows, fit < most ? fit : most, kBM);
}
int64_t hidden_bytes(const Shape& s) { return held_bytes(tiled_stretch(s), s.hidden); }

// Whether the narrow kernel holds a row's operands and sums in its registers:
// 8 (KD pieces + OB) of them, beside some 100 others.
constexpr bool narrow_fits(int pieces, int kd, int ob) { return 8 * (kd * pieces + ob) <= 152; }
int64_t narrow_chunk_bytes(const Shape& s, int kd, int ob) {
    const int in = s.dtype == GSX_F32 ? 3 : 1, out = s.dtype == GSX_BF16 ? 1 : in + 1;
    return (int64_t)(4 * kd * in + ob * (s.dtype == GSX_F32 ? 3 : out)) * 1024;
}
int narrow_kd(const Shape& s) { return s.d_in <= 32 ? 1 : s.d_in <= 64 ? 2 : 4; }
int narrow_ob(const Shape& s) {
    return s.d_out <= 16 ? 1 : s.d_out <= 32 ? 2 : s.d_out <= 64 ? 4 : s.d_out <= 128 ? 8 : 16;
}
// Weights that shared memory holds whole are staged once; others by every
// workgroup for every 256 rows, which many rows have to pay for.  Against the
// tiled path, us a call (131 072, 16 384, 64 rows): 32 -> 128 -> 64 float32, held
// whole, 33 / 84, 17 / 24, 15 / 23; 128 -> 1024 -> 64 float32 431 / 918, 200 / 142,
// 190 / 58; 128 -> 512 -> 64 bf16 86 / 175, 36 / 29, 33 / 21, f16 93 / 185, 39 / 33,
// 37 / 24.
constexpr int64_t kStreamRows = 32768;

bool narrow_fwd(const Shape& s) {
    if (s.d_in > 128 || s.d_out > 256) return false;
    const int kd = narrow_kd(s), ob = narrow_ob(s);
    if (!narrow_fits(s.dtype == GSX_F32 ? 3 : 1, kd, ob)) return false;
    return (s.hidden + 31) / 32 * narrow_chunk_bytes(s, kd, ob) <= kNarrowLds ||
           s.rows >= kStreamRows;
}

int64_t fwd_bytes(const Shape& s) {
    if (s.rows == 0 || narrow_fwd(s)) return 0;
    return hidden_bytes(s) + (s.dtype == GSX_F16 ? held_bytes(s.d_out, s.hidden) : 0);
}

template <class E, int KD, int OB>
int launch_narrow_fwd(const Shape& s, const void* x, int64_t ldx, const void* wg, const void* wu,
                      const void* wd, void* y, hipStream_t st) {
    using T = typename E::T;
    Narrow<E> q{(const T*)x, (const T*)wg, (const T*)wu, (const T*)wd, (T*)y, ldx,
                s.rows,      s.d_in,       s.hidden,     s.d_out,      s.act, 0, 0};
    const int64_t chunk = narrow_chunk_bytes(s, KD, OB);
    q.chunks = (s.hidden + 31) / 32;
    q.resident = (int)(kNarrowLds / chunk);
    if (q.resident > q.chunks) q.resident = q.chunks;
    const int64_t lds = q.resident * chunk;
    const int64_t tiles = (s.rows + kNarrowThreads / 64 * kNarrowRows - 1) /
                          (kNarrowThreads / 64 * kNarrowRows);
    int64_t per_cu = 160 * 1024 / lds;
    if (per_cu > 2) per_cu = 2;
    const int64_t grid = tiles < 256 * per_cu ? tiles : 256 * per_cu;
    const auto kernel = s.act == GSX_ACT_GELU ? k_narrow_fwd<E, KD, OB, true>
                                              : k_narrow_fwd<E, KD, OB, false>;
    if (hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                            (int)kNarrowLds) != hipSuccess)
        return GSX_ERR_HIP;
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(kNarrowThreads), (unsigned)lds, st, q);
    GSX_LAUNCH_CHECK();
    return GSX_OK;
}

template <class E, int KD, int OB, class... A>
int narrow_if(const Shape& s, A... a) {
    if constexpr (narrow_fits(Wide<E>::PIECES, KD, OB))
        return launch_narrow_fwd<E, KD, OB>(s, a...);
    else
        return GSX_ERR_INVALID;  // narrow_fwd() keeps these out
}
template <class E, int KD, class... A>
int narrow_forward(const Shape& s, A... a) {
    switch (narrow_ob(s)) {
        case 1: return narrow_if<E, KD, 1>(s, a...);
        case 2: return narrow_if<E, KD, 2>(s, a...);
        case 4: return narrow_if<E, KD, 4>(s, a...);
        case 8: return narrow_if<E, KD, 8>(s, a...);
        default: return narrow_if<E, KD, 16>(s, a...);
    }
}

// The float16 backward's pieces: of a stretch of x and of dy, of both pair weights.
int64_t pieces_bytes(const Shape& s) {
    if (s.dtype != GSX_F16) return 0;
    return held_bytes(tiled_stretch(s), s.d_in) + held_bytes(tiled_stretch(s), s.d_out) +
           2 * held_bytes(s.hidden, s.d_in);
}

// One split of one stretch leaves the gradient itself; else each leaves partial
// sums, kept over the stretches.
bool direct_grad(const Shape& s, int m) {
    const int64_t rows = tiled_stretch(s);
    return rows == s.rows && splits_of(rows, m, s.hidden).count == 1;
}
// of one weight matrix with m columns or rows beside the hidden ones
int64_t sums_bytes(const Shape& s, int m) {
    if (direct_grad(s, m)) return 0;
    return splits_of(tiled_stretch(s), m, s.hidden).count * (int64_t)s.hidden * m * 4;
}
int64_t pair_parts_bytes(const Shape& s) { return up_to(2 * sums_bytes(s, s.d_in), 256); }
int64_t parts_bytes(const Shape& s) {
    return pair_parts_bytes(s) + up_to(sums_bytes(s, s.d_out), 256);
}

// The narrow backward: which widths fit its registers (weights in both orders
// and their gradients' sums), its workgroups and its workspace.
constexpr bool narrow_bwd_fits(int dtype, int kd, int ko) {
    return dtype == GSX_F32 ? kd + ko <= 3 : kd < 4 || ko <= 2;
}
// Faster than the tiled path wherever its registers and shared memory hold the
// widths, us a call (131 072 rows; of few the host's 100 in both): 32 -> 128 -> 64
// float32 101 / 591, bf16 96 / 350, f16 98 / 441; 32 -> 512 -> 64, four groups,
// 276 / 1604, 155 / 732, 202 / 857; 128 -> 512 -> 64 bf16 395 / 788, f16 503 / 927.
// Hidden widths are bounded by the groups' parts of dx, a float32 array of a stretch of
// x each.
constexpr int kNarrowHidden = 2048;
int narrow_ko(const Shape& s) { return s.d_out <= 32 ? 1 : s.d_out <= 64 ? 2 : 4; }
bool narrow_bwd(const Shape& s) {
    return s.d_in <= 128 && s.d_out <= 128 && s.hidden <= kNarrowHidden &&
           narrow_bwd_fits(s.dtype, narrow_kd(s), narrow_ko(s));
}
struct BwdPlan {
    int pairs, groups, blocks;
    int64_t stretch;  // rows of one launch
    int64_t parts, dx_parts, bytes;
};
BwdPlan bwd_plan(const Shape& s) {
    BwdPlan p{};
    const int kd = narrow_kd(s), ko = narrow_ko(s), chunks = (s.hidden + 31) / 32;
    p.groups = (chunks + kBwdPairs - 1) / kBwdPairs;
    p.pairs = chunks < kBwdPairs ? chunks : kBwdPairs;
    p.stretch = p.groups == 1 ? s.rows
                              : even_stretch(s.rows, kStretchBytes / (p.groups * s.d_in * 4),
                                             kBwdRows);
    const int64_t tiles = (p.stretch + kBwdRows - 1) / kBwdRows;
    const int per_unit = (s.dtype == GSX_BF16 ? 2 : 1) * kBwdPairs / p.pairs;
    int64_t want = 256 * per_unit / p.groups;
    if (want > tiles) want = tiles;
    p.blocks = (int)(want < 1 ? 1 : want);
    p.parts = up_to((int64_t)p.blocks * p.groups * 2 * kBwdPairs * (16 * kd + 8 * ko) * 256, 256);
    p.dx_parts = p.groups > 1 ? up_to(p.groups * p.stretch * s.d_in * 4, 256) : 0;
    p.bytes = p.parts + p.dx_parts;
    return p;
}

int64_t bwd_bytes(const Shape& s) {
    if (s.rows == 0) return 0;
    return narrow_bwd(s) ? bwd_plan(s).bytes
                         : 3 * hidden_bytes(s) + pieces_bytes(s) + parts_bytes(s);
}

struct BwdArgs {
    const void* x;
    int64_t ldx;
    const void *wg, *wu, *wd, *dy;
    int64_t lddy;
    void *dx, *dwg, *dwu, *dwd, *ws;
    hipStream_t st;
};

template <class E, int KD, int KO>
int launch_narrow_bwd(const Shape& s, const BwdArgs& a) {
    constexpr int dtype = std::is_same_v<E, F32>    ? GSX_F32
                          : std::is_same_v<E, BF16> ? GSX_BF16
                                                    : GSX_F16;
    if constexpr (!narrow_bwd_fits(dtype, KD, KO)) {
        return GSX_ERR_INVALID;  // narrow_bwd() keeps these out
    } else {
        using T = typename E::T;
        using S = BwdShape<E, KD, KO>;
        const BwdPlan p = bwd_plan(s);
        float* parts = (float*)a.ws;
        float* dx_parts = p.groups > 1 ? (float*)((char*)a.ws + p.parts) : nullptr;
        if (!a.dx) dx_parts = nullptr;
        const int64_t lds = S::lds(p.pairs);
        const auto kernel = s.act == GSX_ACT_GELU ? k_narrow_bwd<E, KD, KO, true>
                                                  : k_narrow_bwd<E, KD, KO, false>;
        if (hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                                160 * 1024) != hipSuccess)
            return GSX_ERR_HIP;
        for (int64_t row0 = 0; row0 < s.rows; row0 += p.stretch) {
            const int64_t rows = s.rows - row0 < p.stretch ? s.rows - row0 : p.stretch;
            T* dx = a.dx ? (T*)a.dx + row0 * s.d_in : nullptr;
            const NarrowBwd<E> q{(const T*)a.x + row0 * a.ldx, (const T*)a.wg, (const T*)a.wu,
                                 (const T*)a.wd, (const T*)a.dy + row0 * a.lddy,
                                 p.groups > 1 ? nullptr : dx, dx_parts, parts, a.ldx, a.lddy, rows,
                                 s.d_in, s.hidden, s.d_out, s.act, row0 > 0};
            hipLaunchKernelGGL(kernel, dim3(p.blocks, p.groups), dim3(128 * p.pairs),
                               (unsigned)lds, a.st, q);
            GSX_LAUNCH_CHECK();
            if (dx_parts) {
                const int64_t n = rows * s.d_in;
                hipLaunchKernelGGL((k_join<E>), groups_for(n), dim3(kThreads), 0, a.st, dx_parts,
                                   n, p.groups, dx);
                GSX_LAUNCH_CHECK();
            }
        }
        if (a.dwg || a.dwd) {
            const int halves = p.groups * 2 * kBwdPairs;
            hipLaunchKernelGGL((k_narrow_join<E, KD, KO>), dim3(halves * S::SUMS), dim3(kThreads),
                               0, a.st, parts, p.blocks, p.groups, s.d_in, s.hidden, s.d_out,
                               (T*)a.dwg, (T*)a.dwu, (T*)a.dwd);
            GSX_LAUNCH_CHECK();
        }
        return GSX_OK;
    }
}
template <class E, int KD>
int launch_narrow_bwd(const Shape& s, const BwdArgs& a) {
    switch (narrow_ko(s)) {
        case 1: return launch_narrow_bwd<E, KD, 1>(s, a);
        case 2: return launch_narrow_bwd<E, KD, 2>(s, a);
        default: return launch_narrow_bwd<E, KD, 4>(s, a);
    }
}

// Launches the split of float16 rows into two planes at `to`, and describes them.
int pieces(void* to, const void* x, int64_t ld, int64_t rows, int cols, Operand* o,
           hipStream_t st) {
    const int wide = (int)pitch(cols);
    hipLaunchKernelGGL(k_pieces, groups_for(rows * ((cols + 1) / 2)), dim3(kThreads), 0, st,
                       (const uint16_t*)x, ld, rows, cols, wide, (uint16_t*)to);
    GSX_LAUNCH_CHECK();
    o->p = to;
    o->lo = (uint16_t*)to + rows * wide;
    o->ld = wide;
    return GSX_OK;
}

template <class E>
int forward(const Shape& s, const void* x, int64_t ldx, const void* wg, const void* wu,
            const void* wd, void* y, void* ws, hipStream_t st) {
    if (narrow_fwd(s)) {
        switch (narrow_kd(s)) {
            case 1: return narrow_forward<E, 1>(s, x, ldx, wg, wu, wd, y, st);
            case 2: return narrow_forward<E, 2>(s, x, ldx, wg, wu, wd, y, st);
            default: return narrow_forward<E, 4>(s, x, ldx, wg, wu, wd, y, st);
        }
    }
    using T = typename E::T;
    const int64_t ph = pitch(s), stretch = tiled_stretch(s), plane = stretch * ph;
    Operand down{wd, s.hidden, s.d_out};
    if constexpr (std::is_same_v<E, F16>)
        if (int e = pieces((char*)ws + hidden_bytes(s), wd, s.hidden, s.d_out, s.hidden, &down, st))
            return e;
    for (int64_t row0 = 0; row0 < s.rows; row0 += stretch) {
        const int rows = (int)(s.rows - row0 < stretch ? s.rows - row0 : stretch);
        Tile q{};
        q.a = Operand{(const T*)x + row0 * ldx, ldx, rows};
        q.b0 = Operand{wg, s.d_in, s.hidden};
        q.b1 = Operand{wu, s.d_in, s.hidden};
        q.k = s.d_in;
        q.m = rows;
        q.n = s.hidden;
        q.out[0] = ws;
        q.ldo = ph;
        q.plane = plane;
        q.act = s.act;
        if (int e = launch_tile<E, HIDDEN>(q, 1, st)) return e;
        Tile r{};
        r.a = Operand{ws, ph, rows, (uint16_t*)ws + plane};
        r.b0 = down;
        r.k = s.hidden;
        r.m = rows;
        r.n = s.d_out;
        r.out[0] = (T*)y + row0 * s.d_out;
        r.ldo = s.d_out;
        if (int e = launch_tile<E, PLAIN>(r, 1, st)) return e;
    }
    return GSX_OK;
}

// A weight gradient's sums over the stretch of rows that begins at row0, in splits
// that each add to their own part; the last stretch adds the parts up.
template <class E>
int weight_grad(const Tile& base, const Shape& s, int64_t row0, int64_t stretch,
                void* const* outs, int count, float* parts, hipStream_t st) {
    const Splits sp = splits_of(stretch, base.m, base.n);
    const int64_t n = (int64_t)base.m * base.n;
    const bool direct = direct_grad(s, base.m), last = row0 + stretch >= s.rows;
    Tile q = base;
    q.k = last ? s.rows - row0 : stretch;
    q.split_k = sp.depth;
    q.split_out = direct ? 0 : n;
    q.add = row0 > 0;
    q.ldo = count == 2 ? base.m : base.n;
    for (int i = 0; i < count; ++i)
        q.out[i] = direct ? outs[i] : (void*)(parts + i * sp.count * n);
    const int splits = (int)((q.k + sp.depth - 1) / sp.depth);
    const int e = count == 2 ? launch_tile<E, WGRAD2>(q, splits, st)
                             : launch_tile<E, WGRAD>(q, splits, st);
    if (e) return e;
    if (!direct && last)
        for (int i = 0; i < count; ++i) {
            hipLaunchKernelGGL((k_join<E>), groups_for(n), dim3(kThreads), 0, st,
                               parts + i * sp.count * n, n, sp.count, (typename E::T*)outs[i]);
            GSX_LAUNCH_CHECK();
        }
    return GSX_OK;
}

template <class E>
int backward(const Shape& s, const void* x, int64_t ldx, const void* wg, const void* wu,
             const void* wd, const void* dy, int64_t lddy, void* dx, void* dwg, void* dwu,
             void* dwd, void* ws, hipStream_t st) {
    if (narrow_bwd(s)) {
        const BwdArgs a{x, ldx, wg, wu, wd, dy, lddy, dx, dwg, dwu, dwd, ws, st};
        switch (narrow_kd(s)) {
            case 1: return launch_narrow_bwd<E, 1>(s, a);
            case 2: return launch_narrow_bwd<E, 2>(s, a);
            default: return launch_narrow_bwd<E, 4>(s, a);
        }
    }
    using T = typename E::T;
    const int64_t ph = pitch(s), hb = hidden_bytes(s), stretch = tiled_stretch(s);
    const int64_t plane = stretch * ph;
    void* dg = ws;
    void* du = (char*)ws + hb;
    void* h = (char*)ws + 2 * hb;
    auto held = [&](const void* p, int n) {
        return Operand{p, ph, n, (const uint16_t*)p + plane};
    };
    // float16: the pieces of x and dy, of the pair's weights
    char* x_pieces = (char*)ws + 3 * hb;
    char* dy_pieces = x_pieces + held_bytes(stretch, s.d_in);
    char* w_pieces = dy_pieces + held_bytes(stretch, s.d_out);
    // the pair's parts, then the down weights'
    float* pair_parts = (float*)((char*)ws + 3 * hb + pieces_bytes(s));
    float* down_parts = (float*)((char*)pair_parts + pair_parts_bytes(s));
    Operand gate{wg, s.d_in, s.d_in}, up{wu, s.d_in, s.d_in};
    if constexpr (std::is_same_v<E, F16>)
        if (dx) {
            const int64_t one = held_bytes(s.hidden, s.d_in);
            if (int e = pieces(w_pieces, wg, s.d_in, s.hidden, s.d_in, &gate, st)) return e;
            if (int e = pieces(w_pieces + one, wu, s.d_in, s.hidden, s.d_in, &up, st)) return e;
        }
    for (int64_t row0 = 0; row0 < s.rows; row0 += stretch) {
        const int rows = (int)(s.rows - row0 < stretch ? s.rows - row0 : stretch);
        const T* xs = (const T*)x + row0 * ldx;
        const T* dys = (const T*)dy + row0 * lddy;
        Tile q{};
        q.a = Operand{xs, ldx, rows};
        q.b0 = Operand{wg, s.d_in, s.hidden};
        q.b1 = Operand{wu, s.d_in, s.hidden};
        q.k = s.d_in;
        q.a2 = Operand{dys, lddy, rows};
        q.b2 = Operand{wd, s.hidden, s.hidden};
        q.k2 = s.d_out;
        q.m = rows;
        q.n = s.hidden;
        q.out[0] = dg;
        q.out[1] = du;
        q.out[2] = h;
        q.ldo = ph;
        q.plane = plane;
        q.act = s.act;
        if (int e = launch_tile<E, BWD_HIDDEN>(q, 1, st)) return e;
        if (dx) {
            Tile r{};
            r.a = held(dg, rows);
            r.b0 = gate;
            r.a2 = held(du, rows);
            r.b2 = up;
            r.k = s.hidden;
            r.m = rows;
            r.n = s.d_in;
            r.out[0] = (T*)dx + row0 * s.d_in;
            r.ldo = s.d_in;
            if (int e = launch_tile<E, SUM2>(r, 1, st)) return e;
        }
        if (dwg) {
            Tile r{};
            r.a = Operand{xs, ldx, s.d_in};
            if constexpr (std::is_same_v<E, F16>)
                if (int e = pieces(x_pieces, xs, ldx, rows, s.d_in, &r.a, st)) return e;
            r.b0 = held(dg, s.hidden);
            r.b1 = held(du, s.hidden);
            r.m = s.d_in;
            r.n = s.hidden;
            void* outs[2] = {dwg, dwu};
            if (int e = weight_grad<E>(r, s, row0, stretch, outs, 2, pair_parts, st)) return e;
        }
        if (dwd) {
            Tile r{};
            r.a = Operand{dys, lddy, s.d_out};
            if constexpr (std::is_same_v<E, F16>)
                if (int e = pieces(dy_pieces, dys, lddy, rows, s.d_out, &r.a, st)) return e;
            r.b0 = held(h, s.hidden);
            r.m = s.d_out;
            r.n = s.hidden;
            void* outs[1] = {dwd};
            if (int e = weight_grad<E>(r, s, row0, stretch, outs, 1, down_parts, st)) return e;
        }
    }
    return GSX_OK;
}

int zero(void* p, int64_t bytes, hipStream_t st) {
    if (!p) return GSX_OK;
    hipLaunchKernelGGL(k_zero_bytes, groups_for(bytes), dim3(kThreads), 0, st, (uint8_t*)p, bytes);
    GSX_LAUNCH_CHECK();
    return GSX_OK;
}

bool misaligned(const void* p, int size) { return (uintptr_t)p % (uintptr_t)size != 0; }

}  // namespace

extern "C" {

int64_t gsx_ffn_fwd_workspace_bytes(int32_t dtype, int32_t act, int64_t rows, int32_t d_in,
                                    int32_t hidden, int32_t d_out) {
    const Shape s{dtype, act, rows, d_in, hidden, d_out};
    if (int e = check_shape(s)) return e;
    return fwd_bytes(s);
}

int gsx_ffn_fwd(int32_t dtype, int32_t act, int64_t rows, int32_t d_in, int32_t hidden,
                int32_t d_out, const void* x, int64_t x_stride, const void* w_gate,
                const void* w_up, const void* w_down, void* y, void* workspace,
                int64_t workspace_bytes, void* stream) {
    const Shape s{dtype, act, rows, d_in, hidden, d_out};
    if (int e = check_shape(s)) return e;
    if (rows == 0) return GSX_OK;
    if (!x || !w_gate || !w_up || !w_down || !y || x_stride < d_in) return GSX_ERR_INVALID;
    for (const void* p : {x, w_gate, w_up, w_down, (const void*)y})
        if (misaligned(p, s.size())) return GSX_ERR_INVALID;
    if (workspace_bytes < fwd_bytes(s) || (fwd_bytes(s) && !workspace)) return GSX_ERR_WORKSPACE;
    if (misaligned(workspace, 16)) return GSX_ERR_INVALID;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == GSX_F32)
        return forward<F32>(s, x, x_stride, w_gate, w_up, w_down, y, workspace, st);
    if (dtype == GSX_BF16)
        return forward<BF16>(s, x, x_stride, w_gate, w_up, w_down, y, workspace, st);
    return forward<F16>(s, x, x_stride, w_gate, w_up, w_down, y, workspace, st);
}

int64_t gsx_ffn_bwd_workspace_bytes(int32_t dtype, int32_t act, int64_t rows, int32_t d_in,
                                    int32_t hidden, int32_t d_out) {
    const Shape s{dtype, act, rows, d_in, hidden, d_out};
    if (int e = check_shape(s)) return e;
    return bwd_bytes(s);
}

int gsx_ffn_bwd(int32_t dtype, int32_t act, int64_t rows, int32_t d_in, int32_t hidden,
                int32_t d_out, const void* x, int64_t x_stride, const void* w_gate,
                const void* w_up, const void* w_down, const void* g_y, int64_t g_y_stride,
                void* g_x, void* g_w_gate, void* g_w_up, void* g_w_down, void* workspace,
                int64_t workspace_bytes, void* stream) {
    const Shape s{dtype, act, rows, d_in, hidden, d_out};
    if (int e = check_shape(s)) return e;
    if (!g_w_gate != !g_w_up) return GSX_ERR_INVALID;
    for (const void* p : {x, w_gate, w_up, w_down, g_y, (const void*)g_x, (const void*)g_w_gate,
                          (const void*)g_w_up, (const void*)g_w_down})
        if (misaligned(p, s.size())) return GSX_ERR_INVALID;
    hipStream_t st = (hipStream_t)stream;
    if (rows == 0) {  // sums over no rows
        const int64_t in = (int64_t)hidden * d_in * s.size();
        if (int e = zero(g_w_gate, in, st)) return e;
        if (int e = zero(g_w_up, in, st)) return e;
        return zero(g_w_down, (int64_t)hidden * d_out * s.size(), st);
    }
    if (!x || !w_gate || !w_up || !w_down || !g_y || x_stride < d_in || g_y_stride < d_out)
        return GSX_ERR_INVALID;
    if (workspace_bytes < bwd_bytes(s) || !workspace) return GSX_ERR_WORKSPACE;
    if (misaligned(workspace, 16)) return GSX_ERR_INVALID;
    if (dtype == GSX_F32)
        return backward<F32>(s, x, x_stride, w_gate, w_up, w_down, g_y, g_y_stride, g_x, g_w_gate,
                             g_w_up, g_w_down, workspace, st);
    if (dtype == GSX_BF16)
        return backward<BF16>(s, x, x_stride, w_gate, w_up, w_down, g_y, g_y_stride, g_x, g_w_gate,
                              g_w_up, g_w_down, workspace, st);
    return backward<F16>(s, x, x_stride, w_gate, w_up, w_down, g_y, g_y_stride, g_x, g_w_gate,
                         g_w_up, g_w_down, workspace, st);
}

}  // extern "C"
