// feedforward.hip -- the gated feed-forward block that decodes rows of
// features, and its gradient.
//
//   g = x Wg^T,  u = x Wu^T,  h = act(g) u,  y = h Wd^T
//   dh = dy Wd,  du = dh act(g),  dg = dh u act'(g)
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dWd = dy^T h
//
// x (rows, d_in), Wg and Wu (hidden, d_in), Wd (d_out, hidden), row-major.
//
// The tiled path (any sizes): products over 128 x 64 tiles with the
// elementwise work in their epilogue.  g and u share one pass over x, so only
// h leaves the first kernel; the backward forms g and u again instead of
// keeping them (a pass over x against two arrays of hidden width).  h, dg and
// du are kept in the tensors' own type between the kernels, in 16 bits rounded
// once each: the same as the rounding of an operand, which the matrix units
// need anyway.  Weight gradients sum over the rows in splits, each split's
// partial sums in float32, added up in a fixed order.
#include <hip/hip_runtime.h>

#include <cmath>

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
__device__ __forceinline__ float activate(int act, float g, float& slope) {
    if (act == GSX_ACT_GELU) {
        const float cdf = 0.5f * (1.0f + erff(g * 0.70710678118654752f));
        slope = cdf + g * 0.39894228040143268f * __expf(-0.5f * g * g);
        return g * cdf;
    }
    const float s = 1.0f / (1.0f + __expf(-g));
    if (act == GSX_ACT_SIGMOID) {
        slope = s * (1.0f - s);
        return s;
    }
    slope = s * (1.0f + g * (1.0f - s));
    return g * s;
}

// ---------------------------------------------------------------- tiles --

// One operand: element (row, k) is p[row * ld + k] where KC (the summed index
// is contiguous), else p[k * ld + row].  `vec`: its 16-byte pieces (KC) or its
// pieces of a few rows are aligned.
struct Operand {
    const void* p;
    int64_t ld;
    int rows;
    int vec;
};

// ROWS rows times two fragments' depth of one operand, kept in fragment order
// (row block, fragment, lane): reads and writes are whole 16-byte lanes.
template <class E, int ROWS, bool KC>
struct Stage {
    using T = typename E::T;
    static constexpr int VEC = E::VEC;
    static constexpr int STEP = 8 * VEC;  // depth of a stage
    static constexpr int N = ROWS / 32;   // 16-byte pieces of a thread
    u32x4 r[N];

    static __device__ __forceinline__ int slot(int row, int piece) {
        return ((row >> 4) * 2 + (piece >> 2)) * 64 + (piece & 3) * 16 + (row & 15);
    }

    __device__ __forceinline__ void load(const Operand& o, int row0, int64_t k0, int64_t k1) {
        const T* p = (const T*)o.p;
        const int t = threadIdx.x;
        if constexpr (KC) {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int row = row0 + (t >> 3) + 32 * n;
                const int64_t k = k0 + (t & 7) * VEC;
                const T* at = p + (int64_t)row * o.ld + k;
                if (row < o.rows && k + VEC <= k1 && o.vec) {
                    r[n] = *(const u32x4*)at;
                } else {
                    T v[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; ++i)
                        v[i] = (row < o.rows && k + i < k1) ? at[i] : (T)0;
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
                if (k + i < k1 && row + N <= o.rows && o.vec) {
                    __builtin_memcpy(v[i], __builtin_assume_aligned(at, N * sizeof(T)),
                                     N * sizeof(T));
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

// c0 += A B0^T and (NB == 2) c1 += A B1^T over the summed index [k0, k1).  The
// next stage's loads are in flight while the present one is multiplied.
template <class E, bool AKC, bool BKC, int NB>
__device__ __forceinline__ void multiply(u32x4* lds, const Operand& A, const Operand& B0,
                                         const Operand& B1, int m0, int n0, int64_t k0, int64_t k1,
                                         Acc& c0, Acc& c1) {
    using SA = Stage<E, kBM, AKC>;
    using SB = Stage<E, kBN, BKC>;
    u32x4* la = lds;
    u32x4* lb0 = lds + kBM * 8;
    u32x4* lb1 = lb0 + kBN * 8;
    SA a;
    SB b0, b1;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int wm = (wave >> 1) * 4, wn = (wave & 1) * 2;  // in blocks of 16
    if (k0 < k1) {
        a.load(A, m0, k0, k1);
        b0.load(B0, n0, k0, k1);
        if constexpr (NB == 2) b1.load(B1, n0, k0, k1);
    }
    for (int64_t k = k0; k < k1; k += SA::STEP) {
        __syncthreads();  // the last stage's reads
        a.store(la);
        b0.store(lb0);
        if constexpr (NB == 2) b1.store(lb1);
        __syncthreads();
        if (k + SA::STEP < k1) {
            a.load(A, m0, k + SA::STEP, k1);
            b0.load(B0, n0, k + SA::STEP, k1);
            if constexpr (NB == 2) b1.load(B1, n0, k + SA::STEP, k1);
        }
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            u32x4 fa[4], fb[2];
#pragma unroll
            for (int i = 0; i < 4; ++i) fa[i] = la[((wm + i) * 2 + f) * 64 + lane];
#pragma unroll
            for (int j = 0; j < 2; ++j) fb[j] = lb0[((wn + j) * 2 + f) * 64 + lane];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) c0[i][j] = E::mma(fb[j], fa[i], c0[i][j]);
            if constexpr (NB == 2) {
#pragma unroll
                for (int j = 0; j < 2; ++j) fb[j] = lb1[((wn + j) * 2 + f) * 64 + lane];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) c1[i][j] = E::mma(fb[j], fa[i], c1[i][j]);
            }
        }
    }
}

// Four consecutive columns of one row; the row's end cuts them short.
template <class E>
__device__ __forceinline__ void put(typename E::T* p, int64_t ld, int row, int col, int rows,
                                    int cols, bool vec, f32x4 v) {
    using T = typename E::T;
    if (row >= rows || col >= cols) return;
    T w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = E::down(v[i]);
    T* at = p + (int64_t)row * ld + col;
    if (vec && col + 4 <= cols) {
        __builtin_memcpy(__builtin_assume_aligned(at, 4 * sizeof(T)), w, 4 * sizeof(T));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (col + i < cols) at[i] = w[i];
    }
}

enum Mode {
    HIDDEN,      // out0 = act(A B0^T) (A B1^T)
    PLAIN,       // out0 = A B0^T
    BWD_HIDDEN,  // g, u as in HIDDEN, dh = A2 B2^T: out0 = dg, out1 = du, out2 = h
    SUM2,        // out0 = A B0^T + A2 B2^T
    WGRAD2,      // out0^T = A B0^T, out1^T = A B1^T over a split of the summed index
    WGRAD        // out0^T = A B0^T over a split
};

struct Tile {
    Operand a, b0, b1, a2, b2;
    int64_t k, k2;        // depths
    int m, n;             // rows of A, rows of B
    void* out[3];
    int64_t ldo;
    int vec_out;
    int act;
    int64_t split_k;      // depth of a split (WGRAD*)
    int64_t split_out;    // floats of a split's partial sums; 0: out itself, in E
};

template <class E, Mode MODE>
__global__ __launch_bounds__(kThreads) void k_tile(const Tile q) {
    using T = typename E::T;
    __shared__ u32x4 lds[(kBM + 2 * kBN) * 8];
    constexpr bool wgrad = MODE == WGRAD || MODE == WGRAD2;
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
        multiply<E, true, true, 1>(lds, q.a, q.b0, q.b0, m0, n0, 0, q.k, c0, c0);
    } else if constexpr (MODE == SUM2) {
        multiply<E, true, false, 1>(lds, q.a, q.b0, q.b0, m0, n0, 0, q.k, c0, c0);
        multiply<E, true, false, 1>(lds, q.a2, q.b2, q.b2, m0, n0, 0, q.k, c0, c0);
    } else {
        const int64_t k0 = blockIdx.y * q.split_k;
        const int64_t k1 = k0 + q.split_k < q.k ? k0 + q.split_k : q.k;
        if constexpr (MODE == WGRAD2) clear(c1);
        multiply<E, false, false, MODE == WGRAD2 ? 2 : 1>(lds, q.a, q.b0, q.b1, m0, n0, k0, k1, c0,
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
            if constexpr (wgrad) {
                // the gradients lie (B row, A row): lanes run along A's
                if (row >= q.m) continue;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (col + e >= q.n) continue;
                    const int64_t at = (int64_t)(col + e) * q.ldo + row;
                    if (q.split_out) {
                        const int64_t s = blockIdx.y * q.split_out;
                        ((float*)q.out[0])[s + at] = c0[i][j][e];
                        if constexpr (MODE == WGRAD2) ((float*)q.out[1])[s + at] = c1[i][j][e];
                    } else {
                        ((T*)q.out[0])[at] = E::down(c0[i][j][e]);
                        if constexpr (MODE == WGRAD2) ((T*)q.out[1])[at] = E::down(c1[i][j][e]);
                    }
                }
            } else if constexpr (MODE == HIDDEN) {
                f32x4 h;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float slope;
                    h[e] = activate(q.act, c0[i][j][e], slope) * c1[i][j][e];
                }
                put<E>((T*)q.out[0], q.ldo, row, col, q.m, q.n, q.vec_out, h);
            } else if constexpr (MODE == BWD_HIDDEN) {
                f32x4 dg, du, h;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float slope;
                    const float a = activate(q.act, c0[i][j][e], slope);
                    const float u = c1[i][j][e], dh = c2[i][j][e];
                    h[e] = a * u;
                    du[e] = dh * a;
                    dg[e] = dh * u * slope;
                }
                put<E>((T*)q.out[0], q.ldo, row, col, q.m, q.n, q.vec_out, dg);
                put<E>((T*)q.out[1], q.ldo, row, col, q.m, q.n, q.vec_out, du);
                put<E>((T*)q.out[2], q.ldo, row, col, q.m, q.n, q.vec_out, h);
            } else {
                put<E>((T*)q.out[0], q.ldo, row, col, q.m, q.n, q.vec_out, c0[i][j]);
            }
        }
}

// Adds up the splits' partial sums in their order.
template <class E>
__global__ __launch_bounds__(kThreads) void k_join(const float* parts, int64_t n, int splits,
                                                   typename E::T* out) {
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= n) return;
    float s = 0.f;
    for (int k = 0; k < splits; ++k) s += parts[k * n + i];
    out[i] = E::down(s);
}

__global__ __launch_bounds__(kThreads) void k_zero_bytes(uint8_t* p, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i < n) p[i] = 0;
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

// Workgroups of one product; the grid's x holds all of them.
int64_t tiles(int64_t m, int64_t n) { return up_to(m, kBM) / kBM * (up_to(n, kBN) / kBN); }

// Splits of the rows for a weight gradient of m x n: enough workgroups for
// twice the 256 compute units, no split under eight stages of 64 rows.
struct Splits {
    int count;
    int64_t depth;
};
Splits splits_of(int64_t rows, int64_t m, int64_t n) {
    int64_t want = (512 + tiles(m, n) - 1) / tiles(m, n);
    const int64_t most = (rows + 511) / 512;
    if (want > most) want = most;
    if (want < 1) want = 1;
    const int64_t depth = up_to((rows + want - 1) / want, 64);
    return Splits{(int)((rows + depth - 1) / depth), depth};
}

template <class E>
Operand operand(const void* p, int64_t ld, int64_t rows, bool kc, int n_rc) {
    const int64_t a = kc ? 16 : n_rc * (int64_t)sizeof(typename E::T);
    const bool vec = (uintptr_t)p % a == 0 && ld * (int64_t)sizeof(typename E::T) % a == 0;
    return Operand{p, ld, (int)rows, vec ? 1 : 0};
}
// the first operand's patches are four rows wide, the second's two
template <class E>
Operand first(const void* p, int64_t ld, int64_t rows, bool kc) {
    return operand<E>(p, ld, rows, kc, kBM / 32);
}
template <class E>
Operand second(const void* p, int64_t ld, int64_t rows, bool kc) {
    return operand<E>(p, ld, rows, kc, kBN / 32);
}

template <class E>
bool out_vec(const void* p, int64_t ld) {
    const int64_t a = 4 * sizeof(typename E::T);
    return (uintptr_t)p % a == 0 && ld * (int64_t)sizeof(typename E::T) % a == 0;
}

template <class E, Mode MODE>
int launch_tile(const Tile& q, int splits, hipStream_t st) {
    const int64_t n = tiles(q.m, q.n);
    if (n >= (1LL << 31)) return GSX_ERR_TOO_LARGE;
    hipLaunchKernelGGL((k_tile<E, MODE>), dim3((unsigned)n, (unsigned)splits), dim3(kThreads), 0,
                       st, q);
    GSX_LAUNCH_CHECK();
    return GSX_OK;
}

// hidden's row pitch in the workspace: whole 16-byte pieces
int64_t pitch(const Shape& s) { return up_to(s.hidden, 8); }
int64_t hidden_bytes(const Shape& s) { return up_to(s.rows * pitch(s) * s.size(), 256); }

int64_t fwd_bytes(const Shape& s) { return s.rows == 0 ? 0 : hidden_bytes(s); }

int64_t parts_bytes(const Shape& s) {
    const Splits a = splits_of(s.rows, s.d_in, s.hidden), b = splits_of(s.rows, s.hidden, s.d_out);
    const int64_t in = 2 * a.count * (int64_t)s.hidden * s.d_in;
    const int64_t out = b.count * (int64_t)s.d_out * s.hidden;
    return up_to((in > out ? in : out) * 4, 256);
}

int64_t bwd_bytes(const Shape& s) { return s.rows == 0 ? 0 : 3 * hidden_bytes(s) + parts_bytes(s); }

template <class E>
int forward(const Shape& s, const void* x, int64_t ldx, const void* wg, const void* wu,
            const void* wd, void* y, int64_t ldy, void* ws, hipStream_t st) {
    const int64_t ph = pitch(s);
    Tile q{};
    q.a = first<E>(x, ldx, s.rows, true);
    q.b0 = second<E>(wg, s.d_in, s.hidden, true);
    q.b1 = second<E>(wu, s.d_in, s.hidden, true);
    q.k = s.d_in;
    q.m = (int)s.rows;
    q.n = s.hidden;
    q.out[0] = ws;
    q.ldo = ph;
    q.vec_out = 1;
    q.act = s.act;
    if (int e = launch_tile<E, HIDDEN>(q, 1, st)) return e;
    Tile r{};
    r.a = first<E>(ws, ph, s.rows, true);
    r.b0 = second<E>(wd, s.hidden, s.d_out, true);
    r.k = s.hidden;
    r.m = (int)s.rows;
    r.n = s.d_out;
    r.out[0] = y;
    r.ldo = ldy;
    r.vec_out = out_vec<E>(y, ldy);
    return launch_tile<E, PLAIN>(r, 1, st);
}

template <class E>
int weight_grad(const Tile& base, int64_t rows, void* const* outs, int count, float* parts,
                hipStream_t st) {
    const Splits sp = splits_of(rows, base.m, base.n);
    const int64_t n = (int64_t)base.m * base.n;
    Tile q = base;
    q.k = rows;
    q.split_k = sp.depth;
    q.split_out = sp.count > 1 ? n : 0;
    q.ldo = base.m;
    for (int i = 0; i < count; ++i)
        q.out[i] = sp.count > 1 ? (void*)(parts + i * sp.count * n) : outs[i];
    const int e = count == 2 ? launch_tile<E, WGRAD2>(q, sp.count, st)
                             : launch_tile<E, WGRAD>(q, sp.count, st);
    if (e) return e;
    if (sp.count > 1)
        for (int i = 0; i < count; ++i) {
            hipLaunchKernelGGL((k_join<E>), dim3((unsigned)((n + kThreads - 1) / kThreads)),
                               dim3(kThreads), 0, st, parts + i * sp.count * n, n, sp.count,
                               (typename E::T*)outs[i]);
            GSX_LAUNCH_CHECK();
        }
    return GSX_OK;
}

template <class E>
int backward(const Shape& s, const void* x, int64_t ldx, const void* wg, const void* wu,
             const void* wd, const void* dy, int64_t lddy, void* dx, void* dwg, void* dwu,
             void* dwd, void* ws, hipStream_t st) {
    const int64_t ph = pitch(s), hb = hidden_bytes(s);
    void* dg = ws;
    void* du = (char*)ws + hb;
    void* h = (char*)ws + 2 * hb;
    float* parts = (float*)((char*)ws + 3 * hb);
    Tile q{};
    q.a = first<E>(x, ldx, s.rows, true);
    q.b0 = second<E>(wg, s.d_in, s.hidden, true);
    q.b1 = second<E>(wu, s.d_in, s.hidden, true);
    q.k = s.d_in;
    q.a2 = first<E>(dy, lddy, s.rows, true);
    q.b2 = second<E>(wd, s.hidden, s.hidden, false);
    q.k2 = s.d_out;
    q.m = (int)s.rows;
    q.n = s.hidden;
    q.out[0] = dg;
    q.out[1] = du;
    q.out[2] = h;
    q.ldo = ph;
    q.vec_out = 1;
    q.act = s.act;
    if (int e = launch_tile<E, BWD_HIDDEN>(q, 1, st)) return e;
    if (dx) {
        Tile r{};
        r.a = first<E>(dg, ph, s.rows, true);
        r.b0 = second<E>(wg, s.d_in, s.d_in, false);
        r.a2 = first<E>(du, ph, s.rows, true);
        r.b2 = second<E>(wu, s.d_in, s.d_in, false);
        r.k = s.hidden;
        r.m = (int)s.rows;
        r.n = s.d_in;
        r.out[0] = dx;
        r.ldo = s.d_in;
        r.vec_out = out_vec<E>(dx, s.d_in);
        if (int e = launch_tile<E, SUM2>(r, 1, st)) return e;
    }
    if (dwg) {
        Tile r{};
        r.a = first<E>(x, ldx, s.d_in, false);
        r.b0 = second<E>(dg, ph, s.hidden, false);
        r.b1 = second<E>(du, ph, s.hidden, false);
        r.m = s.d_in;
        r.n = s.hidden;
        void* outs[2] = {dwg, dwu};
        if (int e = weight_grad<E>(r, s.rows, outs, 2, parts, st)) return e;
    }
    if (dwd) {
        Tile r{};
        r.a = first<E>(h, ph, s.hidden, false);
        r.b0 = second<E>(dy, lddy, s.d_out, false);
        r.m = s.hidden;
        r.n = s.d_out;
        void* outs[1] = {dwd};
        if (int e = weight_grad<E>(r, s.rows, outs, 1, parts, st)) return e;
    }
    return GSX_OK;
}

int zero(void* p, int64_t bytes, hipStream_t st) {
    if (!p) return GSX_OK;
    hipLaunchKernelGGL(k_zero_bytes, dim3((unsigned)((bytes + kThreads - 1) / kThreads)),
                       dim3(kThreads), 0, st, (uint8_t*)p, bytes);
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
    if (workspace_bytes < fwd_bytes(s) || !workspace) return GSX_ERR_WORKSPACE;
    if (misaligned(workspace, 16)) return GSX_ERR_INVALID;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == GSX_F32)
        return forward<F32>(s, x, x_stride, w_gate, w_up, w_down, y, d_out, workspace, st);
    if (dtype == GSX_BF16)
        return forward<BF16>(s, x, x_stride, w_gate, w_up, w_down, y, d_out, workspace, st);
    return forward<F16>(s, x, x_stride, w_gate, w_up, w_down, y, d_out, workspace, st);
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
