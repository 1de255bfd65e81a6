// layernorm.hip -- layer norm over the rows' last dimension, and its gradient with
// the weights' reduction.
//
// With the row's mean m, r = (var + eps)^(-1/2) and h = (x - m) r:
//   y  = h w + b
//   dx = r (g - mean(g) - h mean(g h)),  g = dy w
//   dw = sum over rows of dy h,  db = sum over rows of dy
//
// The variance is formed from differences d to the mean as float32 rounded it, and
// what that rounding left (the differences' own mean) is taken out again, so rows
// far from zero keep their digits.  The gradient forms the statistics again: it has
// to read x anyway, and nothing is kept from the forward pass.  Its four sums over a
// row (d, d^2, g, g d) are one reduction.  All sums are float32 in a fixed order.
//
// A team of lanes, a part of a wave, a wave or a workgroup, holds a row in its
// registers, so each value is read once.  Longer rows are walked by a workgroup,
// which reads them again for each sum.  In the gradient a team keeps its columns of
// dw and db in registers over all its rows; a workgroup leaves one partial row of
// each, and a second launch adds those up.
//
// Memory bounds both directions: 118 MB of 32 float32 columns take 39 us forward (6.1
// TB/s) and 65 backward (5.5), 199 million bfloat16 in rows of 96 145 us forward (5.5).
// The vector units are busy for 45 to 51 % of that, and waves wait in between, so what a
// row costs beside its elements counts, in 16 bits the more: teams are as small as whole
// lines allow, with two or three pieces a lane, so that a sum takes few steps and few
// lanes are idle (120 MB of bfloat16, forward and backward: 300 columns 53 and 83 us, on
// 64 lanes with one piece each 83 and 120; 48 columns 51 and 84 for 67 and 91), and the
// next row is asked for before this one's sums.
// Odd widths cost up to a quarter more in 16 bits: their vectors straddle lines.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "gsx.h"
#include "gsx_device.h"
#include "lanes.h"
#include "matrix_tile.h"
#include "row_pieces.h"

using namespace gsx;

namespace {

constexpr int kThreads = 256;
// Workgroups of a gradient, whose partial rows are joined: two to four a compute unit, no
// more than its registers hold at once (a second generation waits for the first).  120 MB,
// gradient and join, us, with 512 / 768 / 1024: a row a lane, 5 bfloat16 columns 128 / 114 /
// 113; one piece a lane, 32 float32 70 / 69 / 72, 32 bfloat16 80 / 75 / 75; more, 64
// bfloat16 74 / 77 / 85, 512 float32 75 / 75 / 76.
constexpr int kMostGroups = 1024;
template <int V, int G, int N>
constexpr int groups_of = V == 1 ? kMostGroups : N == 1 && G <= 64 ? 768 : 512;
constexpr int kLongStrips = 256;  // of long rows, in the sums of their columns
constexpr int kFwdGroups = 8192;  // workgroups of a forward pass at most
constexpr int kMostWidth = 8192;  // of a row that a workgroup holds

struct Norm {
    const void *x, *weight, *bias, *g_y;
    int64_t rows, x_stride, g_stride;
    int width;
    float inv_width, eps;
    void *y, *g_x;
    float* parts;  // (workgroups, 2, width): dw and db, or NULL
    float* stats;  // longer rows: (rows, 3)
};

// The threads of a workgroup whose teams have G lanes.
template <int G>
constexpr int threads_of = G > kThreads ? G : kThreads;

// Sums of K values over a team of G lanes; every lane gets them.  A workgroup's team
// goes through shared memory, `turn` telling two rooms apart so that one barrier a sum
// is enough.
template <int G, int K>
__device__ __forceinline__ void team_sum(float* v, int turn) {
    constexpr int L = G < 64 ? G : 64, kWaves = G / L;
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = group_sum<L>(v[k]);
    if constexpr (kWaves > 1) {
        __shared__ float room[2][K][kWaves];
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (lane == 0) room[turn][k][wave] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            v[k] = 0.f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) v[k] += room[turn][k][w];
        }
    }
}

// (var + eps)^(-1/2): the hardware's root (a unit in the last place) and a Newton step;
// 0 where the variance overflows.
__device__ __forceinline__ float inverse_root(float v) {
    const float r = __builtin_amdgcn_rsqf(v);
    const float e = fmaf(-v * r, r, 1.f);
    return r == 0.f ? 0.f : fmaf(0.5f * r, e, r);
}

// The places of a lane's N pieces in a row.  The team's lanes hold the pieces in turn,
// so all of them but the last of each lane lie inside the row (the choice of G and N
// sees to that) and are a piece's length apart; the last ends with the row.  Its first
// `skip` elements belong to the piece before, or all of them to another lane (skip = V):
// `in` is 0 there and 1 elsewhere, and sums take them times that.  Outputs are formed
// for them, too: what two lanes write to one place is the same.
template <class E, int V, int G, int N>
struct Places {
    using P = Piece<E, V>;
    using T = typename E::T;
    int first, last, skip;
    float in[V];
    __device__ __forceinline__ Places(int width) {
        const int lane = threadIdx.x % G;
        first = lane * V;
        const int p = ((N - 1) * G + lane) * V;
        last = min(p, width - V);
        skip = min(p - last, V);
#pragma unroll
        for (int e = 0; e < V; ++e) in[e] = e >= skip ? 1.f : 0.f;
    }
    __device__ __forceinline__ int at(int k) const {
        return k < N - 1 ? first + k * G * V : last;
    }
    // element i of the lane's N V, as sums take it
    __device__ __forceinline__ float inside(int i, float v) const {
        return V == 1 || i < (N - 1) * V ? v : v * in[i - (N - 1) * V];
    }
    __device__ __forceinline__ void load(const void* rows, int64_t row, typename P::Raw* r) const {
#pragma unroll
        for (int k = 0; k < N; ++k) r[k] = P::load((const T*)rows + row + at(k));
    }
    __device__ __forceinline__ void up(const typename P::Raw* r, float* v) const {
#pragma unroll
        for (int k = 0; k < N; ++k) P::up(r[k], v + k * V);
    }
    // weights of the pieces, or `other` where there are none
    __device__ __forceinline__ void weights(const void* w, float other, float* v) const {
#pragma unroll
        for (int k = 0; k < N; ++k) {
#pragma unroll
            for (int e = 0; e < V; ++e) v[k * V + e] = other;
            if (w) P::up(P::load((const T*)w + at(k)), v + k * V);
        }
    }
    // whether element e of piece k is this lane's
    __device__ __forceinline__ bool own(int k, int e) const { return k < N - 1 || e >= skip; }
    __device__ __forceinline__ void store(void* rows, int64_t row, int k, const float* v) const {
        if (k < N - 1 || skip < V) P::store((T*)rows + row + at(k), P::down(v));
    }
};

// Differences to the rounded mean.
template <class At, int V, int G, int N>
__device__ __forceinline__ void center(const Norm& q, const At& at, float* v, int turn) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N * V; ++i)
        s = V == 1 || i < (N - 1) * V ? s + v[i] : fmaf(v[i], at.in[i - (N - 1) * V], s);
    team_sum<G, 1>(&s, turn);
    const float m = s * q.inv_width;
#pragma unroll
    for (int i = 0; i < N * V; ++i) v[i] -= m;
}

// The next row is asked for before this one's sums.
template <class E, int V, int G, int N>
__global__ __launch_bounds__(threads_of<G>) void k_norm_fwd(const Norm q) {
    using At = Places<E, V, G, N>;
    constexpr int kTeams = threads_of<G> / G;
    const At at(q.width);
    float w[N * V], b[N * V];
    at.weights(q.weight, 1.f, w);
    at.weights(q.bias, 0.f, b);
    const int64_t step = (int64_t)gridDim.x * kTeams;
    int64_t own = (int64_t)blockIdx.x * kTeams + threadIdx.x / G;
    typename At::P::Raw raw[N];
    at.load(q.x, min(own, q.rows - 1) * q.x_stride, raw);
    int turn = 0;
    // whole waves stay together, as their lanes' sums need
    for (int64_t base = (int64_t)blockIdx.x * kTeams; base < q.rows;
         base += step, own += step, turn ^= 1) {
        float v[N * V];
        at.up(raw, v);
        at.load(q.x, min(own + step, q.rows - 1) * q.x_stride, raw);
        center<At, V, G, N>(q, at, v, turn);
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < N * V; ++i) {
            const float d = at.inside(i, v[i]);
            s[0] += d;
            s[1] = fmaf(d, v[i], s[1]);
        }
        team_sum<G, 2>(s, turn);
        const float off = s[0] * q.inv_width;
        const float r = inverse_root(fmaxf(fmaf(-off, off, s[1] * q.inv_width), 0.f) + q.eps);
        const float c = -off * r;
#pragma unroll
        for (int i = 0; i < N * V; ++i) v[i] = fmaf(fmaf(v[i], r, c), w[i], b[i]);
        if (own < q.rows) {
#pragma unroll
            for (int k = 0; k < N; ++k) at.store(q.y, own * q.width, k, v + k * V);
        }
    }
}

// dx = g r + d B + A with B = -r^2 mean(g h) and A what the means leave: two products an
// element, and one more for h, which dw needs.
template <class E, int V, int G, int N>
__global__ __launch_bounds__(threads_of<G>) void k_norm_bwd(const Norm q) {
    using At = Places<E, V, G, N>;
    using Raw = typename At::P::Raw;
    constexpr int kTeams = threads_of<G> / G;
    const At at(q.width);
    float w[N * V], dw[N * V], db[N * V];
    at.weights(q.weight, 1.f, w);
#pragma unroll
    for (int i = 0; i < N * V; ++i) dw[i] = db[i] = 0.f;
    const int64_t step = (int64_t)gridDim.x * kTeams;
    int64_t own = (int64_t)blockIdx.x * kTeams + threadIdx.x / G;
    Raw raw_x[N], raw_g[N];
    at.load(q.x, min(own, q.rows - 1) * q.x_stride, raw_x);
    at.load(q.g_y, min(own, q.rows - 1) * q.g_stride, raw_g);
    int turn = 0;
    for (int64_t base = (int64_t)blockIdx.x * kTeams; base < q.rows;
         base += step, own += step, turn ^= 1) {
        const bool there = own < q.rows;
        float v[N * V], g[N * V];
        at.up(raw_x, v);
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (!there) raw_g[k] = Raw{};  // a row past the end adds nothing
            At::P::up(raw_g[k], g + k * V);
        }
        at.load(q.x, min(own + step, q.rows - 1) * q.x_stride, raw_x);
        at.load(q.g_y, min(own + step, q.rows - 1) * q.g_stride, raw_g);
        center<At, V, G, N>(q, at, v, turn);
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < N * V; ++i) {
            const float d = at.inside(i, v[i]), gw = at.inside(i, g[i] * w[i]);
            s[0] += d;
            s[1] = fmaf(d, v[i], s[1]);
            s[2] += gw;
            s[3] = fmaf(gw, v[i], s[3]);
        }
        team_sum<G, 4>(s, turn);
        const float off = s[0] * q.inv_width;
        const float r = inverse_root(fmaxf(fmaf(-off, off, s[1] * q.inv_width), 0.f) + q.eps);
        const float c = -off * r;
        const float mean_gh = fmaf(-off, s[2], s[3]) * r * q.inv_width;
        const float B = -r * mean_gh * r, A = fmaf(-off, B, -r * (s[2] * q.inv_width));
#pragma unroll
        for (int k = 0; k < N; ++k) {
            float dx[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int i = k * V + e;
                dx[e] = fmaf(g[i] * w[i], r, fmaf(v[i], B, A));
                dw[i] = fmaf(g[i], fmaf(v[i], r, c), dw[i]);
                db[i] += g[i];
            }
            if (q.g_x && there) at.store(q.g_x, own * q.width, k, dx);
        }
    }
    if (!q.parts) return;
    float* to = q.parts + (int64_t)blockIdx.x * 2 * q.width;
    if constexpr (G > 64) {
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (at.own(k, e)) {
                    to[at.at(k) + e] = dw[k * V + e];
                    to[q.width + at.at(k) + e] = db[k * V + e];
                }
    } else {
        // a wave's teams, then the waves one after another
        extern __shared__ float cols[];  // (2, width)
#pragma unroll
        for (int i = 0; i < N * V; ++i)
#pragma unroll
            for (int o = G; o < 64; o <<= 1) {
                dw[i] += __shfl_xor(dw[i], o, 64);
                db[i] += __shfl_xor(db[i], o, 64);
            }
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        for (int t = 0; t < kThreads / 64; ++t) {
            if (wave == t && lane < G) {
#pragma unroll
                for (int k = 0; k < N; ++k)
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (at.own(k, e)) {
                            float* col = cols + at.at(k) + e;
                            col[0] = t ? col[0] + dw[k * V + e] : dw[k * V + e];
                            col[q.width] = t ? col[q.width] + db[k * V + e] : db[k * V + e];
                        }
            }
            __syncthreads();
        }
        for (int i = threadIdx.x; i < 2 * q.width; i += kThreads) to[i] = cols[i];
    }
}

// ---- longer rows: a workgroup each, which reads them again for each sum ----
// (120 MB of 9000 float32 columns: 67 us forward, 112 + 46 + 10 backward)

// Calls f with the place of each piece of a row that this thread takes, and with its
// elements' shares in sums (0 for those of the piece before).
constexpr int kLongThreads = 512;
template <int V, class F>
__device__ __forceinline__ void long_pieces(const Norm& q, F f) {
    for (int p = threadIdx.x * V; p < q.width; p += kLongThreads * V) {
        const int at = min(p, q.width - V);
        float in[V];
#pragma unroll
        for (int e = 0; e < V; ++e) in[e] = e >= p - at ? 1.f : 0.f;
        f(at, in);
    }
}

template <class E>
__device__ __forceinline__ float3 long_stats(const Norm& q, const typename E::T* x) {
    constexpr int V = E::VEC;
    using P = Piece<E, V>;
    float s = 0.f;
    long_pieces<V>(q, [&](int at, const float* in) {
        float v[V];
        P::up(P::load(x + at), v);
#pragma unroll
        for (int e = 0; e < V; ++e) s = fmaf(v[e], in[e], s);
    });
    team_sum<kLongThreads, 1>(&s, 0);
    const float m = s * q.inv_width;
    float t[2] = {0.f, 0.f};
    long_pieces<V>(q, [&](int at, const float* in) {
        float v[V];
        P::up(P::load(x + at), v);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float d = (v[e] - m) * in[e];
            t[0] += d;
            t[1] = fmaf(d, d, t[1]);
        }
    });
    team_sum<kLongThreads, 2>(t, 0);
    const float off = t[0] * q.inv_width;
    const float var = fmaxf(fmaf(-off, off, t[1] * q.inv_width), 0.f);
    return make_float3(m, off, inverse_root(var + q.eps));
}

// V columns of weights, or 1 or 0 where there are none.
template <class E, int V>
__device__ __forceinline__ void long_weights(const void* w, int at, float other, float* v) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = other;
    if (w) Piece<E, V>::up(Piece<E, V>::load((const typename E::T*)w + at), v);
}

template <class E>
__global__ __launch_bounds__(kLongThreads) void k_long_fwd(const Norm q) {
    constexpr int V = E::VEC;
    using P = Piece<E, V>;
    using T = typename E::T;
    for (int64_t row = blockIdx.x; row < q.rows; row += gridDim.x) {
        const T* x = (const T*)q.x + row * q.x_stride;
        T* y = (T*)q.y + row * q.width;
        const float3 st = long_stats<E>(q, x);
        long_pieces<V>(q, [&](int at, const float*) {
            float v[V], w[V], b[V];
            P::up(P::load(x + at), v);
            long_weights<E, V>(q.weight, at, 1.f, w);
            long_weights<E, V>(q.bias, at, 0.f, b);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = fmaf((v[e] - st.x - st.y) * st.z, w[e], b[e]);
            P::store(y + at, P::down(v));
        });
    }
}

template <class E>
__global__ __launch_bounds__(kLongThreads) void k_long_bwd(const Norm q) {
    constexpr int V = E::VEC;
    using P = Piece<E, V>;
    using T = typename E::T;
    for (int64_t row = blockIdx.x; row < q.rows; row += gridDim.x) {
        const T* x = (const T*)q.x + row * q.x_stride;
        const T* dy = (const T*)q.g_y + row * q.g_stride;
        const float3 st = long_stats<E>(q, x);
        if (q.parts && threadIdx.x == 0) {
            float* to = q.stats + row * 3;
            to[0] = st.x;
            to[1] = st.y;
            to[2] = st.z;
        }
        if (!q.g_x) continue;
        auto values = [&](int at, float* h, float* g) {
            float w[V];
            P::up(P::load(x + at), h);
            P::up(P::load(dy + at), g);
            long_weights<E, V>(q.weight, at, 1.f, w);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                h[e] = (h[e] - st.x - st.y) * st.z;
                g[e] *= w[e];
            }
        };
        float s[2] = {0.f, 0.f};
        long_pieces<V>(q, [&](int at, const float* in) {
            float h[V], g[V];
            values(at, h, g);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float t = g[e] * in[e];
                s[0] += t;
                s[1] = fmaf(t, h[e], s[1]);
            }
        });
        team_sum<kLongThreads, 2>(s, 1);
        const float mean_g = s[0] * q.inv_width, mean_gh = s[1] * q.inv_width;
        T* dx = (T*)q.g_x + row * q.width;
        long_pieces<V>(q, [&](int at, const float*) {
            float h[V], g[V];
            values(at, h, g);
#pragma unroll
            for (int e = 0; e < V; ++e) g[e] = (g[e] - mean_g - h[e] * mean_gh) * st.z;
            P::store(dx + at, P::down(g));
        });
    }
}

// A strip of rows' sums of each column.
template <class E>
__global__ __launch_bounds__(kThreads) void k_long_columns(const Norm q) {
    using T = typename E::T;
    const int c = blockIdx.y * kThreads + threadIdx.x;
    if (c >= q.width) return;
    float dw = 0.f, db = 0.f;
    for (int64_t row = blockIdx.x; row < q.rows; row += gridDim.x) {
        const float* st = q.stats + row * 3;
        const float g = E::up(((const T*)q.g_y)[row * q.g_stride + c]);
        const float x = E::up(((const T*)q.x)[row * q.x_stride + c]);
        dw = fmaf(g, (x - st[0] - st[1]) * st[2], dw);
        db += g;
    }
    float* to = q.parts + (int64_t)blockIdx.x * 2 * q.width + c;
    to[0] = dw;
    to[q.width] = db;
}

// ---- the workgroups' partial rows: 16 columns a workgroup, in 64 stretches ----
// (1024 rows of 2 x 32 columns 4 us, one after another 6)

constexpr int kJoinColumns = 16, kJoinParts = 64, kJoinBatch = 16;
template <class E>
__global__ __launch_bounds__(kJoinColumns * kJoinParts) void k_norm_join(const float* parts,
                                                                         int groups, int width,
                                                                         void* g_w, void* g_b) {
    __shared__ float room[kJoinParts][kJoinColumns];
    const int col = threadIdx.x % kJoinColumns, part = threadIdx.x / kJoinColumns;
    const int c = blockIdx.x * kJoinColumns + col;
    float s = 0.f;
    if (c < 2 * width) {
        // a stretch's rows are asked for together
        for (int k = part; k < groups; k += kJoinBatch * kJoinParts) {
            float v[kJoinBatch];
#pragma unroll
            for (int u = 0; u < kJoinBatch; ++u)
                v[u] = parts[(int64_t)min(k + u * kJoinParts, groups - 1) * 2 * width + c];
#pragma unroll
            for (int u = 0; u < kJoinBatch; ++u)
                s += k + u * kJoinParts < groups ? v[u] : 0.f;
        }
    }
    for (int n = kJoinParts / 2; n > 0; n /= 2) {
        room[part][col] = s;
        __syncthreads();
        if (part < n) s += room[part + n][col];
        __syncthreads();
    }
    if (part != 0 || c >= 2 * width) return;
    typename E::T* to = (typename E::T*)(c < width ? g_w : g_b);
    if (to) to[c < width ? c : c - width] = E::down(s);
}

// ----------------------------------------------------------------- host --

int64_t up_to(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

int check_shape(int dtype, int64_t rows, int32_t width) {
    if (dtype != GSX_F32 && dtype != GSX_BF16 && dtype != GSX_F16) return GSX_ERR_INVALID;
    if (rows < 0 || width <= 0) return GSX_ERR_INVALID;
    if (rows > 1 << 30 || width > 1 << 20) return GSX_ERR_TOO_LARGE;
    return GSX_OK;
}

// What both directions check: element-aligned pointers, rows that hold the width, an
// eps that float32 holds as a normal number.
int check_args(int dtype, int64_t rows, int32_t width, const void* x, int64_t stride,
               const void* weight, float eps) {
    if (int e = check_shape(dtype, rows, width)) return e;
    const uintptr_t size = dtype == GSX_F32 ? 4 : 2;
    if (!(eps >= 1.2e-38f) || eps > 3.0e38f) return GSX_ERR_INVALID;
    if ((rows > 0 && !x) || stride < width) return GSX_ERR_INVALID;
    if ((uintptr_t)x % size || (uintptr_t)weight % size) return GSX_ERR_INVALID;
    return GSX_OK;
}


// Workgroups that walk the rows, as many rows a workgroup as it has teams.
int64_t groups_for(int64_t rows, int teams, int64_t most) {
    const int64_t n = (rows + teams - 1) / teams;
    return n < most ? n : most;
}

// For the forward pass: about four rounds each, the same for all, so that what a workgroup
// begins with (its weights) is paid for; one where there are few, more where there are
// many.  118 million bfloat16 in rows of 127, 14.8 thousand rounds in all, us: one round
// a workgroup 67, one or two 55, four 50; 400 MB in rows of 512, 49 thousand: one 172, six
// 152, twelve 158.
int64_t forward_groups(int64_t rows, int teams) {
    const int64_t rounds = (rows + teams - 1) / teams;
    int64_t groups = (rounds + 3) / 4;
    if (groups < kFwdGroups / 4) groups = kFwdGroups / 4;
    if (groups > kFwdGroups) groups = kFwdGroups;
    const int64_t each = (rounds + groups - 1) / groups;
    return (rounds + each - 1) / each;
}

// Calls f with the elements of a piece, the lanes of a team and the pieces of a lane
// that hold a row of `width`, or returns false.  n pieces take the first pair with
// G N >= n; the list goes by rising G N, so that n > G (N - 1).  (Float32 rows of 17 to 32
// columns: eight lanes with a piece each 39 us forward, four with two 46: half the line a
// load; in 16 bits four with two are ahead, 46 to 52.)
template <class E, class F>
bool for_width(int width, F f) {
    auto with = [&](auto v, auto g, auto n) { f(v, g, n); };
    if (width > kMostWidth) return false;
    auto lanes = [&](auto v) {
        constexpr int V = decltype(v)::value;
        const int n = (width + V - 1) / V;
#define GSX_TEAM(G, N)                                                  \
    if (n <= G * N)                                                     \
        return with(v, std::integral_constant<int, G>{}, std::integral_constant<int, N>{})
        if constexpr (V == 1) {
            // a row a lane
            GSX_TEAM(1, 1);
            GSX_TEAM(1, 2);
            GSX_TEAM(1, 3);
            if constexpr (E::VEC > 4) {
                GSX_TEAM(1, 4);
                GSX_TEAM(1, 5);
                GSX_TEAM(1, 6);
                GSX_TEAM(1, 7);
            }
        } else {
            GSX_TEAM(1, 1);
            GSX_TEAM(2, 1);
            GSX_TEAM(4, 1);
            if constexpr (V == 4) {
                GSX_TEAM(8, 1);
            } else {
                GSX_TEAM(4, 2);
                GSX_TEAM(4, 3);
            }
            GSX_TEAM(8, 2);
            GSX_TEAM(8, 3);
            GSX_TEAM(16, 2);
            GSX_TEAM(16, 3);
            GSX_TEAM(32, 2);
            GSX_TEAM(32, 3);
            GSX_TEAM(64, 2);
            GSX_TEAM(64, 3);
            GSX_TEAM(256, 1);
            GSX_TEAM(256, 2);
            GSX_TEAM(256, 3);
            if constexpr (V == 4) {
                GSX_TEAM(256, 4);
                GSX_TEAM(512, 3);
                GSX_TEAM(512, 4);
            } else {
                GSX_TEAM(512, 2);
            }
        }
#undef GSX_TEAM
    };
    if (width < E::VEC) lanes(std::integral_constant<int, 1>{});
    else lanes(std::integral_constant<int, E::VEC>{});
    return true;
}

template <class E>
int forward(const Norm& q, hipStream_t st) {
    const bool held = for_width<E>(q.width, [&](auto v, auto g, auto n) {
        constexpr int V = decltype(v)::value, G = decltype(g)::value, N = decltype(n)::value;
        const int64_t groups = forward_groups(q.rows, threads_of<G> / G);
        hipLaunchKernelGGL((k_norm_fwd<E, V, G, N>), dim3((unsigned)groups), dim3(threads_of<G>),
                           0, st, q);
    });
    if (!held)
        hipLaunchKernelGGL((k_long_fwd<E>), dim3((unsigned)groups_for(q.rows, 1, 1 << 16)),
                           dim3(kLongThreads), 0, st, q);
    GSX_LAUNCH_CHECK();
    return GSX_OK;
}

// Partial rows of a gradient: the workgroups that leave one, or the strips of long rows.
template <class E>
int64_t partial_rows(int64_t rows, int width) {
    int64_t groups = groups_for(rows, 1, kLongStrips);
    for_width<E>(width, [&](auto v, auto g, auto n) {
        constexpr int V = decltype(v)::value, G = decltype(g)::value, N = decltype(n)::value;
        groups = groups_for(rows, threads_of<G> / G, groups_of<V, G, N>);
    });
    return groups;
}

// A gradient's workspace: the partial rows, then a long row's statistics.
struct Layout {
    int64_t stats, total;
};

Layout layout(int dtype, int64_t rows, int width) {
    const int64_t parts = dtype == GSX_F32    ? partial_rows<F32>(rows, width)
                          : dtype == GSX_BF16 ? partial_rows<BF16>(rows, width)
                                              : partial_rows<F16>(rows, width);
    const int64_t stats = up_to(parts * 2 * width * 4, 256);
    return {stats, 256 + stats + (width > kMostWidth ? rows * 12 : 0)};
}

template <class E>
int backward(const Norm& q, void* g_w, void* g_b, hipStream_t st) {
    const int64_t groups = partial_rows<E>(q.rows, q.width);
    if (q.rows > 0) {
        const bool held = for_width<E>(q.width, [&](auto v, auto g, auto n) {
            constexpr int V = decltype(v)::value, G = decltype(g)::value, N = decltype(n)::value;
            hipLaunchKernelGGL((k_norm_bwd<E, V, G, N>), dim3((unsigned)groups), dim3(threads_of<G>),
                               (unsigned)(q.parts && G <= 64 ? 2 * q.width * 4 : 0), st, q);
        });
        if (!held) {
            hipLaunchKernelGGL((k_long_bwd<E>), dim3((unsigned)groups_for(q.rows, 1, 1 << 16)),
                               dim3(kLongThreads), 0, st, q);
            GSX_LAUNCH_CHECK();
            if (q.parts)
                hipLaunchKernelGGL((k_long_columns<E>),
                                   dim3((unsigned)groups,
                                        (unsigned)((q.width + kThreads - 1) / kThreads)),
                                   dim3(kThreads), 0, st, q);
        }
        GSX_LAUNCH_CHECK();
    }
    if (q.parts) {
        hipLaunchKernelGGL((k_norm_join<E>),
                           dim3((unsigned)((2 * q.width + kJoinColumns - 1) / kJoinColumns)),
                           dim3(kJoinColumns * kJoinParts), 0, st, q.parts, (int)groups, q.width,
                           g_w, g_b);
        GSX_LAUNCH_CHECK();
    }
    return GSX_OK;
}

}  // namespace

extern "C" {

int gsx_layer_norm_fwd(int32_t dtype, int64_t rows, int32_t width, const void* x, int64_t x_stride,
                       const void* weight, const void* bias, float eps, void* y, void* stream) {
    if (int e = check_args(dtype, rows, width, x, x_stride, weight, eps)) return e;
    const uintptr_t size = dtype == GSX_F32 ? 4 : 2;
    if ((uintptr_t)bias % size || (uintptr_t)y % size) return GSX_ERR_INVALID;
    if (rows == 0) return GSX_OK;
    if (!y) return GSX_ERR_INVALID;
    Norm q{};
    q.x = x;
    q.x_stride = x_stride;
    q.weight = weight;
    q.bias = bias;
    q.rows = rows;
    q.width = width;
    q.inv_width = 1.0f / (float)width;
    q.eps = eps;
    q.y = y;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == GSX_F32) return forward<F32>(q, st);
    if (dtype == GSX_BF16) return forward<BF16>(q, st);
    return forward<F16>(q, st);
}

int64_t gsx_layer_norm_bwd_workspace_bytes(int32_t dtype, int64_t rows, int32_t width) {
    if (int e = check_shape(dtype, rows, width)) return e;
    return layout(dtype, rows, width).total;
}

int gsx_layer_norm_bwd(int32_t dtype, int64_t rows, int32_t width, const void* x, int64_t x_stride,
                       const void* weight, const void* g_y, int64_t g_y_stride, float eps,
                       void* g_x, void* g_weight, void* g_bias, void* workspace,
                       int64_t workspace_bytes, void* stream) {
    if (int e = check_args(dtype, rows, width, x, x_stride, weight, eps)) return e;
    const uintptr_t size = dtype == GSX_F32 ? 4 : 2;
    if ((rows > 0 && !g_y) || g_y_stride < width) return GSX_ERR_INVALID;
    if ((uintptr_t)g_y % size || (uintptr_t)g_x % size || (uintptr_t)g_weight % size ||
        (uintptr_t)g_bias % size || (uintptr_t)workspace % 16)
        return GSX_ERR_INVALID;
    const bool params = g_weight || g_bias;
    if (!params && (!g_x || rows == 0)) return GSX_OK;
    const Layout l = layout(dtype, rows, width);
    if (params && (!workspace || workspace_bytes < l.total)) return GSX_ERR_WORKSPACE;
    Norm q{};
    q.x = x;
    q.x_stride = x_stride;
    q.weight = weight;
    q.g_y = g_y;
    q.g_stride = g_y_stride;
    q.rows = rows;
    q.width = width;
    q.inv_width = 1.0f / (float)width;
    q.eps = eps;
    q.g_x = g_x;
    q.parts = params ? (float*)workspace : nullptr;
    q.stats = (float*)((char*)workspace + l.stats);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == GSX_F32) return backward<F32>(q, g_weight, g_bias, st);
    if (dtype == GSX_BF16) return backward<BF16>(q, g_weight, g_bias, st);
    return backward<F16>(q, g_weight, g_bias, st);
}

}  // extern "C"
