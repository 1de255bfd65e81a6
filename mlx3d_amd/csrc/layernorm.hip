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
constexpr int kWaves = kThreads / 64;
constexpr int kMostGroups = 1024;  // workgroups of a gradient, whose partial rows are joined
constexpr int kPieces = 4;         // of a row on a lane at most

struct Norm {
    const void *x, *weight, *bias, *g_y;
    int64_t rows, x_stride, g_stride;
    int width;
    float inv_width, eps;
    void *y, *g_x;
    float* parts;  // (workgroups, 2, width): dw and db, or NULL
    float* stats;  // longer rows: (rows, 3)
};

// Sums of K values over a team of G lanes; every lane gets them.  A workgroup's team
// goes through shared memory, `turn` telling two rooms apart so that one barrier a sum
// is enough.
template <int G, int K>
__device__ __forceinline__ void team_sum(float* v, int turn) {
    constexpr int L = G < 64 ? G : 64;
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = group_sum<L>(v[k]);
    if constexpr (G > 64) {
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

// The places of a lane's N pieces in a row: where each begins, and how many of its
// elements belong to the piece before (all of them: the lane has no such piece).
template <int V, int G, int N>
struct Places {
    int at[N], skip[N];
    __device__ __forceinline__ Places(int width) {
        const int lane = threadIdx.x % G;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int p = (k * G + lane) * V;
            at[k] = min(p, width - V);
            skip[k] = min(p - at[k], V);
        }
    }
};

// Differences to the rounded mean, zero outside the row.
template <int V, int G, int N>
__device__ __forceinline__ void center(const Norm& q, const Places<V, G, N>& at, float* v,
                                       int turn) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) s += e >= at.skip[k] ? v[k * V + e] : 0.f;
    team_sum<G, 1>(&s, turn);
    const float m = s * q.inv_width;
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) v[k * V + e] -= m;
}

template <class E, int V, int G, int N>
__global__ __launch_bounds__(kThreads) void k_norm_fwd(const Norm q) {
    using P = Piece<E, V>;
    using T = typename E::T;
    constexpr int kTeams = kThreads / G;
    const Places<V, G, N> at(q.width);
    float w[N * V], b[N * V];
#pragma unroll
    for (int i = 0; i < N * V; ++i) w[i] = 1.f, b[i] = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        if (q.weight) P::up(P::load((const T*)q.weight + at.at[k]), w + k * V);
        if (q.bias) P::up(P::load((const T*)q.bias + at.at[k]), b + k * V);
    }
    const int64_t step = (int64_t)gridDim.x * kTeams;
    int turn = 0;
    // whole waves stay together, as their lanes' sums need
    for (int64_t base = (int64_t)blockIdx.x * kTeams; base < q.rows; base += step, turn ^= 1) {
        const int64_t own = base + threadIdx.x / G, row = min(own, q.rows - 1);
        float v[N * V];
#pragma unroll
        for (int k = 0; k < N; ++k)
            P::up(P::load((const T*)q.x + row * q.x_stride + at.at[k]), v + k * V);
        center<V, G, N>(q, at, v, turn);
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = e >= at.skip[k] ? v[k * V + e] : 0.f;
                s[0] += d;
                s[1] = fmaf(d, d, s[1]);
            }
        team_sum<G, 2>(s, turn);
        const float off = s[0] * q.inv_width;
        const float r = 1.0f / sqrtf(fmaxf(fmaf(-off, off, s[1] * q.inv_width), 0.f) + q.eps);
#pragma unroll
        for (int k = 0; k < N; ++k) {
#pragma unroll
            for (int e = 0; e < V; ++e)
                v[k * V + e] = fmaf((v[k * V + e] - off) * r, w[k * V + e], b[k * V + e]);
            if (own < q.rows && at.skip[k] < V)
                P::store((T*)q.y + row * q.width + at.at[k], P::down(v + k * V));
        }
    }
}

template <class E, int V, int G, int N>
__global__ __launch_bounds__(kThreads) void k_norm_bwd(const Norm q) {
    using P = Piece<E, V>;
    using T = typename E::T;
    constexpr int kTeams = kThreads / G;
    const Places<V, G, N> at(q.width);
    float w[N * V], dw[N * V], db[N * V];
#pragma unroll
    for (int i = 0; i < N * V; ++i) w[i] = 1.f, dw[i] = db[i] = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k)
        if (q.weight) P::up(P::load((const T*)q.weight + at.at[k]), w + k * V);
    const int64_t step = (int64_t)gridDim.x * kTeams;
    int turn = 0;
    for (int64_t base = (int64_t)blockIdx.x * kTeams; base < q.rows; base += step, turn ^= 1) {
        const int64_t own = base + threadIdx.x / G, row = min(own, q.rows - 1);
        float v[N * V], g[N * V];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            P::up(P::load((const T*)q.x + row * q.x_stride + at.at[k]), v + k * V);
            P::up(P::load((const T*)q.g_y + row * q.g_stride + at.at[k]), g + k * V);
        }
        center<V, G, N>(q, at, v, turn);
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int i = k * V + e;
                const bool in = e >= at.skip[k];
                const float d = in ? v[i] : 0.f, gw = in ? g[i] * w[i] : 0.f;
                s[0] += d;
                s[1] = fmaf(d, d, s[1]);
                s[2] += gw;
                s[3] = fmaf(gw, d, s[3]);
            }
        team_sum<G, 4>(s, turn);
        const float off = s[0] * q.inv_width;
        const float r = 1.0f / sqrtf(fmaxf(fmaf(-off, off, s[1] * q.inv_width), 0.f) + q.eps);
        const float mean_g = s[2] * q.inv_width;
        const float mean_gh = fmaf(-off, s[2], s[3]) * r * q.inv_width;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            float dx[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int i = k * V + e;
                const float h = (v[i] - off) * r;
                dx[e] = (g[i] * w[i] - mean_g - h * mean_gh) * r;
                if (own < q.rows && e >= at.skip[k]) {
                    dw[i] = fmaf(g[i], h, dw[i]);
                    db[i] += g[i];
                }
            }
            if (q.g_x && own < q.rows && at.skip[k] < V)
                P::store((T*)q.g_x + row * q.width + at.at[k], P::down(dx));
        }
    }
    if (!q.parts) return;
    float* to = q.parts + (int64_t)blockIdx.x * 2 * q.width;
    if constexpr (G > 64) {
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (e >= at.skip[k]) {
                    to[at.at[k] + e] = dw[k * V + e];
                    to[q.width + at.at[k] + e] = db[k * V + e];
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
        for (int t = 0; t < kWaves; ++t) {
            if (wave == t && lane < G) {
#pragma unroll
                for (int k = 0; k < N; ++k)
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (e >= at.skip[k]) {
                            float* c = cols + at.at[k] + e;
                            c[0] = t ? c[0] + dw[k * V + e] : dw[k * V + e];
                            c[q.width] = t ? c[q.width] + db[k * V + e] : db[k * V + e];
                        }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < 2 * q.width; c += kThreads) to[c] = cols[c];
    }
}

// ---- longer rows: a workgroup each, element by element ----

template <class E>
__device__ __forceinline__ float3 long_stats(const Norm& q, const typename E::T* x) {
    float s = 0.f;
    for (int c = threadIdx.x; c < q.width; c += kThreads) s += E::up(x[c]);
    team_sum<kThreads, 1>(&s, 0);
    const float m = s * q.inv_width;
    float t[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < q.width; c += kThreads) {
        const float d = E::up(x[c]) - m;
        t[0] += d;
        t[1] = fmaf(d, d, t[1]);
    }
    team_sum<kThreads, 2>(t, 0);
    const float off = t[0] * q.inv_width;
    const float var = fmaxf(fmaf(-off, off, t[1] * q.inv_width), 0.f);
    return make_float3(m, off, 1.0f / sqrtf(var + q.eps));
}

template <class E>
__global__ __launch_bounds__(kThreads) void k_long_fwd(const Norm q) {
    using T = typename E::T;
    for (int64_t row = blockIdx.x; row < q.rows; row += gridDim.x) {
        const T* x = (const T*)q.x + row * q.x_stride;
        T* y = (T*)q.y + row * q.width;
        const float3 st = long_stats<E>(q, x);
        for (int c = threadIdx.x; c < q.width; c += kThreads) {
            const float w = q.weight ? E::up(((const T*)q.weight)[c]) : 1.f;
            const float b = q.bias ? E::up(((const T*)q.bias)[c]) : 0.f;
            y[c] = E::down(fmaf((E::up(x[c]) - st.x - st.y) * st.z, w, b));
        }
    }
}

template <class E>
__global__ __launch_bounds__(kThreads) void k_long_bwd(const Norm q) {
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
        float s[2] = {0.f, 0.f};
        for (int c = threadIdx.x; c < q.width; c += kThreads) {
            const float g = E::up(dy[c]) * (q.weight ? E::up(((const T*)q.weight)[c]) : 1.f);
            s[0] += g;
            s[1] = fmaf(g, (E::up(x[c]) - st.x - st.y) * st.z, s[1]);
        }
        team_sum<kThreads, 2>(s, 1);
        const float mean_g = s[0] * q.inv_width, mean_gh = s[1] * q.inv_width;
        T* dx = (T*)q.g_x + row * q.width;
        for (int c = threadIdx.x; c < q.width; c += kThreads) {
            const float g = E::up(dy[c]) * (q.weight ? E::up(((const T*)q.weight)[c]) : 1.f);
            const float h = (E::up(x[c]) - st.x - st.y) * st.z;
            dx[c] = E::down((g - mean_g - h * mean_gh) * st.z);
        }
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

constexpr int kJoinColumns = 16, kJoinParts = 64;
template <class E>
__global__ __launch_bounds__(kJoinColumns * kJoinParts) void k_norm_join(const float* parts,
                                                                         int groups, int width,
                                                                         void* g_w, void* g_b) {
    __shared__ float room[kJoinParts][kJoinColumns];
    const int col = threadIdx.x % kJoinColumns, part = threadIdx.x / kJoinColumns;
    const int c = blockIdx.x * kJoinColumns + col;
    float s = 0.f;
    if (c < 2 * width)
        for (int k = part; k < groups; k += kJoinParts) s += parts[(int64_t)k * 2 * width + c];
    room[part][col] = s;
    __syncthreads();
    if (part != 0 || c >= 2 * width) return;
    for (int k = 1; k < kJoinParts; ++k) s += room[k][col];
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

bool is_long(int dtype, int width) {
    return width > kThreads * kPieces * (dtype == GSX_F32 ? F32::VEC : BF16::VEC);
}

// Workgroups that walk the rows, as many rows a workgroup as it has teams.
int64_t groups_for(int64_t rows, int teams, int64_t most) {
    const int64_t n = (rows + teams - 1) / teams;
    return n < most ? n : most;
}

// Calls f with the elements of a piece, the lanes of a team and the pieces of a lane
// that hold a row of `width`, or returns false.
template <class E, class F>
bool for_width(int width, F f) {
    auto with = [&](auto v, auto g, auto n) { f(v, g, n); };
    auto lanes = [&](auto v) {
        constexpr int V = decltype(v)::value;
        const int n = (width + V - 1) / V;
#define GSX_TEAM(G, N)                                                  \
    if (n <= G * N)                                                     \
        return with(v, std::integral_constant<int, G>{}, std::integral_constant<int, N>{})
        GSX_TEAM(1, 1);
        GSX_TEAM(2, 1);
        GSX_TEAM(4, 1);
        GSX_TEAM(8, 1);
        if constexpr (V > 1) {
            GSX_TEAM(16, 1);
            GSX_TEAM(32, 1);
            GSX_TEAM(64, 1);
            GSX_TEAM(64, 2);
            GSX_TEAM(64, 4);
            GSX_TEAM(256, 2);
            GSX_TEAM(256, 4);
        }
#undef GSX_TEAM
    };
    if (width > kThreads * kPieces * E::VEC) return false;
    if (width < E::VEC) lanes(std::integral_constant<int, 1>{});
    else lanes(std::integral_constant<int, E::VEC>{});
    return true;
}

template <class E>
int forward(const Norm& q, hipStream_t st) {
    const bool held = for_width<E>(q.width, [&](auto v, auto g, auto n) {
        constexpr int V = decltype(v)::value, G = decltype(g)::value, N = decltype(n)::value;
        const int64_t groups = groups_for(q.rows, kThreads / G, 1 << 16);
        hipLaunchKernelGGL((k_norm_fwd<E, V, G, N>), dim3((unsigned)groups), dim3(kThreads), 0, st,
                           q);
    });
    if (!held)
        hipLaunchKernelGGL((k_long_fwd<E>), dim3((unsigned)groups_for(q.rows, 1, 1 << 16)),
                           dim3(kThreads), 0, st, q);
    GSX_LAUNCH_CHECK();
    return GSX_OK;
}

template <class E>
int backward(const Norm& q, void* g_w, void* g_b, hipStream_t st) {
    int64_t groups = 0;
    if (q.rows > 0) {
        const bool held = for_width<E>(q.width, [&](auto v, auto g, auto n) {
            constexpr int V = decltype(v)::value, G = decltype(g)::value, N = decltype(n)::value;
            groups = groups_for(q.rows, kThreads / G, kMostGroups);
            hipLaunchKernelGGL((k_norm_bwd<E, V, G, N>), dim3((unsigned)groups), dim3(kThreads),
                               (unsigned)(q.parts && G <= 64 ? 2 * q.width * 4 : 0), st, q);
        });
        if (!held) {
            hipLaunchKernelGGL((k_long_bwd<E>), dim3((unsigned)groups_for(q.rows, 1, 1 << 16)),
                               dim3(kThreads), 0, st, q);
            GSX_LAUNCH_CHECK();
            groups = groups_for(q.rows, 1, kMostGroups);
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
    const int64_t most = rows < kMostGroups ? rows : kMostGroups;
    return 256 + up_to(most * 2 * width * 4, 256) + (is_long(dtype, width) ? rows * 12 : 0);
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
    if (params &&
        (!workspace || workspace_bytes < gsx_layer_norm_bwd_workspace_bytes(dtype, rows, width)))
        return GSX_ERR_WORKSPACE;
    const int64_t most = rows < kMostGroups ? rows : kMostGroups;
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
    q.stats = (float*)((char*)workspace + up_to(most * 2 * width * 4, 256));
    hipStream_t st = (hipStream_t)stream;
    if (dtype == GSX_F32) return backward<F32>(q, g_weight, g_bias, st);
    if (dtype == GSX_BF16) return backward<BF16>(q, g_weight, g_bias, st);
    return backward<F16>(q, g_weight, g_bias, st);
}

}  // extern "C"
