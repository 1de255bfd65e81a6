// distil.hip -- the loss of a student's logits against the few largest that a
// teacher kept for each row, and its gradient.
//
// Row by row, with temperature T, student z = s / T, q = softmax(z), and the
// row's entries (value t_k, index i_k):
//   teacher logits:     p = softmax(t / T) over the entries
//   teacher log-probs:  p = exp(t), and r = max(0, 1 - sum p) for the rest of
//                       the vocabulary, one bucket of student mass Q
//   L = T^2 [sum_k p_k (log p_k - log q_{i_k})  (+ r (log r - log Q))]
//   dL/ds_j = T [S q_j - sum_{k: i_k = j} p_k   (- r q_j / Q where j has no entry)]
// with S = sum p (+ r).  An entry whose index lies outside the vocabulary or
// whose value is -inf is absent; a row without entries has loss 0 and gradient
// 0 whatever its logits hold, and the mean does not count it.  The bucket is
// left out where the student has no mass outside the entries.
//
// The entries' columns are taken out of the row (set to -inf) once their
// logits are read, so that the sum over the rest is a sum and no difference of
// two: Q keeps its relative accuracy however small it is, and the rest has its
// own running maximum.  Statistics are float32, sums over rows double.
//
// Rows up to kRowBytes: a workgroup stages whole rows in shared memory in one
// flat copy (rows of odd length need no alignment), G lanes share a row, and
// the gradient goes back over the staged logits and out in one flat copy: each
// logit is read once and each gradient written once.  Longer rows are cut into
// segments, so that few rows still fill the chip: one launch leaves every
// segment's maximum and sum, a second joins them, a third writes the gradient.
#include <hip/hip_runtime.h>

#include <cmath>

#include "gsx.h"
#include "gsx_device.h"
#include "matrix_tile.h"

using namespace gsx;

namespace {

constexpr int kThreads = 256;
constexpr int kRowBytes = 8192;    // longest row of the one-launch path
constexpr int kSegBytes = 16384;   // a segment of a longer row
constexpr int kCountParts = 256;   // workgroups of the count of supervised rows
constexpr float kLog2e = 1.44269504088896341f;

struct Distil {
    const void* logits;
    int64_t stride;
    const float* values;
    const void* indices;
    int index64;
    int64_t rows;
    int vocab, top;
    float temp, inv_temp;
    int log_probs;
    float* loss_rows;        // or NULL
    double* loss_parts;      // a sum for each workgroup, or NULL
    void* grad;              // or NULL
    const float* upstream;   // one for each row, or one, or NULL (scale alone)
    int upstream_rows;
    const int* counts;       // kCountParts counts of supervised rows (mean), or NULL
    float scale;
    float* seg_parts;        // longer rows: (rows, segments, 2) maximum and sum
    float* stats;            // longer rows: (rows, 8)
    int seg, segs;
};

struct Entry {
    int index;  // -1: absent
    float value;
};

__device__ __forceinline__ Entry entry(const Distil& q, int64_t row, int k) {
    const int64_t at = row * q.top + k;
    const int64_t i = q.index64 ? ((const int64_t*)q.indices)[at] : ((const int32_t*)q.indices)[at];
    const float v = q.values[at];
    return Entry{(i >= 0 && i < q.vocab && v != -INFINITY) ? (int)i : -1, v};
}

template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
    return v;
}
template <int G>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, kWave));
    return v;
}

// exp((s - m) / T) as a power of two; c = log2(e) / T.  m is the maximum, so
// the product's rounding matters only where the term itself is small.
__device__ __forceinline__ float expo(float s, float m, float c) {
    return __builtin_amdgcn_exp2f((s - m) * c);
}

// What the entries and the rest of a row say: the loss, and what the gradient
// needs.  rest_m, rest_s: maximum logit and sum of exp over the rest (-inf, 0:
// nothing there).  Runs on G lanes; ei, ep, es: the row's entries in shared
// memory (index, value then probability, logit).
struct RowStats {
    float loss;     // without T^2
    float m, inv;   // maximum over all, S / (sum of exp over all)
    float rest;     // the rest's factor on exp((s - rest_m) / T)
    bool active;
};

template <int G>
__device__ __forceinline__ RowStats row_stats(const Distil& q, int lane, const int* ei, float* ep,
                                              const float* es, float rest_m, float rest_s) {
    const float c = kLog2e * q.inv_temp;
    float tm = -INFINITY, m = rest_m;
    int any = 0;
    for (int k = lane; k < q.top; k += G)
        if (ei[k] >= 0) {
            any = 1;
            tm = fmaxf(tm, ep[k]);
            m = fmaxf(m, es[k]);
        }
    RowStats r;
    r.active = group_max<G>((float)any) > 0.f;
    tm = group_max<G>(tm);
    m = group_max<G>(m);
    const bool has_rest = rest_m != -INFINITY;
    float total = 0.f, t_sum = 0.f;
    for (int k = lane; k < q.top; k += G)
        if (ei[k] >= 0) {
            bool again = false;  // a column that two entries name counts once
            for (int j = 0; j < k; ++j) again |= ei[j] == ei[k];
            if (!again) total += es[k] == -INFINITY ? 0.f : expo(es[k], m, c);
            t_sum += q.log_probs ? 0.f : expo(ep[k], tm, c);
        }
    const float shift = has_rest ? expo(rest_m, m, c) : 0.f;
    total = group_sum<G>(total) + (has_rest ? rest_s * shift : 0.f);
    t_sum = group_sum<G>(t_sum);
    const float log_total = logf(total), log_t = logf(t_sum);
    float loss = 0.f, mass = 0.f;
    for (int k = lane; k < q.top; k += G)
        if (ei[k] >= 0) {
            float lp, p;
            if (q.log_probs) {
                lp = ep[k];
                p = expf(lp);
            } else {
                lp = (ep[k] - tm) * q.inv_temp - log_t;
                p = expo(ep[k], tm, c) / t_sum;
            }
            if (p != 0.f) loss += p * (lp - ((es[k] - m) * q.inv_temp - log_total));
            mass += p;
            ep[k] = p;
        }
    loss = group_sum<G>(loss);
    mass = group_sum<G>(mass);
    float share = 0.f;
    if (q.log_probs && has_rest) {
        const float left = 1.0f - mass;
        if (left > 0.f) {
            const float log_q = (rest_m - m) * q.inv_temp + logf(rest_s) - log_total;
            loss += left * (logf(left) - log_q);
            share = left / rest_s;
            mass += left;
        }
    }
    r.loss = loss;
    r.m = m;
    r.inv = mass / total;
    r.rest = r.inv * shift - share;
    return r;
}

// The factor on a row's gradient: T, the upstream gradient, 1 / supervised rows.
__device__ __forceinline__ float row_scale(const Distil& q, int64_t row, float inv_count) {
    float s = q.scale * q.temp * inv_count;
    if (q.upstream) s *= q.upstream[q.upstream_rows ? row : 0];
    return s;
}

// 1 / supervised rows (1 where nothing asks for the mean), from the count's parts.
__device__ __forceinline__ float inverse_count(const Distil& q, int* scratch) {
    if (!q.counts) return 1.f;
    int v = threadIdx.x < kCountParts ? q.counts[threadIdx.x] : 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    int n = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) n += scratch[w];
    __syncthreads();
    return 1.f / (float)(n > 0 ? n : 1);
}

// n elements from global to shared memory or back, where both have the same
// offset from a 16-byte boundary: whole 16-byte pieces between ragged ends.
template <class T>
__device__ __forceinline__ void copy_flat(T* dst, const T* src, int64_t n) {
    constexpr int V = 16 / sizeof(T);
    int64_t head = (V - ((uintptr_t)src / sizeof(T)) % V) % V;
    if (head > n) head = n;
    const int64_t body = (n - head) / V;
    for (int64_t i = threadIdx.x; i < head; i += kThreads) dst[i] = src[i];
    for (int64_t i = threadIdx.x; i < body; i += kThreads)
        *(u32x4*)(dst + head + i * V) = *(const u32x4*)(src + head + i * V);
    for (int64_t i = head + body * V + threadIdx.x; i < n; i += kThreads) dst[i] = src[i];
}

// Rows in shared memory, G lanes each.  LDS: the rows (with up to a piece of
// slack so that they lie as in global memory), then the entries.
template <class E, int G>
__global__ __launch_bounds__(kThreads) void k_rows(const Distil q) {
    using T = typename E::T;
    constexpr int R = kThreads / G;
    extern __shared__ u32x4 smem[];
    __shared__ int scratch[kThreads / 64];
    __shared__ double sums[R];
    const int64_t row0 = (int64_t)blockIdx.x * R;
    const int n_rows = q.rows - row0 < R ? (int)(q.rows - row0) : R;
    const int64_t n = (int64_t)n_rows * q.vocab;
    const T* src = (const T*)q.logits + row0 * q.stride;
    const bool flat = q.stride == q.vocab;
    T* tile = (T*)smem + (flat ? ((uintptr_t)src % 16) / sizeof(T) : 0);
    const int64_t tile_bytes = ((int64_t)R * q.vocab * sizeof(T) + 31) / 16 * 16;
    int* ei = (int*)((char*)smem + tile_bytes);
    float* ep = (float*)(ei + R * q.top);
    float* es = ep + R * q.top;
    const int sub = threadIdx.x / G, lane = threadIdx.x % G;
    const int64_t row = row0 + sub;
    const bool mine = sub < n_rows;
    T* my = tile + (int64_t)sub * q.vocab;
    ei += sub * q.top;
    ep += sub * q.top;
    es += sub * q.top;

    if (flat)
        copy_flat(tile, src, n);
    else if (mine)
        for (int j = lane; j < q.vocab; j += G) my[j] = src[(int64_t)sub * q.stride + j];
    const float inv_count = q.grad ? inverse_count(q, scratch) : 1.f;
    if (mine)
        for (int k = lane; k < q.top; k += G) {
            const Entry e = entry(q, row, k);
            ei[k] = e.index;
            ep[k] = e.value;
        }
    __syncthreads();
    if (mine)
        for (int k = lane; k < q.top; k += G) es[k] = ei[k] >= 0 ? E::up(my[ei[k]]) : 0.f;
    __syncthreads();
    if (mine)
        for (int k = lane; k < q.top; k += G)
            if (ei[k] >= 0) my[ei[k]] = E::down(-INFINITY);
    __syncthreads();
    const float c = kLog2e * q.inv_temp;
    RowStats r{};
    float rest_m = -INFINITY;
    if (mine) {
        for (int j = lane; j < q.vocab; j += G) rest_m = fmaxf(rest_m, E::up(my[j]));
        rest_m = group_max<G>(rest_m);
        float rest_s = 0.f;
        for (int j = lane; j < q.vocab; j += G) {
            const float s = E::up(my[j]);
            rest_s += s == -INFINITY ? 0.f : expo(s, rest_m, c);
        }
        rest_s = group_sum<G>(rest_s);
        r = row_stats<G>(q, lane, ei, ep, es, rest_m, rest_s);
        if (lane == 0) {
            const float loss = r.active ? q.temp * q.temp * r.loss : 0.f;
            if (q.loss_rows) q.loss_rows[row] = loss;
            sums[sub] = loss;
        }
    } else if (lane == 0) {
        sums[sub] = 0.0;
    }
    __syncthreads();  // the entries' probabilities too
    if (q.loss_parts && threadIdx.x == 0) {
        double s = 0.0;
        for (int i = 0; i < R; ++i) s += sums[i];
        q.loss_parts[blockIdx.x] = s;
    }
    if (!q.grad) return;
    if (mine) {
        if (!r.active) {
            for (int j = lane; j < q.vocab; j += G) my[j] = E::down(0.f);
        } else {
            const float f = row_scale(q, row, inv_count);
            const float rest = r.rest * f;
            for (int j = lane; j < q.vocab; j += G) {
                const float s = E::up(my[j]);
                my[j] = E::down(s == -INFINITY ? 0.f * rest : expo(s, rest_m, c) * rest);
            }
        }
    }
    __syncthreads();
    if (mine && r.active) {
        const float f = row_scale(q, row, inv_count);
        for (int k = lane; k < q.top; k += G)
            if (ei[k] >= 0) {
                float p = 0.f;
                for (int j = 0; j < q.top; ++j)
                    if (ei[j] == ei[k]) p += ep[j];
                const float e = es[k] == -INFINITY ? 0.f : expo(es[k], r.m, c);
                my[ei[k]] = E::down(f * (e * r.inv - p));
            }
    }
    __syncthreads();
    T* dst = (T*)q.grad + row0 * q.vocab;
    if (flat && ((uintptr_t)dst - (uintptr_t)src) % 16 == 0)
        copy_flat(dst, tile, n);
    else
        for (int64_t i = threadIdx.x; i < n; i += kThreads) dst[i] = tile[i];
}

// A segment of a longer row: maximum and sum of its rest.
template <class E>
__global__ __launch_bounds__(kThreads) void k_seg_sum(const Distil q) {
    using T = typename E::T;
    __shared__ u32x4 smem[kSegBytes / 16 + 1];
    __shared__ float red[kThreads / 64];
    const int64_t row = blockIdx.x / q.segs;
    const int seg = (int)(blockIdx.x % q.segs);
    const int j0 = seg * q.seg, n = q.vocab - j0 < q.seg ? q.vocab - j0 : q.seg;
    const T* src = (const T*)q.logits + row * q.stride + j0;
    T* tile = (T*)smem + ((uintptr_t)src % 16) / sizeof(T);
    copy_flat(tile, src, n);
    __syncthreads();
    for (int k = threadIdx.x; k < q.top; k += kThreads) {
        const int i = entry(q, row, k).index - j0;
        if (i >= 0 && i < n) tile[i] = E::down(-INFINITY);
    }
    __syncthreads();
    const float c = kLog2e * q.inv_temp;
    float m = -INFINITY;
    for (int j = threadIdx.x; j < n; j += kThreads) m = fmaxf(m, E::up(tile[j]));
    m = group_max<64>(m);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) m = fmaxf(m, red[w]);
    float s = 0.f;
    for (int j = threadIdx.x; j < n; j += kThreads) {
        const float v = E::up(tile[j]);
        s += v == -INFINITY ? 0.f : expo(v, m, c);
    }
    s = group_sum<64>(s);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.f;
#pragma unroll
        for (int w = 0; w < kThreads / 64; ++w) s += red[w];
        q.seg_parts[2 * blockIdx.x] = m;
        q.seg_parts[2 * blockIdx.x + 1] = s;
    }
}

// Joins a row's segments: its loss, and what the gradient's launch reads.  One
// wave for a row.
template <class E>
__global__ __launch_bounds__(64) void k_seg_join(const Distil q) {
    using T = typename E::T;
    extern __shared__ u32x4 smem[];
    int* ei = (int*)smem;
    float* ep = (float*)(ei + q.top);
    float* es = ep + q.top;
    const int64_t row = blockIdx.x;
    const int lane = threadIdx.x;
    const T* src = (const T*)q.logits + row * q.stride;
    for (int k = lane; k < q.top; k += 64) {
        const Entry e = entry(q, row, k);
        ei[k] = e.index;
        ep[k] = e.value;
        es[k] = e.index >= 0 ? E::up(src[e.index]) : 0.f;
    }
    __syncthreads();
    const float c = kLog2e * q.inv_temp;
    const float* parts = q.seg_parts + row * q.segs * 2;
    float m = -INFINITY, s = 0.f;
    for (int i = lane; i < q.segs; i += 64) m = fmaxf(m, parts[2 * i]);
    m = group_max<64>(m);
    for (int i = lane; i < q.segs; i += 64) {
        const float pm = parts[2 * i], ps = parts[2 * i + 1];
        s += pm == -INFINITY ? ps : ps * expo(pm, m, c);  // ps is 0, or NaN
    }
    s = group_sum<64>(s);
    const RowStats r = row_stats<64>(q, lane, ei, ep, es, m, s);
    if (lane == 0) {
        const float loss = r.active ? q.temp * q.temp * r.loss : 0.f;
        if (q.loss_rows) q.loss_rows[row] = loss;
        if (q.loss_parts) q.loss_parts[row] = loss;
        float* st = q.stats + row * 8;
        st[0] = m;
        st[1] = r.rest;
        st[2] = r.m;
        st[3] = r.inv;
        st[4] = r.active ? 1.f : 0.f;
    }
    // the entries' probabilities, for the gradient
    float* probs = q.stats + q.rows * 8 + row * q.top;
    for (int k = lane; k < q.top; k += 64) probs[k] = ep[k];
}

// A segment's gradient.
template <class E>
__global__ __launch_bounds__(kThreads) void k_seg_grad(const Distil q) {
    using T = typename E::T;
    __shared__ u32x4 smem[kSegBytes / 16 + 1];
    __shared__ int scratch[kThreads / 64];
    const int64_t row = blockIdx.x / q.segs;
    const int seg = (int)(blockIdx.x % q.segs);
    const int j0 = seg * q.seg, n = q.vocab - j0 < q.seg ? q.vocab - j0 : q.seg;
    const T* src = (const T*)q.logits + row * q.stride + j0;
    T* dst = (T*)q.grad + row * q.vocab + j0;
    T* tile = (T*)smem + ((uintptr_t)src % 16) / sizeof(T);
    const float inv_count = inverse_count(q, scratch);
    const float* st = q.stats + row * 8;
    const bool active = st[4] != 0.f;
    const float f = row_scale(q, row, inv_count);
    const float c = kLog2e * q.inv_temp;
    const float rest_m = st[0], rest = st[1] * f;
    if (active) copy_flat(tile, src, n);
    __syncthreads();
    for (int j = threadIdx.x; j < n; j += kThreads) {
        float g = 0.f;
        if (active) {
            const float s = E::up(tile[j]);
            g = s == -INFINITY ? 0.f * rest : expo(s, rest_m, c) * rest;
        }
        tile[j] = E::down(g);
    }
    __syncthreads();
    if (active) {
        const float* probs = q.stats + q.rows * 8 + row * q.top;
        for (int k = threadIdx.x; k < q.top; k += kThreads) {
            const int i = entry(q, row, k).index;
            if (i < j0 || i >= j0 + n) continue;
            float p = 0.f;
            for (int j = 0; j < q.top; ++j)
                if (entry(q, row, j).index == i) p += probs[j];
            const float s = E::up(src[i - j0]);
            const float e = s == -INFINITY ? 0.f : expo(s, st[2], c);
            tile[i - j0] = E::down(f * (e * st[3] - p));
        }
    }
    __syncthreads();
    if (((uintptr_t)dst - (uintptr_t)src) % 16 == 0)
        copy_flat(dst, tile, n);
    else
        for (int i = threadIdx.x; i < n; i += kThreads) dst[i] = tile[i];
}

// Rows that have an entry, a count for each of kCountParts workgroups.
__global__ __launch_bounds__(kThreads) void k_count(const Distil q, int* counts) {
    __shared__ int red[kThreads / 64];
    int n = 0;
    for (int64_t row = (int64_t)blockIdx.x * kThreads + threadIdx.x; row < q.rows;
         row += (int64_t)kCountParts * kThreads) {
        int any = 0;
        for (int k = 0; k < q.top && !any; ++k) any = entry(q, row, k).index >= 0;
        n += any;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, kWave);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        n = 0;
#pragma unroll
        for (int w = 0; w < kThreads / 64; ++w) n += red[w];
        counts[blockIdx.x] = n;
    }
}

// The sum (or mean) of the rows' losses, in a fixed order.
__global__ __launch_bounds__(kThreads) void k_total(const double* parts, int64_t n,
                                                    const int* counts, float scale, float* out) {
    __shared__ double red[kThreads];
    __shared__ int cnt[kThreads];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += kThreads) s += parts[i];
    red[threadIdx.x] = s;
    cnt[threadIdx.x] = counts && threadIdx.x < kCountParts ? counts[threadIdx.x] : 0;
    __syncthreads();
    for (int o = kThreads / 2; o > 0; o >>= 1) {
        if (threadIdx.x < o) {
            red[threadIdx.x] += red[threadIdx.x + o];
            cnt[threadIdx.x] += cnt[threadIdx.x + o];
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        const double d = counts ? (cnt[0] > 0 ? cnt[0] : 1) : 1.0;
        *out = (float)(red[0] * scale / d);
    }
}

// ----------------------------------------------------------------- host --

int64_t up_to(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

int check_shape(int dtype, int64_t rows, int64_t vocab, int64_t top) {
    if (dtype != GSX_F32 && dtype != GSX_BF16 && dtype != GSX_F16) return GSX_ERR_INVALID;
    if (rows < 0 || vocab <= 0 || top <= 0) return GSX_ERR_INVALID;
    if (top > vocab) return GSX_ERR_INVALID;
    if (rows >= (1LL << 30) || vocab >= (1LL << 30) || top > GSX_DISTIL_MAX_TOP)
        return GSX_ERR_TOO_LARGE;
    return GSX_OK;
}

int elem(int dtype) { return dtype == GSX_F32 ? 4 : 2; }
bool short_rows(int dtype, int64_t vocab) { return vocab * elem(dtype) <= kRowBytes; }

// Lanes for a row: about eight logits each, 4 to 64.
int lanes_for(int64_t vocab) {
    int g = 4;
    while (g < 64 && g * 8 < vocab) g *= 2;
    return g;
}

// The workspace: the count's parts, the workgroups' losses, then for longer
// rows the segments' sums, the rows' statistics and the entries' probabilities.
struct Layout {
    int64_t parts, segs, stats, total;
    int64_t n_parts;
    int seg, n_segs;
};
Layout layout(int dtype, int64_t rows, int64_t vocab, int64_t top) {
    Layout l{};
    l.parts = kCountParts * 4;
    if (short_rows(dtype, vocab)) {
        const int r = kThreads / lanes_for(vocab);
        l.n_parts = (rows + r - 1) / r;
        l.segs = l.stats = l.total = up_to(l.parts + l.n_parts * 8, 256);
        return l;
    }
    l.seg = kSegBytes / elem(dtype);
    l.n_segs = (int)((vocab + l.seg - 1) / l.seg);
    l.n_parts = rows;
    l.segs = up_to(l.parts + l.n_parts * 8, 256);
    l.stats = up_to(l.segs + rows * l.n_segs * 8, 256);
    l.total = up_to(l.stats + rows * (8 + top) * 4, 256);
    return l;
}

template <class E, int G>
int launch_rows(const Distil& q, hipStream_t st) {
    constexpr int R = kThreads / G;
    const int64_t blocks = (q.rows + R - 1) / R;
    const int64_t tile = ((int64_t)R * q.vocab * sizeof(typename E::T) + 31) / 16 * 16;
    const int64_t lds = tile + (int64_t)R * q.top * 12;
    if (blocks >= (1LL << 31) || lds > 160 * 1024 - 4096) return GSX_ERR_TOO_LARGE;
    hipLaunchKernelGGL((k_rows<E, G>), dim3((unsigned)blocks), dim3(kThreads), (unsigned)lds, st,
                       q);
    GSX_LAUNCH_CHECK();
    return GSX_OK;
}

template <class E>
int run_rows(const Distil& q, hipStream_t st) {
    switch (lanes_for(q.vocab)) {
        case 4: return launch_rows<E, 4>(q, st);
        case 8: return launch_rows<E, 8>(q, st);
        case 16: return launch_rows<E, 16>(q, st);
        case 32: return launch_rows<E, 32>(q, st);
        default: return launch_rows<E, 64>(q, st);
    }
}

// Loss (stats) and, where asked for, gradient.  `sums`: form the statistics;
// false: they are in the workspace (the gradient of an earlier forward).
template <class E>
int run(const Distil& q, bool sums, hipStream_t st) {
    if (q.segs == 0) return run_rows<E>(q, st);
    const int64_t blocks = q.rows * q.segs;
    if (blocks >= (1LL << 31)) return GSX_ERR_TOO_LARGE;
    if (sums) {
        hipLaunchKernelGGL((k_seg_sum<E>), dim3((unsigned)blocks), dim3(kThreads), 0, st, q);
        GSX_LAUNCH_CHECK();
        hipLaunchKernelGGL((k_seg_join<E>), dim3((unsigned)q.rows), dim3(64),
                           (unsigned)(q.top * 12), st, q);
        GSX_LAUNCH_CHECK();
    }
    if (q.grad) {
        hipLaunchKernelGGL((k_seg_grad<E>), dim3((unsigned)blocks), dim3(kThreads), 0, st, q);
        GSX_LAUNCH_CHECK();
    }
    return GSX_OK;
}

int run_any(int dtype, const Distil& q, bool sums, hipStream_t st) {
    if (dtype == GSX_F32) return run<F32>(q, sums, st);
    if (dtype == GSX_BF16) return run<BF16>(q, sums, st);
    return run<F16>(q, sums, st);
}

struct Args {
    int32_t dtype;
    int64_t rows;
    int32_t vocab, top;
    const void* logits;
    int64_t stride;
    const float* values;
    const void* indices;
    int32_t index64;
    float temperature;
    int32_t teacher, reduction;
    void* workspace;
    int64_t workspace_bytes;
};

int check_args(const Args& a) {
    if (int e = check_shape(a.dtype, a.rows, a.vocab, a.top)) return e;
    if (!(a.temperature > 0.f) || a.temperature > 3.0e38f) return GSX_ERR_INVALID;
    if (a.teacher != GSX_TEACHER_LOGITS && a.teacher != GSX_TEACHER_LOG_PROBS)
        return GSX_ERR_INVALID;
    if (a.reduction != GSX_REDUCE_NONE && a.reduction != GSX_REDUCE_SUM &&
        a.reduction != GSX_REDUCE_MEAN)
        return GSX_ERR_INVALID;
    if (a.index64 != 0 && a.index64 != 1) return GSX_ERR_INVALID;
    if (a.rows > 0 && (!a.logits || !a.values || !a.indices || a.stride < a.vocab))
        return GSX_ERR_INVALID;
    if ((uintptr_t)a.logits % elem(a.dtype) || (uintptr_t)a.values % 4 ||
        (uintptr_t)a.indices % (a.index64 ? 8 : 4))
        return GSX_ERR_INVALID;
    if (!a.workspace || (uintptr_t)a.workspace % 16) return GSX_ERR_INVALID;
    if (a.workspace_bytes < layout(a.dtype, a.rows, a.vocab, a.top).total)
        return GSX_ERR_WORKSPACE;
    return GSX_OK;
}

Distil problem(const Args& a, const Layout& l) {
    Distil q{};
    q.logits = a.logits;
    q.stride = a.stride;
    q.values = a.values;
    q.indices = a.indices;
    q.index64 = a.index64;
    q.rows = a.rows;
    q.vocab = a.vocab;
    q.top = a.top;
    q.temp = a.temperature;
    q.inv_temp = 1.0f / a.temperature;
    q.log_probs = a.teacher == GSX_TEACHER_LOG_PROBS;
    q.scale = 1.0f;
    char* ws = (char*)a.workspace;
    q.counts = a.reduction == GSX_REDUCE_MEAN ? (const int*)ws : nullptr;
    q.seg_parts = (float*)(ws + l.segs);
    q.stats = (float*)(ws + l.stats);
    q.seg = l.seg;
    q.segs = l.n_segs;
    return q;
}

int forward(const Args& a, float scale, float* loss, void* grad, void* stream) {
    if (int e = check_args(a)) return e;
    if (!loss && (a.rows > 0 || a.reduction != GSX_REDUCE_NONE)) return GSX_ERR_INVALID;
    if ((uintptr_t)loss % 4 || (uintptr_t)grad % elem(a.dtype)) return GSX_ERR_INVALID;
    hipStream_t st = (hipStream_t)stream;
    const Layout l = layout(a.dtype, a.rows, a.vocab, a.top);
    Distil q = problem(a, l);
    q.scale = scale;
    q.grad = grad;
    double* parts = (double*)((char*)a.workspace + l.parts);
    if (a.reduction == GSX_REDUCE_NONE)
        q.loss_rows = loss;
    else
        q.loss_parts = parts;
    if (a.reduction == GSX_REDUCE_MEAN) {
        hipLaunchKernelGGL(k_count, dim3(kCountParts), dim3(kThreads), 0, st, q,
                           (int*)a.workspace);
        GSX_LAUNCH_CHECK();
    }
    if (a.rows > 0)
        if (int e = run_any(a.dtype, q, true, st)) return e;
    if (a.reduction != GSX_REDUCE_NONE) {
        hipLaunchKernelGGL(k_total, dim3(1), dim3(kThreads), 0, st, parts,
                           a.rows > 0 ? l.n_parts : 0, q.counts, scale, loss);
        GSX_LAUNCH_CHECK();
    }
    return GSX_OK;
}

}  // namespace

extern "C" {

int64_t gsx_distil_workspace_bytes(int32_t dtype, int64_t rows, int32_t vocab, int32_t top) {
    if (int e = check_shape(dtype, rows, vocab, top)) return e;
    return layout(dtype, rows, vocab, top).total;
}

int gsx_distil_fwd(int32_t dtype, int64_t rows, int32_t vocab, int32_t top, const void* logits,
                   int64_t logits_stride, const float* values, const void* indices,
                   int32_t index64, float temperature, int32_t teacher, int32_t reduction,
                   float* loss, void* workspace, int64_t workspace_bytes, void* stream) {
    const Args a{dtype,   rows,    vocab,       top,     logits,    logits_stride, values,
                 indices, index64, temperature, teacher, reduction, workspace,     workspace_bytes};
    return forward(a, 1.0f, loss, nullptr, stream);
}

int gsx_distil_fwd_bwd(int32_t dtype, int64_t rows, int32_t vocab, int32_t top, const void* logits,
                       int64_t logits_stride, const float* values, const void* indices,
                       int32_t index64, float temperature, int32_t teacher, int32_t reduction,
                       float scale, float* loss, void* g_logits, void* workspace,
                       int64_t workspace_bytes, void* stream) {
    const Args a{dtype,   rows,    vocab,       top,     logits,    logits_stride, values,
                 indices, index64, temperature, teacher, reduction, workspace,     workspace_bytes};
    if (reduction == GSX_REDUCE_NONE || (rows > 0 && !g_logits)) return GSX_ERR_INVALID;
    return forward(a, scale, loss, g_logits, stream);
}

int gsx_distil_bwd(int32_t dtype, int64_t rows, int32_t vocab, int32_t top, const void* logits,
                   int64_t logits_stride, const float* values, const void* indices,
                   int32_t index64, float temperature, int32_t teacher, int32_t reduction,
                   const float* g_loss, void* g_logits, void* workspace, int64_t workspace_bytes,
                   void* stream) {
    const Args a{dtype,   rows,    vocab,       top,     logits,    logits_stride, values,
                 indices, index64, temperature, teacher, reduction, workspace,     workspace_bytes};
    if (int e = check_args(a)) return e;
    if (rows == 0) return GSX_OK;
    if (!g_loss || !g_logits || (uintptr_t)g_loss % 4 || (uintptr_t)g_logits % elem(dtype))
        return GSX_ERR_INVALID;
    Distil q = problem(a, layout(dtype, rows, vocab, top));
    q.grad = g_logits;
    q.upstream = g_loss;
    q.upstream_rows = reduction == GSX_REDUCE_NONE;
    return run_any(dtype, q, false, (hipStream_t)stream);
}

}  // extern "C"
