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
// own running maximum.  Statistics are float32, sums over rows double.  Powers are
// the hardware's (a unit in the last place, and their exponent's rounding); a row's
// few logarithms and quotients are the library's, 3 us of 186 at 921 600 rows of 150.
//
// Rows up to kRowBytes: a wave takes as many whole rows as its registers hold, G
// lanes a row, through shared memory in one flat copy (rows of odd length need no
// alignment); the gradient goes out the same way, so each logit is read once and
// each gradient written once.  Longer rows are cut into segments, so that few rows
// still fill the chip: one launch leaves every segment's maximum and sum, a second
// joins them, a third reads the logits again and writes the gradient.
#include <hip/hip_runtime.h>

#include <cmath>

#include "gsx.h"
#include "gsx_device.h"
#include "lanes.h"
#include "matrix_tile.h"

using namespace gsx;

namespace {

constexpr int kThreads = 256;
// Longest row of the one-launch path: where a wave's registers still hold it.
// Against segments, us a call (32 768 and 4 rows): float32 512 columns 45 / 138 and
// 17 / 30, 2048 columns 122 / 237 and 18 / 29, bf16 4096 148 / 260 and 18 / 29.
constexpr int kRowBytes = 8192;
constexpr int kSegBytes = 16384;   // a segment of a longer row
constexpr int kCountParts = 256;   // workgroups of the count of supervised rows

struct Distil {
    const void* logits;
    int64_t stride;
    const float* values;
    const void* indices;
    int index64;
    int64_t rows;
    int vocab, top;
    float temp, c, c_lo;     // T, log2(e) / T and what its rounding left
    int log_probs;
    float* loss_rows;        // or NULL
    double* loss_parts;      // a sum for each workgroup, or NULL
    void* grad;              // or NULL
    const float* upstream;   // one for each row, or one, or NULL (scale alone)
    int upstream_rows;
    const int* counts;       // kCountParts counts of supervised rows
    float scale;
    int mean;
    int alone;               // one workgroup walks all rows, and counts them itself
    float* total;            // ... and their sum or mean goes here, or NULL
    float* seg_parts;        // longer rows: (rows, segments, 2) maximum and sum
    float* stats;            // longer rows: (rows, 8)
    int seg, segs;
};

struct Entry {
    int index;  // -1: absent
    float value;
};

// An entry as it lies in memory; told apart from its check so that the loads
// can be in flight for a while.
struct RawEntry {
    int lo, hi;
    float value;
};
__device__ __forceinline__ RawEntry raw_entry(const Distil& q, int64_t row, int k) {
    const int64_t at = row * q.top + k;
    RawEntry e;
    e.value = q.values[at];
    e.hi = 0;
    if (q.index64) {
        const int2 i = ((const int2*)q.indices)[at];
        e.lo = i.x;
        e.hi = i.y;
    } else {
        e.lo = ((const int*)q.indices)[at];
    }
    return e;
}
__device__ __forceinline__ Entry checked(const Distil& q, const RawEntry& e) {
    const bool in = e.hi == 0 && (unsigned)e.lo < (unsigned)q.vocab && e.value != -INFINITY;
    return Entry{in ? e.lo : -1, e.value};
}
__device__ __forceinline__ Entry entry(const Distil& q, int64_t row, int k) {
    return checked(q, raw_entry(q, row, k));
}

// exp((s - m) / T) as the power 2^((s - m) c) with c = log2(e) / T.  The difference
// comes first: it is 0 at the maximum whatever its size, so a row, a rest or a
// segment that only holds a mask's finite lowest value has equal parts, where
// s c - m c would round m c by many powers of two (from |m| of 1e9 on) or
// overflow.  m is finite; s may be -inf (0).
__device__ __forceinline__ float expo(float s, float m, float c) {
    return __builtin_amdgcn_exp2f((s - m) * c);
}

constexpr float kLn2 = 0.69314718055994531f;

// The same to the power's own rounding: what the exponent's product and c lost, to
// first order.  For float32 logits and for a row's few entries; of 16-bit logits
// the gradient's rounding is thousands of times as large.  4099 rows of 50 000
// float32 485 us without, 504 with it; the error against 64 bits 1.7 and 1.0 times
// that of elementary operations.
__device__ __forceinline__ float expo(const Distil& q, float s, float m) {
    const float d = s - m, e = d * q.c, r = __builtin_amdgcn_exp2f(e);
    const float lost = fmaf(d, q.c_lo, fmaf(d, q.c, -e));  // e may be infinite where r is 0
    return r == 0.f ? 0.f : fmaf(r, lost * kLn2, r);
}
template <class E>
__device__ __forceinline__ float expo_of(const Distil& q, float s, float m) {
    if constexpr (sizeof(typename E::T) == 4) return expo(q, s, m);
    return expo(s, m, q.c);
}

// A row's entries on G lanes, KPL in a lane's registers: entry lane + i G.
template <int KPL>
struct Entries {
    int index[KPL];
    float value[KPL];  // the teacher's, then the probability
    float s[KPL];      // the student's logit
    bool again[KPL];   // another entry stands for this column
};
template <int G, int KPL>
__device__ __forceinline__ void read_entries(const Distil& q, int64_t row, int lane,
                                             Entries<KPL>& e) {
#pragma unroll
    for (int i = 0; i < KPL; ++i) {
        e.index[i] = -1;
        if (lane + i * G < q.top) {
            const Entry t = entry(q, row, lane + i * G);
            e.index[i] = t.index;
            e.value[i] = t.value;
        }
    }
}

// What the entries and the rest of a row say: the loss, and what the gradient
// needs.  rest_m, rest_s: maximum logit and sum of exp over the rest (-inf, 0:
// nothing there).  Turns the entries' values into their probabilities.
//
// The loss is summed times T^2, T log q and the like: T^2 p (log p - log q) is
// p T (T (log p + log total) - (s - m)), which needs no quotient by T that could
// overflow next to a mask.
struct RowStats {
    float loss;
    float m, inv;   // the maximum over all, S / (sum of exp over all)
    float rest;     // the rest's factor on exp((s - rest_m) / T)
    bool active;
};

// (A teacher of logits: rest_m and rest_s run over the whole row, the entries'
// columns among them.)
template <int G, int KPL, bool LOG_PROBS>
__device__ __forceinline__ RowStats row_stats(const Distil& q, Entries<KPL>& e, float rest_m,
                                              float rest_s) {
    const float temp = q.temp;
    float tm = -INFINITY, m = rest_m, any = 0.f;
#pragma unroll
    for (int i = 0; i < KPL; ++i)
        if (e.index[i] >= 0) {
            any = 1.f;
            tm = fmaxf(tm, e.value[i]);
            m = fmaxf(m, e.s[i]);
        }
    RowStats r;
    r.active = group_max<G>(any) > 0.f;
    // NaN leaves no maximum; a sum over anything else than -inf is 1 or more
    const bool has_rest = rest_s != 0.f;
    float total = rest_s, shift = 1.f;
    if constexpr (LOG_PROBS) {
        m = group_max<G>(m);
        shift = has_rest ? expo(q, rest_m, m) : 0.f;
        total = 0.f;
#pragma unroll
        for (int i = 0; i < KPL; ++i)
            if (e.index[i] >= 0 && !e.again[i] && e.s[i] != -INFINITY)
                total += expo(q, e.s[i], m);
        total = group_sum<G>(total) + (has_rest ? rest_s * shift : 0.f);
    } else {
        m = rest_m;
    }
    const float log_total = logf(total);
    float loss = 0.f, mass = 0.f, t_exp[KPL], inv_t = 1.f, log_t = 0.f;
    if constexpr (!LOG_PROBS) {
        tm = group_max<G>(tm);
        float t_sum = 0.f;
#pragma unroll
        for (int i = 0; i < KPL; ++i)
            if (e.index[i] >= 0) {
                t_exp[i] = expo(q, e.value[i], tm);
                t_sum += t_exp[i];
            }
        t_sum = group_sum<G>(t_sum);
        log_t = logf(t_sum);
        inv_t = 1.0f / t_sum;
    }
#pragma unroll
    for (int i = 0; i < KPL; ++i)
        if (e.index[i] >= 0) {
            float lp, p;  // T log p
            if constexpr (LOG_PROBS) {
                lp = temp * e.value[i];
                p = expf(e.value[i]);
            } else {
                lp = (e.value[i] - tm) - temp * log_t;
                p = t_exp[i] * inv_t;
            }
            if (p != 0.f) loss += (p * temp) * (fmaf(temp, log_total, lp) - (e.s[i] - m));
            mass += p;
            e.value[i] = p;
        }
    loss = group_sum<G>(loss);
    mass = group_sum<G>(mass);
    float share = 0.f;
    if (LOG_PROBS && has_rest) {
        const float left = 1.0f - mass;
        if (left > 0.f) {
            const float logs = logf(left) - logf(rest_s) + log_total;
            loss += (left * temp) * (temp * logs - (rest_m - m));
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

// An entry's gradient without the row's factor; p: the column's probability.
__device__ __forceinline__ float entry_grad(const Distil& q, const RowStats& r, float s, float p) {
    return (s == -INFINITY ? 0.f : expo(q, s, r.m)) * r.inv - p;
}

// The factor on a row's gradient: T, the upstream gradient, 1 / supervised rows.
__device__ __forceinline__ float row_scale(const Distil& q, int64_t row, float inv_count) {
    float s = q.scale * q.temp * inv_count;
    if (q.upstream) s *= q.upstream[q.upstream_rows ? row : 0];
    return s;
}

// Whether a row has an entry: most rows show one in their first, otherwise eight
// are in flight at a time.
__device__ __forceinline__ int supervised(const Distil& q, int64_t row) {
    int found = entry(q, row, 0).index >= 0;
    for (int k = 1; k < q.top && !found; k += 8) {
        RawEntry e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = raw_entry(q, row, k + j < q.top ? k + j : 0);
#pragma unroll
        for (int j = 0; j < 8; ++j) found |= checked(q, e[j]).index >= 0;
    }
    return found;
}

// 1 / supervised rows (1 where nothing asks for the mean), from the count's parts,
// or by the one workgroup that there is.
__device__ __forceinline__ float inverse_count(const Distil& q, int* scratch) {
    if (!q.mean) return 1.f;
    int v = 0;
    if (q.alone) {
        for (int64_t row = threadIdx.x; row < q.rows; row += kThreads) v += supervised(q, row);
    } else {
        v = threadIdx.x < kCountParts ? q.counts[threadIdx.x] : 0;
    }
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
// By THREADS threads, t the caller's number among them.
template <int THREADS, class T>
__device__ __forceinline__ void copy_flat(T* dst, const T* src, int n, int t) {
    constexpr int V = 16 / sizeof(T);
    int head = (int)((V - ((uintptr_t)src / sizeof(T)) % V) % V);
    if (head > n) head = n;
    const int body = (n - head) / V, tail = n - head - body * V;
    const u32x4* from = (const u32x4*)(src + head);
    u32x4* to = (u32x4*)(dst + head);
    for (int i = t; i < body; i += THREADS) to[i] = from[i];
    if (t < head) dst[t] = src[t];
    if (t < tail) dst[n - tail + t] = src[n - tail + t];
}

// The 16-byte pieces of a wave's tile on their way to shared memory: the span of `n`
// elements at `src`, widened to whole pieces.  The few elements of a piece that
// reaches over an end of the tensor [lo, hi) are copied one by one.
template <class T, int P>
struct Ahead {
    static constexpr int V = 16 / sizeof(T);
    u32x4 r[P];
    // the pieces [first, last) that lie in the tensor, counted from src rounded down
    static __device__ __forceinline__ void span(const T* src, int n, const T* lo, const T* hi,
                                                unsigned& first, unsigned& count) {
        const uintptr_t base = (uintptr_t)src & ~(uintptr_t)15;
        first = base < (uintptr_t)lo ? 1 : 0;
        const uintptr_t stop = (uintptr_t)(src + n);
        const unsigned last = (unsigned)((stop - base + (stop > ((uintptr_t)hi & ~(uintptr_t)15)
                                                             ? 0 : 15)) / 16);
        count = last > first ? last - first : 0;
    }
    __device__ __forceinline__ void load(const T* src, int n, const T* lo, const T* hi, unsigned lane) {
        unsigned first, count;
        span(src, n, lo, hi, first, count);
        const u32x4* p = (const u32x4*)((uintptr_t)src & ~(uintptr_t)15);
#pragma unroll
        for (unsigned i = 0; i < P; ++i)
            if (lane + i * 64 - first < count) r[i] = p[lane + i * 64];
    }
    __device__ __forceinline__ void store(u32x4* lds, const T* src, int n, const T* lo, const T* hi,
                                          unsigned lane) const {
        unsigned first, count;
        span(src, n, lo, hi, first, count);
#pragma unroll
        for (unsigned i = 0; i < P; ++i)
            if (lane + i * 64 - first < count)
                lds[lane + i * 64] = r[i];
        const T* stop = src + n;
        const int off = (int)((uintptr_t)src % 16 / sizeof(T));
        T* at = (T*)lds + off;
        if (off && src == lo && lane < V - off && (int)lane < n)
            at[lane] = src[lane];
        // also before a last tile of so few elements that this one ends in the last piece
        const unsigned tail = (unsigned)((uintptr_t)stop % 16 / sizeof(T));
        if ((uintptr_t)stop > ((uintptr_t)hi & ~(uintptr_t)15) && lane < tail && (int)lane < n)
            at[n - 1 - lane] = src[n - 1 - lane];
    }
};

// Shared memory of a tile: its rows with up to 15 bytes before them, and as many
// words behind the last row's beginning as a group reads (the row among them).
__host__ __device__ inline int64_t tile_room(int rows, int words, int64_t vocab, int size) {
    return ((int64_t)(rows - 1) * vocab * size + 16 + 4 * (int64_t)words + 15) / 16 * 16;
}

// Whole rows in shared memory, G lanes each, N 32-bit words and KPL entries of a
// row in a lane's registers.  Each wave walks tiles of 64 / G rows by itself, with
// no barrier: the next tile's loads are in flight while one is worked on, and
// the waves of a unit cover each other's waits.  The logits' exponentials are
// formed once, for the sum, and kept for the gradient.
//
// A row of 16-bit elements may begin inside a word: the elements beside the
// row are masked on the way in, and written around on the way out.  Entries
// that name one column find each other through the column itself: each leaves
// its number there, and one of them reads its own back.  A teacher of logits
// has no bucket, so there the row's sum runs over all columns at once; with one
// of log-probabilities the entries' columns are taken out first.
//
// FULL: words of a lane that lie in every row that this kernel is launched for.
//
// 921 600 rows of 150 bf16 logits and 8 entries, loss and gradient: 166 us,
// 3.7 TB/s (a large copy: 4.8).  A tile's loads, its arithmetic and its stores
// follow each other in a wave, and four waves of a SIMD do not cover all of it; six
// spill.  Stores held back behind the next tile's loads took 7 us more.
template <class E, int G, int N, int KPL, bool LOG_PROBS, int FULL>
__global__ __launch_bounds__(kThreads, N > 14 ? 2 : KPL > 2 ? 3 : 4) void k_rows(const Distil q,
                                                                               int64_t tiles) {
    using T = typename E::T;
    constexpr int R = 64 / G;
    constexpr int W = 4 / sizeof(T);                // elements of a word
    constexpr int P = (R * G * N * 4 / 16 + 64) / 64;  // pieces of a lane
    constexpr int kWaves = kThreads / 64;
    extern __shared__ u32x4 smem[];
    __shared__ int scratch[kThreads / 64];
    __shared__ double sums[kWaves];
    const bool flat = q.stride == q.vocab;
    const T* logits = (const T*)q.logits;
    const T* end = logits + q.rows * q.vocab;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sub = (threadIdx.x & 63) / G, lane = threadIdx.x % G;
    const unsigned l64 = threadIdx.x & 63;
    const int64_t room = tile_room(R, G * N, q.vocab, sizeof(T));
    u32x4* lds = (u32x4*)((char*)smem + wave * room);
    // index and probability of the row's entries, where some name one column
    int* ei = (int*)((char*)smem + kWaves * room) + (wave * R + sub) * q.top;
    float* ep = (float*)ei + kWaves * R * q.top;
    const float inv_count = q.grad || q.total ? inverse_count(q, scratch) : 1.f;
    double group_loss = 0.0;

    Ahead<T, P> ahead;
    RawEntry next[KPL];
    auto rows_of = [&](int64_t t) {
        return q.rows - t * R < R ? (int)(q.rows - t * R) : R;
    };
    auto fetch = [&](int64_t t) {
        const int n_rows = rows_of(t);
        if (flat) ahead.load(logits + t * R * q.vocab, n_rows * q.vocab, logits, end, l64);
        if (sub < n_rows) {
#pragma unroll
            for (int i = 0; i < KPL; ++i)
                if (lane + i * G < q.top) next[i] = raw_entry(q, t * R + sub, lane + i * G);
        }
    };
    const int64_t first = (int64_t)blockIdx.x * kWaves + wave, step = (int64_t)gridDim.x * kWaves;
    if (first < tiles) fetch(first);
    for (int64_t t = first; t < tiles; t += step) {
        const int64_t row0 = t * R, row = row0 + sub;
        const int n_rows = rows_of(t);
        const int n = n_rows * q.vocab;
        const bool mine = sub < n_rows;
        const T* src = logits + row0 * q.stride;
        const int shift = flat ? (int)((uintptr_t)src % 16 / sizeof(T)) : 0;
        T* tile = (T*)lds + shift;
        const int e0 = shift + sub * q.vocab;
        T* my = (T*)lds + e0;
        if (flat) {
            ahead.store(lds, src, n, logits, end, l64);
        } else if (mine) {
#pragma unroll 1
            for (int j = lane; j < q.vocab; j += G) my[j] = src[(int64_t)sub * q.stride + j];
        }
        Entries<KPL> e;
#pragma unroll
        for (int i = 0; i < KPL; ++i) {
            const Entry x = checked(q, next[i]);
            e.index[i] = mine && lane + i * G < q.top ? x.index : -1;
            e.value[i] = x.value;
        }
        wave_fence();
        if (t + step < tiles) fetch(t + step);
        if (mine) {
            bool shared = false;
            auto mark = [&] {  // each entry's number in its column
                wave_fence();
#pragma unroll
                for (int i = 0; i < KPL; ++i)
                    if (e.index[i] >= 0) my[e.index[i]] = E::tag(lane + i * G);
                wave_fence();
            };
            auto find = [&] {
#pragma unroll
                for (int i = 0; i < KPL; ++i) {
                    e.again[i] = e.index[i] >= 0 && !E::is_tag(my[e.index[i]], lane + i * G);
                    shared |= e.again[i];
                }
            };
#pragma unroll
            for (int i = 0; i < KPL; ++i) e.s[i] = e.index[i] >= 0 ? E::up(my[e.index[i]]) : 0.f;
            if constexpr (LOG_PROBS) {
                mark();
                find();
                wave_fence();
#pragma unroll
                for (int i = 0; i < KPL; ++i)
                    if (e.index[i] >= 0) my[e.index[i]] = E::down(-INFINITY);
                wave_fence();
            }
            // the row: words into registers, elements beside it at -inf
            const int skip = W == 2 ? e0 & 1 : 0;
            uint32_t* words = (uint32_t*)lds + e0 / W;
            const int l0 = here(lane);
            float v[N * W];
            float rest_m = -INFINITY;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                // past the row's end: what lies there (the tile has room) is masked
                const int w = l0 + i * G;
                const uint32_t raw = words[w];
#pragma unroll
                for (int h = 0; h < W; ++h) {
                    float x = W == 1 ? __uint_as_float(raw) : E::up((T)(raw >> (16 * h)));
                    if (i >= FULL || i == 0) {
                        const unsigned j = (unsigned)(W * w - skip + h);
                        x = j < (unsigned)q.vocab ? x : -INFINITY;
                    }
                    v[i * W + h] = x;
                    rest_m = fmaxf(rest_m, v[i * W + h]);
                }
            }
            if constexpr (!LOG_PROBS) {
                if (q.grad) mark();
            }
            rest_m = group_max<G>(rest_m);
            const float ref = rest_m == -INFINITY ? 0.f : rest_m;
            float rest_s = 0.f;
#pragma unroll
            for (int i = 0; i < N * W; ++i) {
                v[i] = expo_of<E>(q, v[i], ref);
                rest_s += v[i];
            }
            rest_s = group_sum<G>(rest_s);
            const RowStats r = row_stats<G, KPL, LOG_PROBS>(q, e, rest_m, rest_s);
            if (lane == 0) {
                const float loss = r.active ? r.loss : 0.f;
                if (q.loss_rows) q.loss_rows[row] = loss;
                group_loss += loss;
            }
            if (q.grad) {
                if constexpr (!LOG_PROBS) find();
                const float f = r.active ? row_scale(q, row, inv_count) : 0.f;
                if (!r.active && !(rest_s < INFINITY)) {  // whatever its logits hold
#pragma unroll
                    for (int i = 0; i < N * W; ++i) v[i] = 0.f;
                }
                const float factor = r.active ? r.rest * f : 0.f;
                const int l1 = here(lane);
                wave_fence();
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int w = l1 + i * G;
                    const int j = W * w - skip;
                    if constexpr (W == 1) {
                        if (i < FULL || j < q.vocab) words[w] = __float_as_uint(v[i] * factor);
                    } else {
                        const uint32_t two = E::pair(v[2 * i] * factor, v[2 * i + 1] * factor);
                        if (i > 0 && i < FULL) {
                            words[w] = two;
                            continue;
                        }
                        if ((unsigned)j < (unsigned)(q.vocab - 1)) words[w] = two;
                        if (j == q.vocab - 1) my[j] = (T)two;
                        if (i == 0 && j < 0) my[0] = (T)(two >> 16);
                    }
                }
                // the entries' columns, over what was written there
                if (__builtin_expect(__any(shared), 0)) {
#pragma unroll
                    for (int i = 0; i < KPL; ++i)
                        if (lane + i * G < q.top) {
                            ei[lane + i * G] = e.index[i];
                            ep[lane + i * G] = e.value[i];
                        }
                    wave_fence();
#pragma unroll
                    for (int i = 0; i < KPL; ++i)
                        if (e.index[i] >= 0) {
                            float p = 0.f;
#pragma unroll 1
                            for (int k = 0; k < q.top; ++k)
                                if (ei[k] == e.index[i]) p += ep[k];
                            e.value[i] = p;
                        }
                }
                wave_fence();
#pragma unroll
                for (int i = 0; i < KPL; ++i)
                    if (e.index[i] >= 0)
                        my[e.index[i]] = E::down(f * entry_grad(q, r, e.s[i], e.value[i]));
            }
        }
        wave_fence();
        if (q.grad) {
            T* dst = (T*)q.grad + row0 * q.vocab;
            if (flat && ((uintptr_t)dst - (uintptr_t)src) % 16 == 0) {
                copy_flat<64>(dst, (const T*)tile, n, (int)l64);
            } else {
#pragma unroll 1
                for (int i = (int)l64; i < n; i += 64) dst[i] = tile[i];
            }
        }
        wave_fence();  // the tile is read before the next one is stored
    }
    if (!q.loss_parts && !q.total) return;
#pragma unroll
    for (int o = G; o < 64; o *= 2) group_loss += __shfl_xor(group_loss, o, kWave);
    if (l64 == 0) sums[wave] = group_loss;
    __syncthreads();
    if (threadIdx.x == 0) {
        double s = 0.0;
        for (int i = 0; i < kWaves; ++i) s += sums[i];
        if (q.total)
            *q.total = (float)(s * (double)q.scale * (double)inv_count);
        else
            q.loss_parts[blockIdx.x] = s;
    }
}

// A segment of a longer row: maximum and sum of its rest (with a teacher of
// logits, of all of it).  4099 rows of 50 000 float32: 195 to 213 us, 4 TB/s, bound by
// memory and the vector units (busy for 80 %) in about equal parts.
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
    copy_flat<kThreads>(tile, src, n, threadIdx.x);
    __syncthreads();
    if (q.log_probs) {
        for (int k = threadIdx.x; k < q.top; k += kThreads) {
            const int i = entry(q, row, k).index - j0;
            if (i >= 0 && i < n) tile[i] = E::down(-INFINITY);
        }
        __syncthreads();
    }
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
        s += v == -INFINITY ? 0.f : expo_of<E>(q, v, m);
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
// wave for a row (4099 rows of 7 segments and 32 entries: 8.5 us).
template <class E>
__global__ __launch_bounds__(64) void k_seg_join(const Distil q) {
    using T = typename E::T;
    extern __shared__ u32x4 smem[];
    int* ei = (int*)smem;
    const int64_t row = blockIdx.x;
    const int lane = threadIdx.x;
    const T* src = (const T*)q.logits + row * q.stride;
    constexpr int KPL = GSX_DISTIL_MAX_TOP / 64;
    Entries<KPL> e;
    read_entries<64, KPL>(q, row, lane, e);
#pragma unroll
    for (int i = 0; i < KPL; ++i) {
        if (lane + i * 64 < q.top) ei[lane + i * 64] = e.index[i];
        e.s[i] = e.index[i] >= 0 ? E::up(src[e.index[i]]) : 0.f;
    }
    __syncthreads();
    bool shared = false;
#pragma unroll
    for (int i = 0; i < KPL; ++i) {
        e.again[i] = false;
        if (e.index[i] >= 0)
            for (int k = 0; k < lane + i * 64; ++k) e.again[i] |= ei[k] == e.index[i];
        shared |= e.again[i];
    }
    shared = __any(shared);
    const float* parts = q.seg_parts + row * q.segs * 2;
    float m = -INFINITY, s = 0.f;
    for (int i = lane; i < q.segs; i += 64) m = fmaxf(m, parts[2 * i]);
    m = group_max<64>(m);
    for (int i = lane; i < q.segs; i += 64) {
        const float pm = parts[2 * i], ps = parts[2 * i + 1];
        s += pm == -INFINITY ? ps : ps * expo(q, pm, m);  // 0, or NaN
    }
    s = group_sum<64>(s);
    const RowStats r = q.log_probs ? row_stats<64, KPL, true>(q, e, m, s)
                                   : row_stats<64, KPL, false>(q, e, m, s);
    if (lane == 0) {
        const float loss = r.active ? r.loss : 0.f;
        if (q.loss_rows) q.loss_rows[row] = loss;
        if (q.loss_parts) q.loss_parts[row] = loss;
        float* st = q.stats + row * 8;
        st[0] = m;
        st[1] = r.rest;
        st[2] = r.m;
        st[3] = r.inv;
        st[4] = r.active ? 1.f : 0.f;
        st[5] = shared ? 1.f : 0.f;
    }
    // the entries' probabilities, for the gradient
    float* probs = q.stats + q.rows * 8 + row * q.top;
#pragma unroll
    for (int i = 0; i < KPL; ++i)
        if (lane + i * 64 < q.top) probs[lane + i * 64] = e.value[i];
}

// A segment's gradient.  4099 rows of 50 000 float32: 300 to 329 us, 5 TB/s read and
// written (a large copy: 4.8); taking the rows in reverse, so that it began with those
// that the first pass read last, changed nothing.
template <class E>
__global__ __launch_bounds__(kThreads) void k_seg_grad(const Distil q) {
    using T = typename E::T;
    __shared__ u32x4 smem[kSegBytes / 16 + 1];
    __shared__ int scratch[kThreads / 64];
    __shared__ int ei[GSX_DISTIL_MAX_TOP];
    __shared__ float ep[GSX_DISTIL_MAX_TOP];
    const int64_t row = blockIdx.x / q.segs;
    const int seg = (int)(blockIdx.x % q.segs);
    const int j0 = seg * q.seg, n = q.vocab - j0 < q.seg ? q.vocab - j0 : q.seg;
    const T* src = (const T*)q.logits + row * q.stride + j0;
    T* dst = (T*)q.grad + row * q.vocab + j0;
    T* tile = (T*)smem + ((uintptr_t)src % 16) / sizeof(T);
    const float* st = q.stats + row * 8;
    const bool active = st[4] != 0.f, shared = st[5] != 0.f;
    if (active) {
        copy_flat<kThreads>(tile, src, n, threadIdx.x);
        const float* probs = q.stats + q.rows * 8 + row * q.top;
        for (int k = threadIdx.x; k < q.top; k += kThreads) {
            ei[k] = entry(q, row, k).index;
            ep[k] = probs[k];
        }
    }
    const float inv_count = inverse_count(q, scratch);
    const float f = row_scale(q, row, inv_count);
    const float rest_m = st[0], rest = st[1] * f;
    __syncthreads();
    // this thread's entry of this segment (there are no more entries than threads)
    float own = 0.f;
    int at = -1;
    if (active && threadIdx.x < q.top) {
        const int i = ei[threadIdx.x] - j0;
        if (ei[threadIdx.x] >= 0 && i >= 0 && i < n) {
            at = i;
            float p = ep[threadIdx.x];
            if (shared) {
                p = 0.f;
                for (int j = 0; j < q.top; ++j)
                    if (ei[j] == i + j0) p += ep[j];
            }
            const float s = E::up(tile[i]);
            own = f * ((s == -INFINITY ? 0.f : expo(q, s, st[2])) * st[3] - p);
        }
    }
    __syncthreads();
    for (int j = threadIdx.x; j < n; j += kThreads) {
        float g = 0.f;
        if (active) {
            const float s = E::up(tile[j]);
            g = s == -INFINITY ? 0.f * rest : expo_of<E>(q, s, rest_m) * rest;
        }
        tile[j] = E::down(g);
    }
    __syncthreads();
    if (at >= 0) tile[at] = E::down(own);
    __syncthreads();
    if (((uintptr_t)dst - (uintptr_t)src) % 16 == 0)
        copy_flat<kThreads>(dst, (const T*)tile, n, threadIdx.x);
    else
        for (int i = threadIdx.x; i < n; i += kThreads) dst[i] = tile[i];
}
static_assert(GSX_DISTIL_MAX_TOP <= kThreads, "an entry for each thread");

// Rows that have an entry, a count for each of kCountParts workgroups; four rows
// of a thread are in flight at a time.  A launch of its own because the mean's
// gradient needs it first; it reads an entry of most rows and all of the others'
// (921 600 rows of 8 entries: 16 us).
__global__ __launch_bounds__(1024) void k_count(const Distil q, int* counts) {
    __shared__ int red[1024 / 64];
    constexpr int64_t step = (int64_t)kCountParts * 1024;
    int n = 0;
    for (int64_t row = (int64_t)blockIdx.x * 1024 + threadIdx.x; row < q.rows; row += 4 * step) {
        int found[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            found[i] = row + i * step < q.rows && entry(q, row + i * step, 0).index >= 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            n += found[i] || (row + i * step < q.rows && supervised(q, row + i * step));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, kWave);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        n = 0;
#pragma unroll
        for (int w = 0; w < 1024 / 64; ++w) n += red[w];
        counts[blockIdx.x] = n;
    }
}

// The sum (or mean) of the rows' losses, in a fixed order: 2048 parts, 5 us.
__global__ __launch_bounds__(kThreads) void k_total(const double* parts, int64_t n,
                                                    const int* counts, float scale, float* out) {
    __shared__ double red[kThreads];
    __shared__ int cnt[kThreads];
    double s = 0.0;
    int64_t i = threadIdx.x;
    for (; i + 7 * kThreads < n; i += 8 * kThreads) {  // eight loads in flight
        double v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = parts[i + j * kThreads];
#pragma unroll
        for (int j = 0; j < 8; ++j) s += v[j];
    }
    for (; i < n; i += kThreads) s += parts[i];
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

int elem(int dtype) { return dtype == GSX_F32 ? 4 : 2; }
bool short_rows(int dtype, int64_t vocab) { return vocab * elem(dtype) <= kRowBytes; }
int segments(int dtype, int64_t vocab) {
    const int64_t seg = kSegBytes / elem(dtype);
    return (int)((vocab + seg - 1) / seg);
}

int check_shape(int dtype, int64_t rows, int64_t vocab, int64_t top) {
    if (dtype != GSX_F32 && dtype != GSX_BF16 && dtype != GSX_F16) return GSX_ERR_INVALID;
    if (rows < 0 || vocab <= 0 || top <= 0) return GSX_ERR_INVALID;
    if (top > vocab) return GSX_ERR_INVALID;
    if (rows >= (1LL << 30) || vocab >= (1LL << 30) || top > GSX_DISTIL_MAX_TOP)
        return GSX_ERR_TOO_LARGE;
    // a launch holds fewer than 2^32 threads in all, a workgroup for each segment
    if (!short_rows(dtype, vocab) &&
        rows * segments(dtype, vocab) >= (1LL << 32) / kThreads)
        return GSX_ERR_TOO_LARGE;
    return GSX_OK;
}

// 32-bit words that a row may touch (a 16-bit row may begin inside one), and
// the lanes that hold them: up to kHeld words each (more leave a SIMD two waves
// instead of four, and are for rows that fill 64 lanes), 4 to 64 lanes.  Four
// entries at most on a lane.
int words_of(int dtype, int64_t vocab) {
    return (int)(dtype == GSX_F32 ? vocab : (vocab + 1) / 2 + 1);
}
constexpr int kHeld = 14;
int lanes_for(int dtype, int64_t vocab, int64_t top) {
    int g = 4;
    while (g < 64 && (g * kHeld < words_of(dtype, vocab) || g * 4 < top)) g *= 2;
    return g;
}
// Workgroups' worth of tiles that one walks alone, with the count and the sum in
// its one launch: a patch of 64 rows took 18 us a call instead of 23, whose three
// launches take longer than their work.
constexpr int64_t kAlone = 4;
constexpr int64_t kRowGroups = 2048;  // workgroups that walk the tiles: eight for a unit

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
        const int r = kThreads / lanes_for(dtype, vocab, top);
        l.n_parts = (rows + r - 1) / r;
        if (l.n_parts > kRowGroups) l.n_parts = kRowGroups;
        l.segs = l.stats = l.total = up_to(l.parts + l.n_parts * 8, 256);
        return l;
    }
    l.seg = kSegBytes / elem(dtype);
    l.n_segs = segments(dtype, vocab);
    l.n_parts = rows;
    l.segs = up_to(l.parts + l.n_parts * 8, 256);
    l.stats = up_to(l.segs + rows * l.n_segs * 8, 256);
    l.total = up_to(l.stats + rows * (8 + top) * 4, 256);
    return l;
}

// (42 KB of shared memory at most: 4096 columns of 16 bits and 256 entries.)
template <class E, int G, int N, int KPL, bool LOG_PROBS, int FULL>
int launch_rows(const Distil& q, hipStream_t st) {
    constexpr int R = 64 / G, kWaves = kThreads / 64;
    const int64_t tiles = (q.rows + R - 1) / R, groups = (tiles + kWaves - 1) / kWaves;
    const int64_t lds = kWaves * (tile_room(R, G * N, q.vocab, sizeof(typename E::T)) +
                                  (int64_t)R * q.top * 8);
    hipLaunchKernelGGL((k_rows<E, G, N, KPL, LOG_PROBS, FULL>),
                       dim3(q.alone                ? 1u
                            : groups < kRowGroups ? (unsigned)groups
                                                  : (unsigned)kRowGroups),
                       dim3(kThreads),
                       (unsigned)lds, st, q, tiles);
    GSX_LAUNCH_CHECK();
    return GSX_OK;
}

// For rows of MORE to N words a lane: of 16-bit rows, which may begin inside a
// word, all but the first and the last MORE - 2 are whole words of the row.
template <class E, int G, int N, int KPL, int MORE>
int launch_rows(const Distil& q, hipStream_t st) {
    constexpr int FULL = MORE > 2 ? MORE - 2 : 0;
    return q.log_probs ? launch_rows<E, G, N, KPL, true, FULL>(q, st)
                       : launch_rows<E, G, N, KPL, false, FULL>(q, st);
}

// The kernel whose lanes hold the row's words and entries with the least room to
// spare: a wave works on all the room there is.  Loss and gradient of 300 MB of
// logits, us with the least room / with the next that would hold them:
//   words     3 / 6    12 float32 columns 33.4 / 36.6, 21 bf16 35.3 / 40.0
//             8 / 10   64 float32 93.7 / 95.9, 126 bf16 102 / 104
//             8 / 14   64 float32 93.7 / 101, 126 bf16 102 / 117
//            10 / 14   80 float32 108 / 113, 150 bf16 112 / 125
//            20 / 33   1280 float32 141 / 152, 2558 bf16 154 / 219
//   entries   1 / 4    128 float32 165 / 224, 150 bf16 112 / 184
//             2 / 4    80 float32, 15 entries 131 / 147, 150 bf16 143 / 202
//   four entries with 6 / 14 words  24 float32, 20 entries 90 / 111, 90 bf16, 30
//                      143 / 208
//   two entries with 3 / 6 words    21 bf16, 7 entries 40.4 / 44.8
// Eight lanes and more hold more than seven words each (half of them would do
// otherwise), or over eight entries for every four lanes.
template <class E, int G>
int launch_rows(const Distil& q, int words, hipStream_t st) {
    const int n = (words + G - 1) / G;
    if (q.top > 2 * G) {
        if (n <= 6) return launch_rows<E, G, 6, 4, 0>(q, st);
        if constexpr (G == 64) {
            if (n > 14) return launch_rows<E, G, 33, 4, 15>(q, st);
        }
        return launch_rows<E, G, 14, 4, 7>(q, st);
    }
    if (q.top > G) {
        if constexpr (G == 4) {
            if (n <= 3) return launch_rows<E, G, 3, 2, 0>(q, st);
            if (n <= 6) return launch_rows<E, G, 6, 2, 0>(q, st);
        }
        if constexpr (G == 64) {
            if (n > 14) return launch_rows<E, G, 33, 2, 15>(q, st);
        }
        return launch_rows<E, G, 14, 2, 7>(q, st);
    }
    if constexpr (G == 4) {
        if (n <= 3) return launch_rows<E, G, 3, 1, 0>(q, st);
        if (n <= 6) return launch_rows<E, G, 6, 1, 0>(q, st);
    }
    if (n <= 8) return launch_rows<E, G, 8, 1, 7>(q, st);
    if (n <= 10) return launch_rows<E, G, 10, 1, 9>(q, st);
    if constexpr (G == 64) {
        if (n > 20) return launch_rows<E, G, 33, 1, 21>(q, st);
        if (n > 14) return launch_rows<E, G, 20, 1, 15>(q, st);
    }
    return launch_rows<E, G, 14, 1, 11>(q, st);
}

template <class E>
int run_rows(const Distil& q, hipStream_t st) {
    constexpr int dtype = sizeof(typename E::T) == 4 ? GSX_F32 : GSX_BF16;
    const int words = words_of(dtype, q.vocab);
    switch (lanes_for(dtype, q.vocab, q.top)) {
        case 4: return launch_rows<E, 4>(q, words, st);
        case 8: return launch_rows<E, 8>(q, words, st);
        case 16: return launch_rows<E, 16>(q, words, st);
        case 32: return launch_rows<E, 32>(q, words, st);
        default: return launch_rows<E, 64>(q, words, st);
    }
}

// Loss (stats) and, where asked for, gradient.  `sums`: form the statistics;
// false: they are in the workspace (the gradient of an earlier forward).
template <class E>
int run(const Distil& q, bool sums, hipStream_t st) {
    if (q.segs == 0) return run_rows<E>(q, st);
    const int64_t blocks = q.rows * q.segs;
    if (sums) {
        hipLaunchKernelGGL((k_seg_sum<E>), dim3((unsigned)blocks), dim3(kThreads), 0, st, q);
        GSX_LAUNCH_CHECK();
        hipLaunchKernelGGL((k_seg_join<E>), dim3((unsigned)q.rows), dim3(64),
                           (unsigned)(q.top * 4), st, q);
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
    // 1 / T is a float32, too
    if (!(a.temperature >= 1e-38f) || a.temperature > 3.0e38f) return GSX_ERR_INVALID;
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
    const double c = 1.4426950408889634 / (double)a.temperature;
    q.c = (float)c;
    q.c_lo = (float)(c - (double)q.c);
    q.log_probs = a.teacher == GSX_TEACHER_LOG_PROBS;
    q.scale = 1.0f;
    char* ws = (char*)a.workspace;
    q.counts = (const int*)ws;
    q.mean = a.reduction == GSX_REDUCE_MEAN;
    q.alone = a.rows > 0 && l.n_segs == 0 && l.n_parts <= kAlone;
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
    if (q.alone && a.reduction != GSX_REDUCE_NONE) {
        q.total = loss;
        return run_any(a.dtype, q, true, st);
    }
    if (a.reduction == GSX_REDUCE_NONE)
        q.loss_rows = loss;
    else
        q.loss_parts = parts;
    if (a.reduction == GSX_REDUCE_MEAN) {
        hipLaunchKernelGGL(k_count, dim3(kCountParts), dim3(1024), 0, st, q,
                           (int*)a.workspace);
        GSX_LAUNCH_CHECK();
    }
    if (a.rows > 0)
        if (int e = run_any(a.dtype, q, true, st)) return e;
    if (a.reduction != GSX_REDUCE_NONE) {
        hipLaunchKernelGGL(k_total, dim3(1), dim3(kThreads), 0, st, parts,
                           a.rows > 0 ? l.n_parts : 0, q.mean ? q.counts : nullptr, scale, loss);
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
