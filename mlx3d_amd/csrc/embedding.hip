// embedding.hip -- rows of a table by their indices, and the table's gradient.
//
//   y_i = s T[k_i], zero where k_i lies outside the table
//   dT[v] = s sum over i with k_i = v of dy_i
//
// The gradient sorts the tokens (stably, so that a row's sum has one order) and
// walks them in tiles: a group of lanes adds up a tile's rows of dy as long as the
// key stays the same.  What begins and ends inside a tile is written at once; what a
// tile shares with its neighbours goes into two partial rows, which a last launch
// joins.  So a row that every token names is spread over as many lanes as rows that
// one token names, no sum depends on the order of arrival, and sums stay short: a
// tile's, then the tiles'.
//
// The sort is a stable radix sort by digits of 8 bits, three launches a pass: a
// chunk's counts of each digit, their prefix over the chunks, and the placement.  No
// workgroup waits for another one.  Tokens outside the table are left out of the
// first pass.
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
constexpr int kBits = 8, kRadix = 1 << kBits;
constexpr int kSortThreads = 512, kItems = 8, kChunk = kSortThreads * kItems;
constexpr int kScanGroups = 16;  // of chunks, in the prefix
constexpr int kMostTile = 64;    // sorted tokens that a team of lanes adds up, at most
constexpr int kBatch = 8;        // rows that a team asks for at a time
constexpr int kSpan = 32;        // tiles of a row that a single team joins, at most
constexpr int kJoinThreads = 1024;

struct Embed {
    const void *table, *g_y, *indices;
    void *y, *g_table;
    int64_t count, rows, stride;  // stride of the table's or of g_y's rows
    int width, index64;
    float scale;
};

// Token i's row, or -1.
__device__ __forceinline__ int64_t row_of(const Embed& q, int64_t i) {
    const int64_t k = q.index64 ? ((const int64_t*)q.indices)[i] : ((const int32_t*)q.indices)[i];
    return k >= 0 && k < q.rows ? k : -1;
}

// G lanes a token, a piece of V elements each; blockIdx.y: pieces from 64 on.
template <class E, int V, int G>
__global__ __launch_bounds__(kThreads) void k_lookup(const Embed q) {
    using P = Piece<E, V>;
    using T = typename E::T;
    const int at = (blockIdx.y * G + threadIdx.x % G) * V;
    if (at >= q.width) return;
    const int c = min(at, q.width - V);
    const int64_t step = (int64_t)gridDim.x * (kThreads / G);
    for (int64_t i = (int64_t)blockIdx.x * (kThreads / G) + threadIdx.x / G; i < q.count;
         i += step) {
        const int64_t k = row_of(q, i);
        float v[V] = {};
        if (k >= 0) {
            P::up(P::load((const T*)q.table + k * q.stride + c), v);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] *= q.scale;
        }
        P::store((T*)q.y + i * q.width + c, P::down(v));
    }
}

// ----------------------------------------------------------------- sort --

struct Sort {
    Embed q;
    const uint2* from;  // (key, token), or NULL: the indices
    uint2* to;
    uint32_t* counts;   // (chunks, kRadix)
    uint32_t* totals;   // kRadix
    uint32_t* live;     // how many tokens name a row
    int chunks, shift, bits;
};

__device__ __forceinline__ int64_t live_tokens(const Sort& s) {
    return s.from ? (int64_t)*s.live : s.q.count;
}
// The pair at place i of the pass, if there is one.
__device__ __forceinline__ bool pair_at(const Sort& s, int64_t i, int64_t n, uint2* p) {
    if (i >= n) return false;
    if (s.from) {
        *p = s.from[i];
        return true;
    }
    const int64_t k = row_of(s.q, i);
    *p = make_uint2((uint32_t)k, (uint32_t)i);
    return k >= 0;
}

__global__ __launch_bounds__(kSortThreads) void k_count(const Sort s) {
    __shared__ uint32_t hist[kRadix];
    for (int d = threadIdx.x; d < kRadix; d += kSortThreads) hist[d] = 0;
    __syncthreads();
    const int64_t n = live_tokens(s), first = (int64_t)blockIdx.x * kChunk;
    for (int r = 0; r < kItems; ++r) {
        uint2 p;
        if (pair_at(s, first + r * kSortThreads + threadIdx.x, n, &p))
            atomicAdd(&hist[(p.x >> s.shift) & (kRadix - 1)], 1u);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < kRadix; d += kSortThreads)
        s.counts[(int64_t)blockIdx.x * kRadix + d] = hist[d];
}

// Each digit's prefix over the chunks, in place, and its total: 64 digits a
// workgroup, the chunks in kScanGroups stretches.
__global__ __launch_bounds__(64 * kScanGroups) void k_prefix(const Sort s) {
    __shared__ uint32_t sums[kScanGroups][64];
    const int lane = threadIdx.x & 63, g = threadIdx.x >> 6;
    const int d = blockIdx.x * 64 + lane;
    const int per = (s.chunks + kScanGroups - 1) / kScanGroups;
    const int first = min(g * per, s.chunks), end = min(first + per, s.chunks);
    uint32_t sum = 0;
    for (int c = first; c < end; ++c) sum += s.counts[(int64_t)c * kRadix + d];
    sums[g][lane] = sum;
    __syncthreads();
    uint32_t run = 0, total = 0;
#pragma unroll
    for (int k = 0; k < kScanGroups; ++k) {
        if (k < g) run += sums[k][lane];
        total += sums[k][lane];
    }
    for (int c = first; c < end; ++c) {
        uint32_t* at = s.counts + (int64_t)c * kRadix + d;
        const uint32_t v = *at;
        *at = run;
        run += v;
    }
    if (g == 0) s.totals[d] = total;
}

// Lanes of the wave, among the valid ones, with the same digit.
__device__ __forceinline__ uint64_t same_digit(uint32_t d, bool valid, int bits) {
    uint64_t differ = 0;
    for (int b = 0; b < bits; ++b) {
        const uint64_t set = __ballot(d >> b & 1);
        differ |= set ^ (d >> b & 1 ? ~0ull : 0ull);
    }
    return ~differ & __ballot(valid);
}

__global__ __launch_bounds__(kSortThreads) void k_place(const Sort s) {
    constexpr int kWaves = kSortThreads / 64;
    __shared__ uint32_t cnt[kWaves][kRadix];
    __shared__ uint32_t in_chunk[kRadix], base[kRadix];
    __shared__ uint32_t sums[2][kRadix / 64];
    __shared__ uint2 pairs[kChunk];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int k = tid; k < kWaves * kRadix; k += kSortThreads) (&cnt[0][0])[k] = 0;
    const int64_t n = live_tokens(s);
    const int64_t first = (int64_t)blockIdx.x * kChunk + wave * (64 * kItems);
    uint2 p[kItems];
    bool valid[kItems];
    uint32_t rank[kItems];
#pragma unroll
    for (int r = 0; r < kItems; ++r) {
        p[r] = make_uint2(0, 0);
        valid[r] = pair_at(s, first + r * 64 + lane, n, &p[r]);
    }
    __syncthreads();
    // a wave's tokens in their order: each digit's count so far, and the lanes before
#pragma unroll
    for (int r = 0; r < kItems; ++r) {
        const uint32_t d = (p[r].x >> s.shift) & (kRadix - 1);
        const uint64_t same = same_digit(d, valid[r], s.bits);
        const uint64_t before = same & ((1ull << lane) - 1);
        const uint32_t c = cnt[wave][d];
        rank[r] = c + (uint32_t)__popcll(before);
        wave_fence();
        if (valid[r] && before == 0) cnt[wave][d] = c + (uint32_t)__popcll(same);
        wave_fence();
    }
    __syncthreads();
    // digits' places: in the chunk by the chunk's counts, in the whole by the totals
    uint32_t mine = 0, total = 0, mine_incl = 0, total_incl = 0;
    if (tid < kRadix) {
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const uint32_t c = cnt[w][tid];
            cnt[w][tid] = mine;
            mine += c;
        }
        total = s.totals[tid];
        mine_incl = wave_incl_scan(mine);
        total_incl = wave_incl_scan(total);
        if (lane == 63) {
            sums[0][wave] = mine_incl;
            sums[1][wave] = total_incl;
        }
    }
    __syncthreads();
    if (tid < kRadix) {
        for (int w = 0; w < wave; ++w) {
            mine_incl += sums[0][w];
            total_incl += sums[1][w];
        }
        in_chunk[tid] = mine_incl - mine;
        base[tid] = total_incl - total + s.counts[(int64_t)blockIdx.x * kRadix + tid];
        // the first pass counts the tokens that name a row
        if (!s.from && blockIdx.x == 0 && tid == kRadix - 1) *s.live = total_incl;
    }
    __syncthreads();
    // regrouped by digit, so that stores are runs
#pragma unroll
    for (int r = 0; r < kItems; ++r)
        if (valid[r]) {
            const uint32_t d = (p[r].x >> s.shift) & (kRadix - 1);
            pairs[in_chunk[d] + cnt[wave][d] + rank[r]] = p[r];
        }
    __syncthreads();
    const int held = (int)(sums[0][0] + sums[0][1] + sums[0][2] + sums[0][3]);
    for (int j = tid; j < held; j += kSortThreads) {
        const uint2 e = pairs[j];
        const uint32_t d = (e.x >> s.shift) & (kRadix - 1);
        s.to[base[d] + (uint32_t)j - in_chunk[d]] = e;
    }
}

// ------------------------------------------------------------------ sum --

struct Sum {
    Embed q;
    const uint2* pairs;
    const uint32_t* live;
    int tile;      // sorted tokens of a tile
    float* parts;  // (tiles, 2, width): what a tile shares with the one before, and behind
};

template <class T>
__global__ __launch_bounds__(kThreads) void k_zero(T* p, int64_t n) {
    const int64_t step = (int64_t)gridDim.x * kThreads;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += step) p[i] = 0;
}

// One tile, V columns of it.  A batch of rows is asked for before the first is added.
template <class E, int V>
__device__ __forceinline__ void tile_sum(const Sum& s, int64_t tile, int64_t live, int c) {
    using P = Piece<E, V>;
    using T = typename E::T;
    const Embed& q = s.q;
    const int64_t first = tile * s.tile;
    const int n = (int)min<int64_t>(s.tile, live - first);
    const uint2* pairs = s.pairs + first;
    uint32_t key = pairs[0].x;
    bool open = first > 0 && pairs[-1].x == key;  // the tile before has some of this row
    const bool more = first + n < live && pairs[n].x == pairs[n - 1].x;
    float acc[V] = {};
    float* part = s.parts + tile * 2 * q.width + c;
    auto write = [&]() {
        if (open) {
            store_floats<V>(part, acc);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] *= q.scale;
            P::store((T*)q.g_table + (int64_t)key * q.width + c, P::down(acc));
        }
    };
    for (int j = 0; j < n; j += kBatch) {
        uint2 p[kBatch];
        typename P::Raw raw[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) p[u] = pairs[min(j + u, n - 1)];
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            raw[u] = P::load((const T*)q.g_y + (int64_t)p[u].y * q.stride + c);
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            if (j + u >= n) break;
            if (p[u].x != key) {
                write();
                key = p[u].x;
                open = false;
#pragma unroll
                for (int e = 0; e < V; ++e) acc[e] = 0.f;
            }
            float v[V];
            P::up(raw[u], v);
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] += v[e];
        }
    }
    if (!more) write();
    else store_floats<V>(open ? part : part + q.width, acc);
}

// G lanes a tile, a piece of V columns each.
template <class E, int V, int G>
__global__ __launch_bounds__(kThreads) void k_tile_sums(const Sum s) {
    const int at = (blockIdx.y * G + threadIdx.x % G) * V;
    if (at >= s.q.width) return;
    const int64_t live = *s.live, step = (int64_t)gridDim.x * (kThreads / G);
    for (int64_t tile = (int64_t)blockIdx.x * (kThreads / G) + threadIdx.x / G;
         tile * s.tile < live; tile += step)
        tile_sum<E, V>(s, tile, live, min(at, s.q.width - V));
}

// How many tiles after `tile` share the row that it leaves open and that begins in
// it; 0 if there is none.
__device__ __forceinline__ int64_t span_of(const Sum& s, int64_t tile, int64_t live) {
    const int64_t first = tile * s.tile, next = first + s.tile;
    if (next >= live) return 0;
    const uint32_t key = s.pairs[next - 1].x;
    if (s.pairs[next].x != key) return 0;
    if (first > 0 && s.pairs[first].x == key && s.pairs[first - 1].x == key) return 0;
    // tiles' first keys do not fall: double the reach, then halve it
    const int64_t tiles = (live + s.tile - 1) / s.tile;
    int64_t in = tile + 1, reach = 1;
    while (in + reach < tiles && s.pairs[(in + reach) * s.tile].x == key) {
        in += reach;
        reach *= 2;
    }
    for (; reach > 0; reach /= 2)
        if (in + reach < tiles && s.pairs[(in + reach) * s.tile].x == key) in += reach;
    return in - tile;
}

// Adds up a row's parts in tiles first, first + step, ... below end.
template <int V>
__device__ __forceinline__ void add_parts(const Sum& s, int64_t first, int64_t end, int64_t step,
                                          int c, float* acc) {
    for (int64_t t = first; t < end; t += kBatch * step) {
        float v[kBatch][V];
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            load_floats<V>(s.parts + min(t + u * step, end - 1) * 2 * s.q.width + c, v[u]);
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            if (t + u * step < end) {
#pragma unroll
                for (int e = 0; e < V; ++e) acc[e] += v[u][e];
            }
    }
}

// Rows over several tiles, each by the team of lanes of the tile in which it begins;
// over more than kSpan, by all teams of the workgroup together.
template <class E, int V, int G>
__global__ __launch_bounds__(kJoinThreads) void k_join(const Sum s) {
    using P = Piece<E, V>;
    using T = typename E::T;
    constexpr int kTeams = kJoinThreads / G;
    __shared__ float room[kJoinThreads][V + 1];
    __shared__ int64_t spans[kTeams];
    const Embed& q = s.q;
    const int team = threadIdx.x / G, at = (blockIdx.y * G + threadIdx.x % G) * V;
    const int c = min(at, q.width - V);
    const int64_t live = *s.live, step = (int64_t)gridDim.x * kTeams;
    auto write = [&](int64_t tile, float* acc) {
        const uint32_t key = s.pairs[tile * s.tile + s.tile - 1].x;
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] *= q.scale;
        if (at < q.width) P::store((T*)q.g_table + (int64_t)key * q.width + c, P::down(acc));
    };
    for (int64_t base = (int64_t)blockIdx.x * kTeams; base * s.tile < live; base += step) {
        const int64_t tile = base + team, span = span_of(s, tile, live);
        if (span > 0 && span <= kSpan) {
            float acc[V];
            load_floats<V>(s.parts + (tile * 2 + 1) * q.width + c, acc);
            add_parts<V>(s, tile + 1, tile + 1 + span, 1, c, acc);
            write(tile, acc);
        }
        if (threadIdx.x % G == 0) spans[team] = span;
        if (!__syncthreads_or(span > kSpan)) continue;
        for (int t = 0; t < kTeams; ++t) {
            const int64_t far = spans[t], own = base + t;
            if (far <= kSpan) continue;
            float acc[V] = {};
            if (team == 0) load_floats<V>(s.parts + (own * 2 + 1) * q.width + c, acc);
            add_parts<V>(s, own + 1 + team, own + 1 + far, kTeams, c, acc);
#pragma unroll
            for (int e = 0; e < V; ++e) room[threadIdx.x][e] = acc[e];
            for (int n = kTeams / 2; n > 0; n /= 2) {
                __syncthreads();
                if (team < n) {
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        acc[e] += room[threadIdx.x + n * G][e];
                        room[threadIdx.x][e] = acc[e];
                    }
                }
            }
            if (team == 0) write(own, acc);
            __syncthreads();
        }
    }
}

// ----------------------------------------------------------------- host --

// A launch holds fewer than 2^32 threads: at most 2^21 workgroups of 1024 and
// fewer here, whose threads walk on.
dim3 grid_for(int64_t n, int per_group, int times) {
    const int64_t groups = (n + per_group - 1) / per_group, most = ((int64_t)1 << 21) / times;
    return dim3((unsigned)(groups < most ? groups : most), (unsigned)times);
}

int64_t up_to(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

int check_shape(int dtype, int64_t count, int64_t rows, int32_t width) {
    if (dtype != GSX_F32 && dtype != GSX_BF16 && dtype != GSX_F16) return GSX_ERR_INVALID;
    if (count < 0 || rows <= 0 || width <= 0) return GSX_ERR_INVALID;
    if (count > 1 << 30 || rows > 1 << 30 || width > 1 << 20) return GSX_ERR_TOO_LARGE;
    return GSX_OK;
}

int check_args(int dtype, int64_t count, int64_t rows, int32_t width, const void* indices,
               int32_t index64, const void* data, int64_t stride, float scale) {
    if (int e = check_shape(dtype, count, rows, width)) return e;
    if (index64 != 0 && index64 != 1) return GSX_ERR_INVALID;
    if (count > 0 && (!indices || !data)) return GSX_ERR_INVALID;
    if (stride < width || !(scale >= -3.4e38f && scale <= 3.4e38f)) return GSX_ERR_INVALID;
    if ((uintptr_t)indices % (index64 ? 8 : 4) || (uintptr_t)data % (dtype == GSX_F32 ? 4 : 2))
        return GSX_ERR_INVALID;
    return GSX_OK;
}

struct Layout {
    int chunks, passes, bits, tile;
    int64_t tiles, counts, totals, live, pairs[2], parts, total;
};

Layout layout(int64_t count, int64_t rows, int32_t width) {
    Layout l{};
    l.chunks = (int)((count + kChunk - 1) / kChunk);
    l.bits = 1;
    while (((int64_t)1 << l.bits) < rows) ++l.bits;
    l.passes = (l.bits + kBits - 1) / kBits;
    l.tile = kMostTile;
    l.tiles = (count + l.tile - 1) / l.tile;
    l.counts = 0;
    l.totals = up_to((int64_t)l.chunks * kRadix * 4, 256);
    l.live = l.totals + kRadix * 4;
    l.pairs[0] = l.live + 256;
    l.pairs[1] = up_to(l.pairs[0] + count * 8, 256);
    l.parts = up_to(l.pairs[1] + (l.passes > 1 ? count * 8 : 0), 256);
    l.total = up_to(l.parts + l.tiles * 2 * width * 4, 256);
    return l;
}

// Calls f with the element count of a piece and the lanes of a row, and gives it how
// many times that many lanes a row takes.
template <class E, class F>
int for_width(int width, F f) {
    auto lanes = [&](auto v) -> int {
        constexpr int V = decltype(v)::value;
        const int n = (width + V - 1) / V;
        using I = std::integral_constant<int, V>;
        if (n <= 1) return f(I{}, std::integral_constant<int, 1>{}, 1);
        if (n <= 2) return f(I{}, std::integral_constant<int, 2>{}, 1);
        if (n <= 4) return f(I{}, std::integral_constant<int, 4>{}, 1);
        if (n <= 8) return f(I{}, std::integral_constant<int, 8>{}, 1);
        if constexpr (V > 1) {
            if (n <= 16) return f(I{}, std::integral_constant<int, 16>{}, 1);
            if (n <= 32) return f(I{}, std::integral_constant<int, 32>{}, 1);
            return f(I{}, std::integral_constant<int, 64>{}, (n + 63) / 64);
        }
        return GSX_ERR_INVALID;  // a row of fewer than VEC elements has eight at most
    };
    if (width < E::VEC) return lanes(std::integral_constant<int, 1>{});
    return lanes(std::integral_constant<int, E::VEC>{});
}

template <class E>
int lookup(const Embed& q, hipStream_t st) {
    return for_width<E>(q.width, [&](auto v, auto g, int times) -> int {
        constexpr int V = decltype(v)::value, G = decltype(g)::value;
        hipLaunchKernelGGL((k_lookup<E, V, G>), grid_for(q.count, kThreads / G, times),
                           dim3(kThreads), 0, st, q);
        GSX_LAUNCH_CHECK();
        return GSX_OK;
    });
}

template <class E>
int gradient(const Embed& q, char* ws, hipStream_t st) {
    const Layout l = layout(q.count, q.rows, q.width);
    const int64_t table = q.rows * q.width;
    const int64_t fill = (table + kThreads - 1) / kThreads;
    hipLaunchKernelGGL((k_zero<typename E::T>), dim3((unsigned)(fill < 8192 ? fill : 8192)),
                       dim3(kThreads), 0, st, (typename E::T*)q.g_table, table);
    GSX_LAUNCH_CHECK();
    if (q.count == 0) return GSX_OK;
    Sort s{};
    s.q = q;
    s.counts = (uint32_t*)(ws + l.counts);
    s.totals = (uint32_t*)(ws + l.totals);
    s.live = (uint32_t*)(ws + l.live);
    s.chunks = l.chunks;
    for (int p = 0; p < l.passes; ++p) {
        s.from = p ? (const uint2*)(ws + l.pairs[(p - 1) % 2]) : nullptr;
        s.to = (uint2*)(ws + l.pairs[p % 2]);
        s.shift = p * kBits;
        s.bits = l.bits - s.shift < kBits ? l.bits - s.shift : kBits;
        hipLaunchKernelGGL(k_count, dim3((unsigned)l.chunks), dim3(kSortThreads), 0, st, s);
        GSX_LAUNCH_CHECK();
        hipLaunchKernelGGL(k_prefix, dim3(kRadix / 64), dim3(64 * kScanGroups), 0, st, s);
        GSX_LAUNCH_CHECK();
        hipLaunchKernelGGL(k_place, dim3((unsigned)l.chunks), dim3(kSortThreads), 0, st, s);
        GSX_LAUNCH_CHECK();
    }
    Sum u{};
    u.q = q;
    u.pairs = s.to;
    u.live = s.live;
    u.tile = l.tile;
    u.parts = (float*)(ws + l.parts);
    return for_width<E>(q.width, [&](auto v, auto g, int times) -> int {
        constexpr int V = decltype(v)::value, G = decltype(g)::value;
        const dim3 grid = grid_for(l.tiles, kThreads / G, times);
        hipLaunchKernelGGL((k_tile_sums<E, V, G>), grid, dim3(kThreads), 0, st, u);
        GSX_LAUNCH_CHECK();
        hipLaunchKernelGGL((k_join<E, V, G>), grid_for(l.tiles, kJoinThreads / G, times),
                           dim3(kJoinThreads), 0, st, u);
        GSX_LAUNCH_CHECK();
        return GSX_OK;
    });
}

}  // namespace

extern "C" {

int gsx_embed_fwd(int32_t dtype, int64_t count, int64_t rows, int32_t width, const void* indices,
                  int32_t index64, const void* table, int64_t table_stride, float scale, void* y,
                  void* stream) {
    if (int e = check_args(dtype, count, rows, width, indices, index64, table, table_stride, scale))
        return e;
    if ((uintptr_t)y % (dtype == GSX_F32 ? 4 : 2)) return GSX_ERR_INVALID;
    if (count == 0) return GSX_OK;
    if (!y) return GSX_ERR_INVALID;
    Embed q{};
    q.table = table;
    q.indices = indices;
    q.y = y;
    q.count = count;
    q.rows = rows;
    q.stride = table_stride;
    q.width = width;
    q.index64 = index64;
    q.scale = scale;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == GSX_F32) return lookup<F32>(q, st);
    if (dtype == GSX_BF16) return lookup<BF16>(q, st);
    return lookup<F16>(q, st);
}

int64_t gsx_embed_bwd_workspace_bytes(int32_t dtype, int64_t count, int64_t rows, int32_t width) {
    if (int e = check_shape(dtype, count, rows, width)) return e;
    return layout(count, rows, width).total;
}

int gsx_embed_bwd(int32_t dtype, int64_t count, int64_t rows, int32_t width, const void* indices,
                  int32_t index64, const void* g_y, int64_t g_y_stride, float scale, void* g_table,
                  void* workspace, int64_t workspace_bytes, void* stream) {
    if (int e = check_args(dtype, count, rows, width, indices, index64, g_y, g_y_stride, scale))
        return e;
    if (!g_table || (uintptr_t)g_table % (dtype == GSX_F32 ? 4 : 2)) return GSX_ERR_INVALID;
    if ((uintptr_t)workspace % 16) return GSX_ERR_INVALID;
    if (!workspace || workspace_bytes < layout(count, rows, width).total) return GSX_ERR_WORKSPACE;
    Embed q{};
    q.g_y = g_y;
    q.indices = indices;
    q.g_table = g_table;
    q.count = count;
    q.rows = rows;
    q.stride = g_y_stride;
    q.width = width;
    q.index64 = index64;
    q.scale = scale;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == GSX_F32) return gradient<F32>(q, (char*)workspace, st);
    if (dtype == GSX_BF16) return gradient<BF16>(q, (char*)workspace, st);
    return gradient<F16>(q, (char*)workspace, st);
}

}  // extern "C"
