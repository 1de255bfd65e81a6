// embedding.hip -- rows of a table by their indices, and the table's gradient.
//
//   y_i = s T[k_i], zero where k_i lies outside the table
//   dT[v] = s sum over i with k_i = v of dy_i
//
// The gradient sorts the tokens (stably, so that a row's sum has one order) and
// walks them in tiles: a team of lanes adds up a tile's rows of dy as long as the
// key stays the same.  What begins and ends inside a tile is written at once; what
// tiles of a workgroup share is put together in shared memory, and what its block of
// tiles shares with its neighbours goes into two partial rows, which a last launch
// joins.  So a row that every token names is spread over as many lanes as rows that
// one token names, no sum depends on the order of arrival, and sums stay short: a
// tile's, a block's, then the blocks'.
//
// The sort is a stable radix sort by digits of 8 or 12 bits, three launches a pass: a
// chunk's counts of each digit, their prefix over the chunks, and the placement.  No
// workgroup waits for another one.  Tokens outside the table are left out of the
// first pass.  Up to 16 384 tokens are sorted by one workgroup in one launch.
//
// What a gradient has to move is dy and the table's gradient; the rows of dy are
// gathered, so they come in whole lines only where rows are whole lines.  Figures below
// are of 1 000 003 tokens, 4096 rows of 32 float32, unless they say otherwise.
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
// a chunk of the sort: 16 waves of 4 rounds place it 10 % sooner than 8 of 8
constexpr int kSortThreads = 1024, kItems = 4, kChunk = kSortThreads * kItems;
constexpr int kScanGroups = 16;  // of chunks, in the prefix
constexpr int kFewItems = 16;    // tokens of a thread, where one workgroup sorts them all
constexpr int kMostTile = 256;   // sorted tokens that a team of lanes adds up, at most
constexpr int kLook = 4;         // tokens that a team looks up at a time
constexpr int kBatch = 8;        // rows that a team asks for at a time
constexpr int kSpan = 32;        // blocks of a row that a single team joins, at most
constexpr int kJoinThreads = 512;

struct Embed {
    const void *table, *g_y, *indices;
    void *y, *g_table;
    int64_t count, rows, stride;  // stride of the table's or of g_y's rows
    int width, index64;
    float scale;
};

// Token i's row, or -1.
__device__ __forceinline__ int64_t row_of(const Embed& q, int64_t i) {
    const int64_t k =
        q.index64 ? ((const int64_t*)q.indices)[i] : (int64_t)((const int32_t*)q.indices)[i];
    return k >= 0 && k < q.rows ? k : -1;
}

// G lanes a token, a piece of V elements each; blockIdx.y: pieces from 64 on.  A team
// takes kLook tokens at a time, whose indices are asked for together, and then the rows.
// Bound by y's stores: 34 us, 3.8 TB/s (one token a time 36; 921 600 x 48 bfloat16 26,
// one at a time 31).
template <class E, int V, int G>
__global__ __launch_bounds__(kThreads) void k_lookup(const Embed q) {
    using P = Piece<E, V>;
    using T = typename E::T;
    constexpr int kTeams = kThreads / G;
    const int at = (blockIdx.y * G + threadIdx.x % G) * V;
    if (at >= q.width) return;
    const int c = min(at, q.width - V);
    const int64_t step = (int64_t)gridDim.x * (kTeams * kLook);
    for (int64_t i = (int64_t)blockIdx.x * (kTeams * kLook) + threadIdx.x / G; i < q.count;
         i += step) {
        int64_t k[kLook];
        typename P::Raw raw[kLook];
#pragma unroll
        for (int u = 0; u < kLook; ++u) k[u] = row_of(q, min(i + u * kTeams, q.count - 1));
#pragma unroll
        for (int u = 0; u < kLook; ++u)
            raw[u] = P::load((const T*)q.table + max(k[u], (int64_t)0) * q.stride + c);
#pragma unroll
        for (int u = 0; u < kLook; ++u) {
            if (i + u * kTeams >= q.count) break;
            float v[V];
            P::up(raw[u], v);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = k[u] >= 0 ? v[e] * q.scale : 0.f;
            P::store((T*)q.y + (i + u * kTeams) * q.width + c, P::down(v));
        }
    }
}

// ----------------------------------------------------------------- sort --

struct Sort {
    Embed q;
    const uint2* from;  // (key, token), or NULL: the indices
    uint2* to;
    uint32_t* counts;   // (chunks, 2^BITS)
    uint32_t* totals;   // 2^BITS
    uint32_t* live;     // how many tokens name a row
    int chunks, shift, bits;
    int64_t zeros;      // bytes of the table's gradient, cleared beside the first counts
};

// Clears the table's gradient: workgroup `at` of `of`.
template <int THREADS>
__device__ __forceinline__ void clear(const Sort& s, int64_t at, int64_t of) {
    // whole vectors from the first aligned address on, single bytes before and behind
    uint8_t* p = (uint8_t*)s.q.g_table;
    const int64_t head = min<int64_t>((16 - (uintptr_t)p % 16) % 16, s.zeros);
    const int64_t vectors = (s.zeros - head) / 16, tail = s.zeros - head - vectors * 16;
    u32x4* v = (u32x4*)(p + head);
    for (int64_t i = at * THREADS + threadIdx.x; i < vectors; i += of * THREADS)
        v[i] = u32x4{0, 0, 0, 0};
    if (at == 0 && (int)threadIdx.x < head) p[threadIdx.x] = 0;
    if (at == 0 && (int)threadIdx.x < tail) p[head + vectors * 16 + threadIdx.x] = 0;
}

constexpr uint32_t kNone = ~0u;  // the key of a place without a pair; rows lie below 2^30

// Keys and tokens at places base + own, base + own + step, ... of the pass's n; all are
// asked for before the first is looked at.  base, the same in the whole workgroup, lies
// below the number of tokens.
template <int ITEMS>
__device__ __forceinline__ void load_indices(const Sort& s, int64_t base, int own, int step,
                                             uint32_t* key, uint32_t* token) {
    const int left = (int)min<int64_t>(s.q.count - base, 1 << 20);
    uint32_t high[ITEMS];
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        const uint32_t at = (uint32_t)min(own + r * step, left - 1);
        if (s.q.index64) {
            const uint2 v = ((const uint2*)s.q.indices + base)[at];
            key[r] = v.x;
            high[r] = v.y;
        } else {
            key[r] = ((const uint32_t*)s.q.indices + base)[at];
            high[r] = 0;
        }
    }
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        // an index of 32 bits that is negative is not below 2^30
        const bool there = own + r * step < left && high[r] == 0 && key[r] < (uint32_t)s.q.rows;
        key[r] = there ? key[r] : kNone;
        token[r] = (uint32_t)base + (uint32_t)(own + r * step);
    }
}
template <int ITEMS>
__device__ __forceinline__ void load_pairs(const Sort& s, int64_t base, int own, int step,
                                           uint32_t* key, uint32_t* token) {
    if (!s.from) return load_indices<ITEMS>(s, base, own, step, key, token);
    const int left = (int)min<int64_t>(max<int64_t>((int64_t)*s.live - base, 0), 1 << 20);
    const uint2* from = s.from + base;
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        const uint2 v = from[max(min(own + r * step, left - 1), 0)];
        key[r] = v.x;
        token[r] = v.y;
    }
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) key[r] = own + r * step < left ? key[r] : kNone;
}

// The first s.chunks workgroups count (4 us); those behind clear the gradient.
template <int BITS>
__global__ __launch_bounds__(kSortThreads) void k_count(const Sort s) {
    constexpr int kRadix = 1 << BITS;
    __shared__ uint32_t hist[kRadix];
    if ((int)blockIdx.x >= s.chunks) {
        clear<kSortThreads>(s, blockIdx.x - s.chunks, gridDim.x - s.chunks);
        return;
    }
    for (int d = threadIdx.x; d < kRadix; d += kSortThreads) hist[d] = 0;
    __syncthreads();
    uint32_t key[kItems], token[kItems];
    load_pairs<kItems>(s, (int64_t)blockIdx.x * kChunk, threadIdx.x, kSortThreads, key, token);
#pragma unroll
    for (int r = 0; r < kItems; ++r)
        if (key[r] != kNone) atomicAdd(&hist[key[r] >> s.shift & (kRadix - 1)], 1u);
    __syncthreads();
    for (int d = threadIdx.x; d < kRadix; d += kSortThreads)
        s.counts[(int64_t)blockIdx.x * kRadix + d] = hist[d];
}

// Each digit's prefix over the chunks, in place, and its total: 64 digits a
// workgroup, the chunks in kScanGroups stretches (4 us).
template <int BITS>
__global__ __launch_bounds__(64 * kScanGroups) void k_prefix(const Sort s) {
    constexpr int kRadix = 1 << BITS, kHeld = 16;
    __shared__ uint32_t sums[kScanGroups][64];
    const int lane = threadIdx.x & 63, g = threadIdx.x >> 6;
    const int d = blockIdx.x * 64 + lane;
    const int per = (s.chunks + kScanGroups - 1) / kScanGroups;
    const int first = min(g * per, s.chunks), end = min(first + per, s.chunks);
    // the first kHeld counts stay in registers
    uint32_t v[kHeld], sum = 0;
#pragma unroll
    for (int k = 0; k < kHeld; ++k)
        v[k] = first + k < end ? s.counts[(int64_t)(first + k) * kRadix + d] : 0;
#pragma unroll
    for (int k = 0; k < kHeld; ++k) sum += v[k];
#pragma unroll 8
    for (int c = first + kHeld; c < end; ++c) sum += s.counts[(int64_t)c * kRadix + d];
    sums[g][lane] = sum;
    __syncthreads();
    uint32_t run = 0, total = 0;
#pragma unroll
    for (int k = 0; k < kScanGroups; ++k) {
        if (k < g) run += sums[k][lane];
        total += sums[k][lane];
    }
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
        if (first + k < end) s.counts[(int64_t)(first + k) * kRadix + d] = run;
        run += v[k];
    }
#pragma unroll 8
    for (int c = first + kHeld; c < end; ++c) {
        uint32_t* at = s.counts + (int64_t)c * kRadix + d;
        const uint32_t t = *at;
        *at = run;
        run += t;
    }
    if (g == 0) s.totals[d] = total;
}

// Lanes of the wave, among the valid ones, with the same digit: those that differ in no
// bit.  A bit's ballot, against this lane's bit in all places, gives those that do.
__device__ __forceinline__ uint64_t same_digit(uint32_t d, bool valid, int bits) {
    uint32_t lo = 0, hi = 0;
    for (int b = 0; b < bits; ++b) {
        const uint32_t own = (uint32_t)((int)(d << (31 - b)) >> 31);
        const uint64_t set = __ballot(own);
        lo = __builtin_amdgcn_bitop3_b32(lo, (uint32_t)set, own, 0xf6);  // a | b ^ c
        hi = __builtin_amdgcn_bitop3_b32(hi, (uint32_t)(set >> 32), own, 0xf6);
    }
    return ~((uint64_t)hi << 32 | lo) & __ballot(valid);
}

// The rank of each of a wave's first `rounds` items a lane among those of its digit, in
// their order, with cnt[d] (zero before) left as the digit's count.
template <int ITEMS, int RADIX>
__device__ __forceinline__ void wave_ranks(const uint32_t* key, int shift, int bits, int rounds,
                                           uint16_t* cnt, uint32_t* rank) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        rank[r] = 0;
        if (r < rounds) {
            const uint32_t d = key[r] >> shift & (RADIX - 1);
            const uint64_t same = same_digit(d, key[r] != kNone, bits);
            const uint64_t before = same & ((1ull << lane) - 1);
            const uint32_t c = cnt[d];
            rank[r] = c + (uint32_t)__popcll(before);
            wave_fence();
            if (key[r] != kNone && before == 0) cnt[d] = (uint16_t)(c + (uint32_t)__popcll(same));
            wave_fence();
        }
    }
}

// Exclusive sums over a workgroup of THREADS, with the total.  `room`: THREADS / 64
// words, free again after the next barrier.
template <int THREADS>
__device__ __forceinline__ uint32_t prefix_sum(uint32_t v, uint32_t* room, uint32_t* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t incl = wave_incl_scan(v);
    if (lane == 63) room[wave] = incl;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        if (w < wave) before += room[w];
        all += room[w];
    }
    *total = all;
    return before + incl - v;
}

// Up to 8 bits the chunk is regrouped by digit first, so that stores are runs; with
// more digits than a chunk has tokens there are none.  A wave's counts are 16 bits, two
// digits a word, which are added up as words: a chunk's 4096 tokens do not carry.
// 16 us with 12 bits, most of it scattered stores of 8 bytes, which write 27 MB of lines
// for 8 (counts digit by digit, not in words, 25 us); 10 us and 8 MB with 8 bits.
template <int BITS>
__global__ __launch_bounds__(kSortThreads) void k_place(const Sort s) {
    constexpr int kRadix = 1 << BITS, kWaves = kSortThreads / 64, kWords = kRadix / 2;
    constexpr int kEach = kWords > kSortThreads ? kWords / kSortThreads : 1;  // words a thread
    constexpr bool kRegroup = BITS <= 8;
    using Words = __attribute__((ext_vector_type(kEach))) uint32_t;
    using Bases = __attribute__((ext_vector_type(2 * kEach))) uint32_t;
    static_assert(kChunk < 1 << 16, "counts of 16 bits");
    __shared__ alignas(16) uint16_t cnt[kWaves][kRadix];
    __shared__ alignas(16) uint32_t base[kRadix];
    __shared__ uint32_t room[2][kWaves];
    __shared__ uint32_t in_chunk[kRegroup ? kRadix : 1];
    __shared__ uint2 pairs[kRegroup ? kChunk : 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int k = tid; k < kWaves * kRadix / 8; k += kSortThreads)
        ((u32x4*)cnt)[k] = u32x4{0, 0, 0, 0};
    uint32_t key[kItems], token[kItems], rank[kItems];
    load_pairs<kItems>(s, (int64_t)blockIdx.x * kChunk, wave * (64 * kItems) + lane, 64, key,
                       token);
    Bases before = 0, total = 0;
    const bool mine = tid * kEach < kWords;
    if (mine) {
        total = ((const Bases*)s.totals)[tid];
        before = ((const Bases*)(s.counts + (int64_t)blockIdx.x * kRadix))[tid];
    }
    uint32_t sum = 0, live, held = 0;
#pragma unroll
    for (int k = 0; k < 2 * kEach; ++k) sum += total[k];
    uint32_t at = prefix_sum<kSortThreads>(sum, room[0], &live);  // its barrier: cnt is clear
    wave_ranks<kItems, kRadix>(key, s.shift, s.bits, kItems, cnt[wave], rank);
    // the first pass counts the tokens that name a row
    if (!s.from && blockIdx.x == 0 && tid == 0) *s.live = live;
    __syncthreads();
    Words own = 0;
    if (mine) {
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            Words* c = (Words*)cnt[w] + tid;
            const Words v = *c;
            *c = own;
            own += v;
        }
#pragma unroll
        for (int k = 0; k < 2 * kEach; ++k) {
            before[k] += at;
            at += total[k];
        }
        ((Bases*)base)[tid] = before;
    }
    if constexpr (kRegroup) {
        static_assert(kEach == 1, "two digits a thread");
        const uint32_t first = own[0] & 0xffffu, second = own[0] >> 16;
        const uint32_t start = prefix_sum<kSortThreads>(first + second, room[1], &held);
        if (mine) {
            in_chunk[2 * tid] = start;
            in_chunk[2 * tid + 1] = start + first;
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kItems; ++r)
        if (key[r] != kNone) {
            const uint32_t d = key[r] >> s.shift & (kRadix - 1), k = cnt[wave][d] + rank[r];
            if constexpr (kRegroup) pairs[in_chunk[d] + k] = make_uint2(key[r], token[r]);
            else s.to[base[d] + k] = make_uint2(key[r], token[r]);
        }
    if constexpr (kRegroup) {
        __syncthreads();
        for (int j = tid; j < (int)held; j += kSortThreads) {
            const uint2 e = pairs[j];
            const uint32_t d = (e.x >> s.shift) & (kRadix - 1);
            s.to[base[d] + (uint32_t)j - in_chunk[d]] = e;
        }
    }
}

// All passes over few tokens by one workgroup, in shared memory; the others clear the
// gradient.  The waves share the tokens evenly, `rounds` times 64 each.  8205 tokens of
// 50 000 rows 23 to 25 us, bound by one compute unit's ranking; the six launches of two
// passes take 31 (a gradient of 512 float16 columns 34 us a call, with those 41).
constexpr int kFewThreads = 1024;
template <int ITEMS>
__global__ __launch_bounds__(kFewThreads) void k_sort_few(const Sort s) {
    constexpr int kWaves = kFewThreads / 64, kRadix = 256;
    __shared__ uint2 pairs[kFewThreads * ITEMS];
    __shared__ alignas(16) uint16_t cnt[kWaves][kRadix];
    __shared__ uint32_t start[kRadix], room[kWaves];
    if (blockIdx.x > 0) {
        clear<kFewThreads>(s, blockIdx.x - 1, gridDim.x - 1);
        return;
    }
    const int tid = threadIdx.x, wave = tid >> 6;
    const int rounds = ((int)s.q.count + kFewThreads - 1) / kFewThreads;  // ITEMS at most
    const int first = wave * 64 * rounds + (tid & 63);
    uint32_t key[ITEMS], token[ITEMS];
    load_indices<ITEMS>(s, 0, first, 64, key, token);
#pragma unroll
    for (int r = 0; r < ITEMS; ++r)
        if (r >= rounds) key[r] = kNone;  // another wave's
    uint32_t live = 0;
    for (int shift = 0; shift < s.bits; shift += 8) {
        for (int k = tid; k < kWaves * kRadix / 8; k += kFewThreads)
            ((u32x4*)cnt)[k] = u32x4{0, 0, 0, 0};
        __syncthreads();
        uint32_t rank[ITEMS];
        wave_ranks<ITEMS, kRadix>(key, shift, min(s.bits - shift, 8), rounds, cnt[wave], rank);
        __syncthreads();
        uint32_t mine = 0;
        if (tid < kRadix) {
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const uint32_t c = cnt[w][tid];
                cnt[w][tid] = (uint16_t)mine;
                mine += c;
            }
        }
        const uint32_t at = prefix_sum<kFewThreads>(mine, room, &live);
        if (tid < kRadix) start[tid] = at;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ITEMS; ++r)
            if (key[r] != kNone) {
                // (formed again: kept, the places of 16 digits take too many registers)
                const uint32_t d = (uint32_t)here((int)key[r]) >> shift & (kRadix - 1);
                pairs[start[d] + cnt[wave][d] + rank[r]] = make_uint2(key[r], token[r]);
            }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ITEMS; ++r) {
            const uint32_t i = (uint32_t)(first + r * 64);
            const bool there = r < rounds && i < live;
            const uint2 e = pairs[there ? i : 0];
            key[r] = there ? e.x : kNone;
            token[r] = e.y;
        }
    }
#pragma unroll
    for (int r = 0; r < ITEMS; ++r)
        if (key[r] != kNone) s.to[first + r * 64] = make_uint2(key[r], token[r]);
    if (tid == 0) *s.live = live;
}

// ------------------------------------------------------------------ sum --

struct Sum {
    Embed q;
    const uint2* pairs;
    const uint32_t* live;
    int tile;          // sorted tokens of a tile
    int block;         // and of the tiles of one workgroup
    uint32_t* begins;  // of a row that spans blocks, the first; others' are not set
    float* parts;      // (blocks, 2, width): what a block shares with the one before, and behind
};

// What a tile leaves to others: of the row that was open at its begin, and of the row
// that is open at its end.  A tile within one row (whole) has the first alone.
struct Edges {
    bool open, more, whole;
    uint32_t first_key, last_key;
};

template <class E, int V>
__device__ __forceinline__ void write_row(const Embed& q, uint32_t key, int c, const float* acc) {
    using P = Piece<E, V>;
    float v[V];
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = acc[e] * q.scale;
    P::store((typename E::T*)q.g_table + (int64_t)key * q.width + c, P::down(v));
}

// One tile, V columns of it: rows that begin and end in it are written, the others go to
// head and tail.  A batch of rows is asked for before the first is added: 30 us, 4.3 TB/s
// of gathered rows (row by row 62).
template <class E, int V>
__device__ __forceinline__ Edges tile_sum(const Sum& s, int64_t tile, int64_t live, int c,
                                          float* head, float* tail) {
    using P = Piece<E, V>;
    using T = typename E::T;
    const Embed& q = s.q;
    const int64_t first = tile * s.tile;
    if (first >= live) return Edges{false, false, false, 0, 0};
    const int n = (int)min<int64_t>(s.tile, live - first);
    const uint2* pairs = s.pairs + first;
    uint32_t key = pairs[0].x;
    Edges edges;
    edges.first_key = key;
    edges.open = first > 0 && pairs[-1].x == key;
    edges.more = first + n < live && pairs[n].x == pairs[n - 1].x;
    bool open = edges.open;
    float acc[V] = {};
    auto close = [&]() {
        if (open) {
#pragma unroll
            for (int e = 0; e < V; ++e) head[e] = acc[e];
        } else {
            write_row<E, V>(q, key, c, acc);
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
                close();
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
    edges.last_key = key;
    edges.whole = edges.more && open;
    if (!edges.more || open) {
        close();
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) tail[e] = acc[e];
    }
    return edges;
}

// G lanes a tile, a piece of V columns each.  Rows that span tiles of one workgroup are
// put together in shared memory, each by the team in whose tile it ends; what leaves the
// workgroup's block of tiles goes to its parts.
template <class E, int V, int G>
__global__ __launch_bounds__(kThreads) void k_tile_sums(const Sum s) {
    constexpr int kTeams = kThreads / G;
    constexpr int kBack = V == 8 ? 4 : 8;  // tiles that are looked at together
    __shared__ float heads[kTeams][G][V], tails[kTeams][G][V];
    __shared__ bool whole[kTeams];
    const Embed& q = s.q;
    const int team = threadIdx.x / G, lane = threadIdx.x % G;
    const int at = (blockIdx.y * G + lane) * V;
    const bool here = at < q.width;
    const int c = min(at, q.width - V);
    const int64_t live = *s.live;
    for (int64_t block = blockIdx.x; block * s.block < live; block += gridDim.x) {
        const Edges mine = tile_sum<E, V>(s, block * kTeams + team, live, c, heads[team][lane],
                                    tails[team][lane]);
        if (lane == 0) whole[team] = mine.whole;
        __syncthreads();
        // Adds the tiles before `team`, last first, to where the row begins; true if it
        // begins before this block.
        auto reach_back = [&](float* acc) {
            int begin = team - 1;  // the tile whose tail it is, or -1
            for (bool on = true; on; ) {
                bool within[kBack];
                float v[kBack][V];
#pragma unroll
                for (int u = 0; u < kBack; ++u) {
                    const int t = max(begin - u, 0);
                    within[u] = begin - u >= 0 && whole[t];
#pragma unroll
                    for (int e = 0; e < V; ++e) v[u][e] = heads[t][lane][e];
                }
                int passed = 0;
#pragma unroll
                for (int u = 0; u < kBack; ++u) {
                    on = on && within[u];
                    passed += on;
#pragma unroll
                    for (int e = 0; e < V; ++e) acc[e] += on ? v[u][e] : 0.f;
                }
                begin -= passed;
            }
            if (begin < 0) return true;
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] += tails[begin][lane][e];
            return false;
        };
        float* part = s.parts + block * 2 * q.width + c;
        if (here && mine.open && !mine.whole) {
            float acc[V];
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] = heads[team][lane][e];
            if (reach_back(acc)) store_floats<V>(part, acc);
            else write_row<E, V>(q, mine.first_key, c, acc);
        }
        // the row that goes on behind the block
        if (here && team == kTeams - 1 && mine.more) {
            float acc[V];
            bool before = false;
#pragma unroll
            for (int e = 0; e < V; ++e)
                acc[e] = mine.whole ? heads[team][lane][e] : tails[team][lane][e];
            if (mine.whole) before = reach_back(acc);
            store_floats<V>(before ? part : part + q.width, acc);
            if (!before) s.begins[mine.last_key] = (uint32_t)block;
        }
        __syncthreads();
    }
}

// How many blocks before this one share the row that is open at its begin and ends in
// it; 0 if there is none.
__device__ __forceinline__ int64_t span_of(const Sum& s, int64_t block, int64_t live) {
    const int64_t first = block * s.block, next = first + s.block;
    if (first == 0 || first >= live) return 0;
    const uint32_t key = s.pairs[first].x;
    if (s.pairs[first - 1].x != key || (next < live && s.pairs[next].x == key)) return 0;
    return block - (int64_t)s.begins[key];
}

// Adds up a row's parts in blocks first, first + step, ... below end.
template <int V>
__device__ __forceinline__ void add_parts(const Sum& s, int64_t first, int64_t end, int64_t step,
                                          int c, float* acc) {
    constexpr int kParts = V == 8 ? 12 : 16;  // in flight, as registers allow
    for (int64_t t = first; t < end; t += kParts * step) {
        float v[kParts][V];
#pragma unroll
        for (int u = 0; u < kParts; ++u)
            load_floats<V>(s.parts + min(t + u * step, end - 1) * 2 * s.q.width + c, v[u]);
#pragma unroll
        for (int u = 0; u < kParts; ++u)
            if (t + u * step < end) {
#pragma unroll
                for (int e = 0; e < V; ++e) acc[e] += v[u][e];
            }
    }
}

// Rows over several blocks, each by a team of lanes for the block in which it ends;
// over more than kSpan, by all teams of the workgroup together.  5 us, most of it four
// loads one after another; 7 for 921 600 tokens of 201 rows, 48 bfloat16.  (Parts by the
// tile, not by the block: 7 and 16, and by single teams, however many, 431 and 1198: the
// most popular rows have 62 000 and 157 000 tokens.)
template <class E, int V, int G>
__global__ __launch_bounds__(kJoinThreads) void k_join(const Sum s) {
    constexpr int kTeams = kJoinThreads / G;
    __shared__ float room[kJoinThreads / 64][G][V + 1];
    __shared__ int64_t spans[kTeams];  // the long ones
    __shared__ int teams[kTeams], found;
    const Embed& q = s.q;
    const int team = threadIdx.x / G, at = (blockIdx.y * G + threadIdx.x % G) * V;
    const int c = min(at, q.width - V);
    const int64_t live = *s.live, step = (int64_t)gridDim.x * kTeams;
    auto write = [&](int64_t block, const float* acc) {
        if (at < q.width) write_row<E, V>(q, s.pairs[block * s.block].x, c, acc);
    };
    for (int64_t base = (int64_t)blockIdx.x * kTeams; base * s.block < live; base += step) {
        const int64_t block = base + team, span = span_of(s, block, live);
        if (span > 0 && span <= kSpan) {
            float acc[V];
            load_floats<V>(s.parts + ((block - span) * 2 + 1) * q.width + c, acc);
            add_parts<V>(s, block - span + 1, block + 1, 1, c, acc);
            write(block, acc);
        }
        if (!__syncthreads_or(span > kSpan)) continue;
        if (threadIdx.x == 0) found = 0;
        __syncthreads();
        if (threadIdx.x % G == 0 && span > kSpan) {
            // in any order: each is a sum of its own
            const int k = atomicAdd(&found, 1);
            spans[k] = span;
            teams[k] = team;
        }
        __syncthreads();
        const int n_long = found;
        for (int k = 0; k < n_long; ++k) {
            const int64_t far = spans[k], own = base + teams[k];
            float acc[V] = {};
            if (team == 0) load_floats<V>(s.parts + ((own - far) * 2 + 1) * q.width + c, acc);
            add_parts<V>(s, own - far + 1 + team, own + 1, kTeams, c, acc);
            // a wave's teams, then the waves
#pragma unroll
            for (int e = 0; e < V; ++e)
#pragma unroll
                for (int o = G; o < 64; o <<= 1) acc[e] += __shfl_xor(acc[e], o, 64);
            const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
            if (lane < G) {
#pragma unroll
                for (int e = 0; e < V; ++e) room[wave][lane][e] = acc[e];
            }
            __syncthreads();
            if (team == 0) {
#pragma unroll
                for (int e = 0; e < V; ++e) acc[e] = 0.f;
                for (int w = 0; w < kJoinThreads / 64; ++w)
#pragma unroll
                    for (int e = 0; e < V; ++e) acc[e] += room[w][lane][e];
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
    int chunks, passes, bits, digit, tile, block;
    bool few;
    int64_t blocks, counts, totals, live, pairs[2], begins, parts, total;
};

Layout layout(int dtype, int64_t count, int64_t rows, int32_t width) {
    Layout l{};
    l.chunks = (int)((count + kChunk - 1) / kChunk);
    l.bits = 1;
    while (((int64_t)1 << l.bits) < rows) ++l.bits;
    l.few = count <= kFewThreads * kFewItems;
    // One pass of 12 bits instead of two of 8: 25 us for 34; two of 12 for two of 8 lose
    // (200 000 tokens 39 us for 29), whose stores are runs.
    l.digit = l.bits <= 8 || (l.bits > 12 && l.bits <= 16) ? 8 : 12;
    l.passes = l.few ? 1 : (l.bits + l.digit - 1) / l.digit;
    // Lanes of a team, and teams beside each other, as for_width has them: about 2^16
    // lanes are enough for the sums, in tiles of at least a batch.  8205 x 512 float16 in
    // tiles of 8: 7 us, of 64: 20; more lanes leave more to put together (all kernels of
    // 1 000 003 x 32 float32 with 2^16, 2^17 and 2^18 lanes: 94, 96 and 97 us).
    const int vec = dtype == GSX_F32 ? F32::VEC : BF16::VEC;
    const int64_t pieces = width < vec ? width : (width + vec - 1) / vec;
    l.tile = kMostTile;
    while (l.tile > kBatch && count * pieces < ((int64_t)1 << 16) * l.tile) l.tile /= 2;
    int lanes = 1;
    while (lanes < 64 && lanes < pieces) lanes *= 2;
    l.block = l.tile * (kThreads / lanes);
    l.blocks = (count + l.block - 1) / l.block;
    const int64_t radix = l.few ? 0 : 1 << l.digit;
    l.live = 0;
    l.totals = 256;
    l.counts = l.totals + radix * 4;
    l.pairs[0] = up_to(l.counts + l.chunks * radix * 4, 256);
    l.pairs[1] = up_to(l.pairs[0] + count * 8, 256);
    l.begins = up_to(l.pairs[1] + (l.passes > 1 ? count * 8 : 0), 256);
    l.parts = up_to(l.begins + (l.blocks > 1 ? rows * 4 : 0), 256);
    l.total = up_to(l.parts + l.blocks * 2 * width * 4, 256);
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
        hipLaunchKernelGGL((k_lookup<E, V, G>), grid_for(q.count, kThreads / G * kLook, times),
                           dim3(kThreads), 0, st, q);
        GSX_LAUNCH_CHECK();
        return GSX_OK;
    });
}

template <int BITS>
int passes(Sort s, const Layout& l, char* ws, unsigned fill, hipStream_t st) {
    for (int p = 0; p < l.passes; ++p) {
        s.from = p ? (const uint2*)(ws + l.pairs[(p - 1) % 2]) : nullptr;
        s.to = (uint2*)(ws + l.pairs[p % 2]);
        s.shift = p * BITS;
        s.bits = l.bits - s.shift < BITS ? l.bits - s.shift : BITS;
        hipLaunchKernelGGL((k_count<BITS>), dim3((unsigned)l.chunks + (p ? 0 : fill)),
                           dim3(kSortThreads), 0, st, s);
        GSX_LAUNCH_CHECK();
        hipLaunchKernelGGL((k_prefix<BITS>), dim3((1 << BITS) / 64), dim3(64 * kScanGroups), 0, st,
                           s);
        GSX_LAUNCH_CHECK();
        hipLaunchKernelGGL((k_place<BITS>), dim3((unsigned)l.chunks), dim3(kSortThreads), 0, st, s);
        GSX_LAUNCH_CHECK();
    }
    return GSX_OK;
}

template <class E>
int gradient(int dtype, const Embed& q, char* ws, hipStream_t st) {
    const Layout l = layout(dtype, q.count, q.rows, q.width);
    Sort s{};
    s.q = q;
    s.counts = (uint32_t*)(ws + l.counts);
    s.totals = (uint32_t*)(ws + l.totals);
    s.live = (uint32_t*)(ws + l.live);
    s.chunks = l.chunks;
    s.zeros = q.rows * q.width * (int64_t)sizeof(typename E::T);
    const int64_t fill = (s.zeros + (1 << 15) - 1) >> 15;
    const unsigned fillers = (unsigned)(fill < 2048 ? fill : 2048);
    if (q.count == 0) {
        s.chunks = 0;
        hipLaunchKernelGGL((k_count<8>), dim3(fillers), dim3(kSortThreads), 0, st, s);
        GSX_LAUNCH_CHECK();
        return GSX_OK;
    }
    if (l.few) {
        s.to = (uint2*)(ws + l.pairs[0]);
        s.bits = l.bits;
        const dim3 grid(1 + fillers);
        if (q.count <= kFewThreads)
            hipLaunchKernelGGL((k_sort_few<1>), grid, dim3(kFewThreads), 0, st, s);
        else if (q.count <= kFewThreads * 4)
            hipLaunchKernelGGL((k_sort_few<4>), grid, dim3(kFewThreads), 0, st, s);
        else
            hipLaunchKernelGGL((k_sort_few<kFewItems>), grid, dim3(kFewThreads), 0, st, s);
        GSX_LAUNCH_CHECK();
    } else if (int e = l.digit == 8 ? passes<8>(s, l, ws, fillers, st)
                                    : passes<12>(s, l, ws, fillers, st)) {
        return e;
    }
    Sum u{};
    u.q = q;
    u.pairs = (const uint2*)(ws + l.pairs[(l.passes - 1) % 2]);
    u.begins = (uint32_t*)(ws + l.begins);
    u.live = s.live;
    u.tile = l.tile;
    u.block = l.block;
    u.parts = (float*)(ws + l.parts);
    return for_width<E>(q.width, [&](auto v, auto g, int times) -> int {
        constexpr int V = decltype(v)::value, G = decltype(g)::value;
        const dim3 grid = grid_for(l.blocks, 1, times);
        hipLaunchKernelGGL((k_tile_sums<E, V, G>), grid, dim3(kThreads), 0, st, u);
        GSX_LAUNCH_CHECK();
        if (l.blocks == 1) return GSX_OK;
        hipLaunchKernelGGL((k_join<E, V, G>), grid_for(l.blocks, kJoinThreads / G, times),
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
    return layout(dtype, count, rows, width).total;
}

int gsx_embed_bwd(int32_t dtype, int64_t count, int64_t rows, int32_t width, const void* indices,
                  int32_t index64, const void* g_y, int64_t g_y_stride, float scale, void* g_table,
                  void* workspace, int64_t workspace_bytes, void* stream) {
    if (int e = check_args(dtype, count, rows, width, indices, index64, g_y, g_y_stride, scale))
        return e;
    if (!g_table || (uintptr_t)g_table % (dtype == GSX_F32 ? 4 : 2)) return GSX_ERR_INVALID;
    if ((uintptr_t)workspace % 16) return GSX_ERR_INVALID;
    if (!workspace || workspace_bytes < layout(dtype, count, rows, width).total) return GSX_ERR_WORKSPACE;
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
    if (dtype == GSX_F32) return gradient<F32>(dtype, q, (char*)workspace, st);
    if (dtype == GSX_BF16) return gradient<BF16>(dtype, q, (char*)workspace, st);
    return gradient<F16>(dtype, q, (char*)workspace, st);
}

}  // extern "C"
