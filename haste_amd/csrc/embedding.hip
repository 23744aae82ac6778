// Embedding lookup with scaling, y[n] = s W[t_n], and the table's gradient by sorted tokens,
// dW[v] = s sum_{n: t_n = v} dy[n], summed in fp32 in a fixed order (no float atomics).
// Both are bound by HBM; the gradient's table is written once, rows without a token among it.
// Measured at 65,536 tokens of 32,000 in bf16 rows of 768: lookup 30 us (142 MB, 4.8 TB/s); gradient 85 us
// in seven launches: sort 23, first places 5, sums 37 (132 MB, 3.6 TB/s: rows of dy in the tokens'
// order), joined 7.  8191 tokens of 20,011, fp32 rows of 301: lookup 6, gradient 46, latency of the launches.
#include <algorithm>
#include <type_traits>

#include "elements.hpp"

namespace haste {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ int64_t token_at(const void* t, bool wide, int64_t i) {
    return wide ? static_cast<const int64_t*>(t)[i] : (int64_t)static_cast<const int32_t*>(t)[i];
}

// Threads of a row: a power of two up to a wave that has a 16-byte vector for each.
int row_threads(int64_t vectors) {
    int t = 1;
    while (t < 64 && t < vectors) t *= 2;
    return t;
}

// ---------------------------------------------------------------- lookup ----
template <int DT, int V>
__global__ __launch_bounds__(kThreads) void emb_kernel(const void* tokens, int wide, const char* w,
                                                       int64_t ldw, char* y, int64_t N, int64_t rows,
                                                       int64_t D, float scale, int tpr) {
    constexpr int SZ = kElemBytes<DT>;
    const int64_t n = (int64_t)blockIdx.x * (kThreads / tpr) + threadIdx.x / tpr;
    if (n >= N) return;
    const int64_t t = token_at(tokens, wide, n);
    const bool in = t >= 0 && t < rows;
    const char* src = w + (in ? t : 0) * ldw * SZ;
    char* dst = y + n * D * SZ;
    for (int64_t i = (int64_t)(threadIdx.x % tpr) * V; i < D; i += tpr * V) {
        // (the last vector of a row that is no whole number of them shares elements with the one before)
        const int64_t at = min(i, D - V);
        float f[V];
        if constexpr (V == 1) {
            store_elem<DT>(dst, at, in ? load_elem<DT>(src, at) * scale : 0.f);
        } else {
            Elems<DT, V> v{};
            if (in) v = load<DT, V>(src, at);
            unpack<DT, V>(v, f);
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] *= scale;
            store<DT, V>(dst, at, pack<DT, V>(f));
        }
    }
}

// ------------------------------------------------------------------ sort ----
// Positions by token, stable: passes over digits of the token, least significant first.  A pass
// counts each tile's digits, turns the counts into first places (digits in order, tiles in order
// within a digit), and moves.  Tokens that take no gradient are keyed V, behind all others.
// Up to kSmall tokens are sorted by one workgroup in LDS, all passes in one launch.
constexpr int kTile = 1024, kMaxBins = 1024, kOwnScan = 64;
constexpr int kSmall = 2048, kSmallThreads = 1024;

__device__ __forceinline__ uint32_t sort_key(const void* tokens, bool wide, int64_t i, int64_t V,
                                             int64_t padding) {
    const int64_t t = token_at(tokens, wide, i);
    return (uint32_t)(t >= 0 && t < V && t != padding ? t : V);
}

struct SortPass {
    const void* tokens;            // first pass: keys are made from the tokens
    int wide;
    int64_t V, padding;
    const uint32_t *key_in, *at_in;
    uint32_t *key_out, *at_out;
    uint32_t* counts;
    int64_t N;
    int tiles, shift, bits;
};

// Counts lie by digit and tile for sort_scan_kernel, by tile and digit for the tiles' own sums.
__device__ __forceinline__ int64_t count_at(const SortPass& p, int digit, int tile) {
    return p.tiles > kOwnScan ? (int64_t)digit * p.tiles + tile : ((int64_t)tile << p.bits) + digit;
}

__global__ __launch_bounds__(kThreads) void sort_count_kernel(SortPass p) {
    __shared__ uint32_t hist[kMaxBins];
    const int bins = 1 << p.bits;
    for (int b = threadIdx.x; b < bins; b += kThreads) hist[b] = 0;
    __syncthreads();
    const int64_t i0 = (int64_t)blockIdx.x * kTile;
#pragma unroll
    for (int k = 0; k < kTile; k += kThreads) {
        const int64_t i = i0 + k + threadIdx.x;
        if (i >= p.N) break;
        const uint32_t key = p.tokens ? sort_key(p.tokens, p.wide, i, p.V, p.padding) : p.key_in[i];
        atomicAdd(&hist[(key >> p.shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kThreads) p.counts[count_at(p, b, blockIdx.x)] = hist[b];
}

// The sum of x over the threads before, and over all of them in `all`.  share [THREADS / 64].
template <int THREADS>
__device__ __forceinline__ uint32_t sum_before(uint32_t x, uint32_t* share, uint32_t* all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t in = x;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const uint32_t y = __shfl_up(in, o);
        if (lane >= o) in += y;
    }
    __syncthreads();
    if (lane == 63) share[wave] = in;
    __syncthreads();
    uint32_t before = in - x;
    *all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        before += w < wave ? share[w] : 0;
        *all += share[w];
    }
    return before;
}

// A digit's counts to the sums of the tiles' before, and its sum behind all counts (for more than
// kOwnScan tiles).
__global__ __launch_bounds__(kThreads) void sort_scan_kernel(uint32_t* counts, int tiles) {
    __shared__ uint32_t share[kThreads / 64];
    uint32_t* c = counts + (int64_t)blockIdx.x * tiles;
    uint32_t base = 0;
    for (int t0 = 0; t0 < tiles; t0 += kThreads) {
        const int t = t0 + threadIdx.x;
        uint32_t all;
        const uint32_t at = base + sum_before<kThreads>(t < tiles ? c[t] : 0, share, &all);
        if (t < tiles) c[t] = at;
        base += all;
    }
    if (threadIdx.x == 0) counts[(int64_t)gridDim.x * tiles + blockIdx.x] = base;
}

// The lanes of the wave with the same digit, of those `in`.
__device__ __forceinline__ uint64_t same_digit(uint32_t d, int bits, bool in) {
    uint64_t same = __ballot(in);
    for (int b = 0; b < bits; ++b) {
        const uint64_t set = __ballot((d >> b & 1) != 0);
        same &= (d >> b & 1) ? set : ~set;
    }
    return same;
}

// The place of a lane's key, from the next place of its digit in the wave's keys (in order).
__device__ __forceinline__ uint32_t take_place(uint32_t* next, uint32_t d, int bits, bool in, int lane) {
    const uint64_t same = same_digit(d, bits, in);
    uint32_t at = 0;
    if (in) at = next[d] + __popcll(same & (((uint64_t)1 << lane) - 1));
    wave_sync();
    // (the last of them moves the place on, after all have read it)
    if (in && (same >> lane) == 1) next[d] += __popcll(same);
    wave_sync();
    return at;
}

__global__ __launch_bounds__(kThreads) void sort_move_kernel(SortPass p) {
    constexpr int kWaves = kThreads / 64, kPer = kTile / kWaves;
    __shared__ uint32_t next[kWaves][kMaxBins];  // counts of the waves' parts, then their next places
    __shared__ uint32_t share[kWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, bins = 1 << p.bits;
    // (all loads first: none of them waits for another)
    const int64_t i0 = (int64_t)blockIdx.x * kTile + wave * kPer;
    uint32_t key[kPer / 64], from[kPer / 64];
#pragma unroll
    for (int k = 0; k < kPer / 64; ++k) {
        const int64_t i = min(i0 + k * 64 + lane, p.N - 1);
        key[k] = p.tokens ? sort_key(p.tokens, p.wide, i, p.V, p.padding) : p.key_in[i];
        from[k] = p.at_in ? p.at_in[i] : (uint32_t)i;
    }
    constexpr int kOwn = kMaxBins / kThreads;  // digits to a thread
    uint32_t before[kOwn] = {}, sum[kOwn] = {};
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        const int b = j * kThreads + threadIdx.x;
        if (b >= bins) break;
        if (p.tiles > kOwnScan) {
            before[j] = p.counts[count_at(p, b, blockIdx.x)];
            sum[j] = p.counts[(int64_t)bins * p.tiles + b];
        } else {  // summed here: a launch less than by sort_scan_kernel
#pragma unroll 16
            for (int t = 0; t < p.tiles; ++t) {
                const uint32_t c = p.counts[count_at(p, b, t)];
                before[j] += t < (int)blockIdx.x ? c : 0;
                sum[j] += c;
            }
        }
    }
    for (int b = lane; b < bins; b += 64) next[wave][b] = 0;
    wave_sync();
#pragma unroll
    for (int k = 0; k < kPer / 64; ++k)
        if (i0 + k * 64 + lane < p.N) atomicAdd(&next[wave][(key[k] >> p.shift) & (bins - 1)], 1u);
    __syncthreads();
    uint32_t base = 0;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        const int b = j * kThreads + threadIdx.x;
        if (j * kThreads >= bins) break;
        uint32_t all;
        uint32_t at = base + before[j] + sum_before<kThreads>(sum[j], share, &all);
        base += all;
        if (b < bins)
            for (int w = 0; w < kWaves; ++w) {
                const uint32_t c = next[w][b];
                next[w][b] = at;
                at += c;
            }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kPer / 64; ++k) {
        const bool in = i0 + k * 64 + lane < p.N;
        const uint32_t at = take_place(next[wave], (key[k] >> p.shift) & (bins - 1), p.bits, in, lane);
        if (in) {
            p.key_out[at] = key[k];
            p.at_out[at] = from[k];
        }
    }
}

// All passes over N <= kSmall tokens.
__global__ __launch_bounds__(kSmallThreads) void sort_small_kernel(SortPass p, int passes) {
    constexpr int kWaves = kSmallThreads / 64, kPer = kSmall / kWaves / 64, kBins = 512;
    __shared__ uint32_t keys[kSmall], places[kSmall];
    __shared__ uint32_t next[kWaves][kBins];
    __shared__ uint32_t share[kWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, bins = 1 << p.bits, N = (int)p.N;
    // a wave's keys are side by side, as many to each as the tokens give
    const int per = (N + kWaves * 64 - 1) / (kWaves * 64), i0 = wave * per * 64;
    uint32_t key[kPer], at[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const int i = i0 + k * 64 + lane;
        at[k] = i;
        key[k] = k < per && i < N ? sort_key(p.tokens, p.wide, i, p.V, p.padding) : 0;
    }
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * p.bits;
        for (int b = threadIdx.x; b < kWaves * kBins; b += kSmallThreads) (&next[0][0])[b] = 0;
        __syncthreads();
        // a key's place among the wave's of its digit; their counts are left in `next`
        uint32_t to[kPer];
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            if (k >= per) break;
            to[k] = take_place(next[wave], (key[k] >> shift) & (bins - 1), p.bits,
                               i0 + k * 64 + lane < N, lane);
        }
        __syncthreads();
        uint32_t sum = 0, all;
        const int b = threadIdx.x;
        if (b < bins)
            for (int w = 0; w < kWaves; ++w) sum += next[w][b];
        uint32_t first = sum_before<kSmallThreads>(sum, share, &all);
        if (b < bins)
            for (int w = 0; w < kWaves; ++w) {
                const uint32_t c = next[w][b];
                next[w][b] = first;
                first += c;
            }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            if (k >= per || i0 + k * 64 + lane >= N) break;
            const uint32_t place = next[wave][(key[k] >> shift) & (bins - 1)] + to[k];
            keys[place] = key[k];
            places[place] = at[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const int i = i0 + k * 64 + lane;
            if (k < per && i < N) {
                key[k] = keys[i];
                at[k] = places[i];
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const int i = i0 + k * 64 + lane;
        if (k < per && i < N) {
            p.key_out[i] = key[k];
            p.at_out[i] = at[k];
        }
    }
}

// first[v] = first sorted place whose key is at least v, for v = 0 .. V: by halving, first among 1024
// keys in LDS and then between two of them.
__global__ __launch_bounds__(kThreads) void emb_first_kernel(const uint32_t* key, int64_t N, int64_t V,
                                                             uint32_t* first) {
    constexpr int kSamples = 1024;
    __shared__ uint32_t sample[kSamples];
    const int64_t step = (N + kSamples - 1) / kSamples;
    const int n = step ? (int)((N + step - 1) / step) : 0;  // keys 0, step, 2 step, ...
    for (int k = threadIdx.x; k < n; k += kThreads) sample[k] = key[k * step];
    __syncthreads();
    const int64_t v = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (v > V) return;
    int a = 0, b = n;  // samples under v: [0, a)
    while (a < b) {
        const int mid = (a + b) / 2;
        if (sample[mid] < (uint32_t)v) a = mid + 1;
        else b = mid;
    }
    int64_t lo = a ? (a - 1) * step + 1 : 0, hi = min(N, a * step);
    while (lo < hi) {
        const int64_t mid = (lo + hi) / 2;
        if (key[mid] < (uint32_t)v) lo = mid + 1;
        else hi = mid;
    }
    first[v] = (uint32_t)lo;
}

// -------------------------------------------------------------- gradient ----
// A group of tpr threads sums rows of dy, C vectors of a row to a thread at a time.  A token met up to
// `light` times is summed by one group, one met up to `window` times by a workgroup's groups together.
// The sorted places of one met more often are cut where multiples of `window` lie; the parts are
// summed each by a workgroup, in the same launch, and joined in order by a second.  A window has parts
// of at most two such tokens: of the one at its first place (slot 0), and of another at its last
// (slot 1).
struct Gradient {
    const char* dy;
    int64_t lddy;
    const uint32_t *key, *at, *first;
    float* parts;
    char* dw;
    int64_t rows, D, window, windows;
    float scale;
    int tpr, light;
};

template <int DT, int V, int C>
struct Columns {
    static constexpr int kAhead = 4;
    float f[C][V];
    // column vectors c0, c0 + tpr, ... of a group's thread; the last of a row shares elements
    static __device__ __forceinline__ int64_t at(const Gradient& g, int64_t c0, int c) {
        return min((c0 + c * g.tpr) * V, g.D - V);
    }
    __device__ __forceinline__ void sum(const Gradient& g, int64_t c0, int64_t b, int64_t e) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int k = 0; k < V; ++k) f[c][k] = 0.f;
        // (rows whose loads do not wait for one another: four, or what is left)
        int64_t i = b;
        for (; i + kAhead <= e; i += kAhead) add<kAhead>(g, c0, i);
        if (kAhead > 2 && i + 2 <= e) {
            add<2>(g, c0, i);
            i += 2;
        }
        for (; i < e; ++i) add<1>(g, c0, i);
    }
    template <int n>
    __device__ __forceinline__ void add(const Gradient& g, int64_t c0, int64_t i) {
        typename std::conditional<V == 1, float, Elems<DT, V == 1 ? 4 : V>>::type x[n][C];
        uint32_t at_row[n];
#pragma unroll
        for (int j = 0; j < n; ++j) at_row[j] = g.at[i + j];
#pragma unroll
        for (int j = 0; j < n; ++j) {
            const char* row = g.dy + (int64_t)at_row[j] * g.lddy * kElemBytes<DT>;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                if constexpr (V == 1) x[j][c] = load_elem<DT>(row, at(g, c0, c));
                else x[j][c] = load<DT, V>(row, at(g, c0, c));
            }
        }
#pragma unroll
        for (int j = 0; j < n; ++j)
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float y[V];
                if constexpr (V == 1) y[0] = x[j][c];
                else unpack<DT, V>(x[j][c], y);
#pragma unroll
                for (int k = 0; k < V; ++k) f[c][k] += y[k];
            }
    }
    __device__ __forceinline__ void put(const Gradient& g, int64_t c0, int64_t v) const {
        char* row = g.dw + v * g.D * kElemBytes<DT>;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float x[V];
#pragma unroll
            for (int k = 0; k < V; ++k) x[k] = f[c][k] * g.scale;
            if ((c0 + c * g.tpr) * V >= g.D) continue;
            if constexpr (V == 1) store_elem<DT>(row, at(g, c0, c), x[0]);
            else store<DT, V>(row, at(g, c0, c), pack<DT, V>(x));
        }
    }
};

// Rows [b, e) of the sorted places summed by all groups, into the first group's s.  Every thread calls.
template <int DT, int V, int C>
__device__ __forceinline__ void sum_together(const Gradient& g, Columns<DT, V, C>& s, float* share,
                                             int64_t c0, int64_t b, int64_t e) {
    const int groups = kThreads / g.tpr, group = threadIdx.x / g.tpr;
    const int64_t n = e - b;
    s.sum(g, c0, b + n * group / groups, b + n * (group + 1) / groups);
    __syncthreads();
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int k = 0; k < V; ++k) share[(c * V + k) * kThreads + threadIdx.x] = s.f[c][k];
    __syncthreads();
    if (group == 0)
        for (int o = 1; o < groups; ++o)
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int k = 0; k < V; ++k) s.f[c][k] += share[(c * V + k) * kThreads + o * g.tpr + threadIdx.x];
}

// The first workgroups take the windows; the others rows of the table, `stride` apart (frequent
// tokens tend to lie side by side).
template <int DT, int V, int C>
__global__ __launch_bounds__(kThreads) void emb_grad_kernel(Gradient g, int windows, int64_t row0,
                                                            int64_t rows, int64_t stride) {
    __shared__ float share[C * V * kThreads];
    __shared__ int lengths[kThreads];
    const int groups = kThreads / g.tpr, group = threadIdx.x / g.tpr, lane = threadIdx.x % g.tpr;
    Columns<DT, V, C> s;
    if ((int)blockIdx.x >= windows) {
        const int64_t r = blockIdx.x - windows + group * stride, v = row0 + r;
        const bool mine = r < rows;
        const int64_t b = mine ? g.first[v] : 0, e = mine ? g.first[v + 1] : 0;
        if (mine && e - b <= g.light)
            for (int64_t c0 = lane; c0 * V < g.D; c0 += C * g.tpr) {
                s.sum(g, c0, b, e);
                s.put(g, c0, v);
            }
        if (lane == 0) lengths[group] = (int)(e - b);
        if (!__syncthreads_or(e - b > g.light)) return;
        for (int k = 0; k < groups; ++k) {
            if (lengths[k] <= g.light || lengths[k] > g.window) continue;
            const int64_t u = row0 + blockIdx.x - windows + k * stride, ub = g.first[u];
            for (int64_t i = 0; i * V < g.D; i += C * g.tpr) {
                sum_together(g, s, share, i + lane, ub, ub + lengths[k]);
                if (group == 0) s.put(g, i + lane, u);
            }
        }
        return;
    }
    const int64_t w = blockIdx.x;
    const int64_t live = g.first[g.rows], from = w * g.window, to = min(live, from + g.window);
    for (int slot = 0; slot < 2 && from < live; ++slot) {
        const int64_t v = g.key[slot ? to - 1 : from];
        const int64_t b0 = g.first[v], e0 = g.first[v + 1];
        if (e0 - b0 <= g.window || (slot && b0 <= from)) continue;
        for (int64_t i = 0; i * V < g.D; i += C * g.tpr) {
            sum_together(g, s, share, i + lane, max(b0, from), min(e0, to));
            float* p = g.parts + (2 * w + slot) * g.D;
            if (group == 0)
#pragma unroll
                for (int c = 0; c < C; ++c)
                    if ((i + lane + c * g.tpr) * V < g.D)
#pragma unroll
                        for (int k = 0; k < V; ++k) p[s.at(g, i + lane, c) + k] = s.f[c][k];
        }
    }
}

// A workgroup to a window: the token that starts in it, if it is one of those.
template <int DT, int V>
__global__ __launch_bounds__(kThreads) void emb_join_kernel(Gradient g) {
    __shared__ float share[kThreads * V];
    const int64_t w = blockIdx.x, live = g.first[g.rows], from = w * g.window, to = min(live, from + g.window);
    const int groups = kThreads / g.tpr, group = threadIdx.x / g.tpr, lane = threadIdx.x % g.tpr;
    for (int slot = 0; slot < 2 && from < live; ++slot) {
        const int64_t v = g.key[slot ? to - 1 : from];
        const int64_t b0 = g.first[v], e0 = g.first[v + 1];
        if (e0 - b0 <= g.window || (slot ? b0 <= from : b0 < from)) continue;
        const int64_t n = (e0 - 1) / g.window - w + 1;  // parts, cut evenly among the groups
        const int64_t x0 = n * group / groups, x1 = n * (group + 1) / groups;
        for (int64_t i0 = 0; i0 < g.D; i0 += g.tpr * V) {
            const int64_t i = i0 + (int64_t)lane * V;
            Columns<DT, V, 1> s{};
            const int64_t col = s.at(g, i / V, 0);
#pragma unroll 8
            for (int64_t x = x0; x < x1; ++x) {
                const float* p = g.parts + (2 * (w + x) + (x == 0 ? slot : 0)) * g.D + col;
#pragma unroll
                for (int k = 0; k < V; ++k) s.f[0][k] += p[k];
            }
#pragma unroll
            for (int k = 0; k < V; ++k) share[threadIdx.x * V + k] = s.f[0][k];
            __syncthreads();
            if (group == 0 && i < g.D) {
                for (int o = 1; o < groups; ++o)
#pragma unroll
                    for (int k = 0; k < V; ++k) s.f[0][k] += share[(o * g.tpr + threadIdx.x) * V + k];
                s.put(g, i / V, v);
            }
            __syncthreads();
        }
    }
}

// ------------------------------------------------------------------ host ----
// Places to a window: 1024 windows at most.
int64_t window_of(int64_t N) { return std::max<int64_t>(256, ceil_div(N, 1024)); }

struct Plan {
    int passes, bits;
    int64_t tiles, windows;
    int64_t key[2], at[2], counts, first, parts, bytes;  // places in the workspace
};
Plan plan(int64_t N, int64_t V, int64_t D) {
    Plan p;
    int bits = 1;
    while ((V >> bits) != 0) ++bits;
    const int most = N <= kSmall ? 9 : 10;
    p.passes = (bits + most - 1) / most;
    p.bits = (bits + p.passes - 1) / p.passes;
    p.tiles = ceil_div(N, kTile);
    p.windows = ceil_div(N, window_of(N));
    int64_t next = 0;
    auto take = [&](int64_t bytes) {
        const int64_t at = next;
        next += ceil_div(bytes, 256) * 256;
        return at;
    };
    for (int k = 0; k < 2; ++k) {
        p.key[k] = take(4 * N);
        p.at[k] = take(4 * N);
    }
    p.counts = take(4 * ((p.tiles + 1) << p.bits));
    p.first = take(4 * (V + 1));
    p.parts = take(8 * p.windows * D);
    p.bytes = next;
    return p;
}

int check_sizes(const char* fn, int64_t N, int64_t V, int64_t D, int32_t token_bits, int32_t dtype) {
    HASTE_CHECK_ARG(N >= 0 && V > 0 && D > 0, "%s: bad sizes N=%lld V=%lld D=%lld", fn, (long long)N,
                    (long long)V, (long long)D);
    HASTE_CHECK_ARG(N < (int64_t)1 << 31 && V < ((int64_t)1 << 31) - 1 && D < (int64_t)1 << 31,
                    "%s: too large", fn);
    HASTE_CHECK_ARG(token_bits == 32 || token_bits == 64, "%s: tokens have 32 or 64 bits", fn);
    HASTE_CHECK_ARG(elem_dtype(dtype), "%s: rows must be bf16, f16 or f32", fn);
    return HASTE_OK;
}
int check_tokens(const char* fn, const void* tokens, int32_t token_bits, int64_t N) {
    HASTE_CHECK_ARG(N == 0 || (tokens != nullptr &&
                               reinterpret_cast<uintptr_t>(tokens) % (token_bits / 8) == 0),
                    "%s: tokens are NULL or misaligned", fn);
    return HASTE_OK;
}
int check_rows(const char* fn, const char* what, const void* p, int64_t ld, int64_t D, int32_t dtype) {
    HASTE_CHECK_ARG(p != nullptr && elem_aligned(p, dtype), "%s: %s is NULL or misaligned", fn, what);
    HASTE_CHECK_ARG(ld == 0 || ld >= D, "%s: row pitch of %s is short (%lld < %lld)", fn, what,
                    (long long)ld, (long long)D);
    return HASTE_OK;
}

// `call` with DT and V: 16-byte vectors, or elements where a row is shorter than one.
#define HASTE_EMB_TYPES(call)                                                \
    do {                                                                     \
        const bool one = D < 16 / haste::elem_bytes(dtype);                  \
        if (dtype == HASTE_DTYPE_F32 && one) call(HASTE_DTYPE_F32, 1);       \
        else if (dtype == HASTE_DTYPE_F32) call(HASTE_DTYPE_F32, 4);         \
        else if (dtype == HASTE_DTYPE_BF16 && one) call(HASTE_DTYPE_BF16, 1); \
        else if (dtype == HASTE_DTYPE_BF16) call(HASTE_DTYPE_BF16, 8);       \
        else if (one) call(HASTE_DTYPE_F16, 1);                              \
        else call(HASTE_DTYPE_F16, 8);                                       \
    } while (0)

int threads_of(int64_t D, int32_t dtype) {
    const int64_t V = D < 16 / elem_bytes(dtype) ? 1 : 16 / elem_bytes(dtype);
    return row_threads(ceil_div(D, V));
}

// Threads to a row and vectors of it to a thread at a time: the pair that leaves the fewest idle, and
// among those the one with the fewest threads (more rows to a wave).
struct GroupShape {
    int tpr, columns;
};
GroupShape group_shape(int64_t D, int32_t dtype) {
    const int64_t V = D < 16 / elem_bytes(dtype) ? 1 : 16 / elem_bytes(dtype), n = ceil_div(D, V);
    GroupShape best{64, 1};
    int64_t least = INT64_MAX;
    for (int tpr = 1; tpr <= 64; tpr *= 2)
        for (int c = 1; c <= 3; ++c) {
            const int64_t taken = ceil_div(n, tpr * c) * tpr * c * (tpr * c < n && tpr < 64 ? 4 : 1);
            if (taken < least) {
                least = taken;
                best = GroupShape{tpr, c};
            }
        }
    return best;
}

// f(first, count) over launches of `count` groups of tpr threads, fewer than 2^32 threads each.
template <typename F>
void in_launches(int64_t count, int tpr, F f) {
    const int64_t most = (((int64_t)1 << 31) / tpr);
    for (int64_t i = 0; i < count; i += most) f(i, std::min(most, count - i));
}

}  // namespace
}  // namespace haste

extern "C" int haste_embedding(const void* tokens, int32_t token_bits, const void* w, int64_t ldw,
                               void* y, int64_t N, int64_t V, int64_t D, double scale, int32_t dtype,
                               void* stream) {
    const char* fn = "haste_embedding";
    HASTE_TRY(haste::check_sizes(fn, N, V, D, token_bits, dtype));
    if (N == 0) return HASTE_OK;
    HASTE_TRY(haste::check_tokens(fn, tokens, token_bits, N));
    HASTE_TRY(haste::check_rows(fn, "the table", w, ldw, D, dtype));
    HASTE_TRY(haste::check_rows(fn, "y", y, D, D, dtype));
    const int tpr = haste::threads_of(D, dtype);
    const int64_t size = haste::elem_bytes(dtype);
    hipStream_t st = static_cast<hipStream_t>(stream);
    haste::in_launches(N, tpr, [&](int64_t n0, int64_t n) {
#define HASTE_EMB(DT, VEC)                                                                         \
    haste::emb_kernel<DT, VEC>                                                                     \
        <<<dim3((unsigned)haste::ceil_div(n, haste::kThreads / tpr)), dim3(haste::kThreads), 0, st>>>( \
            static_cast<const char*>(tokens) + n0 * (token_bits / 8), token_bits == 64,           \
            static_cast<const char*>(w), ldw, static_cast<char*>(y) + n0 * D * size, n, V, D,     \
            (float)scale, tpr)
        HASTE_EMB_TYPES(HASTE_EMB);
#undef HASTE_EMB
    });
    HASTE_CHECK_LAUNCH(fn);
    return HASTE_OK;
}

extern "C" int64_t haste_embedding_bwd_workspace_size(int64_t N, int64_t V, int64_t D) {
    if (N < 0 || V <= 0 || D <= 0 || N >= (int64_t)1 << 31 || V >= ((int64_t)1 << 31) - 1 ||
        D >= (int64_t)1 << 31)
        return HASTE_ERR_INVALID_ARG;
    return haste::plan(N, V, D).bytes;
}

extern "C" int haste_embedding_bwd(const void* tokens, int32_t token_bits, const void* dy,
                                   int64_t lddy, void* dw, int64_t N, int64_t V, int64_t D,
                                   double scale, int64_t padding, int32_t dtype, void* ws,
                                   int64_t ws_bytes, void* stream) {
    const char* fn = "haste_embedding_bwd";
    HASTE_TRY(haste::check_sizes(fn, N, V, D, token_bits, dtype));
    HASTE_TRY(haste::check_tokens(fn, tokens, token_bits, N));
    if (N > 0) HASTE_TRY(haste::check_rows(fn, "dy", dy, lddy, D, dtype));
    HASTE_TRY(haste::check_rows(fn, "dw", dw, D, D, dtype));
    const haste::Plan p = haste::plan(N, V, D);
    HASTE_CHECK_ARG(ws != nullptr && haste::aligned16(ws), "%s: workspace is NULL or misaligned", fn);
    if (ws_bytes < p.bytes) {
        haste::set_error("%s: workspace too small (%lld < %lld bytes)", fn, (long long)ws_bytes,
                         (long long)p.bytes);
        return HASTE_ERR_WORKSPACE;
    }
    char* base = static_cast<char*>(ws);
    auto words = [&](int64_t at) { return reinterpret_cast<uint32_t*>(base + at); };
    hipStream_t st = static_cast<hipStream_t>(stream);
    uint32_t *key = words(p.key[0]), *at = words(p.at[0]), *first = words(p.first);
    haste::SortPass s{};
    s.tokens = tokens;
    s.wide = token_bits == 64;
    s.V = V;
    s.padding = padding;
    s.N = N;
    s.bits = p.bits;
    if (N > 0 && N <= haste::kSmall) {
        s.key_out = key;
        s.at_out = at;
        haste::sort_small_kernel<<<dim3(1), dim3(haste::kSmallThreads), 0, st>>>(s, p.passes);
    }
    for (int k = 0; k < p.passes && N > haste::kSmall; ++k) {
        s.tokens = k ? nullptr : tokens;
        s.key_in = key;
        s.at_in = k ? at : nullptr;
        key = s.key_out = words(p.key[(k + 1) % 2]);
        at = s.at_out = words(p.at[(k + 1) % 2]);
        s.counts = words(p.counts);
        s.tiles = (int)p.tiles;
        s.shift = k * p.bits;
        const dim3 grid((unsigned)p.tiles), block(haste::kThreads);
        haste::sort_count_kernel<<<grid, block, 0, st>>>(s);
        if (p.tiles > haste::kOwnScan)
            haste::sort_scan_kernel<<<dim3(1u << p.bits), block, 0, st>>>(s.counts, s.tiles);
        haste::sort_move_kernel<<<grid, block, 0, st>>>(s);
    }
    haste::emb_first_kernel<<<dim3((unsigned)haste::ceil_div(V + 1, haste::kThreads)),
                              dim3(haste::kThreads), 0, st>>>(key, N, V, first);
    const haste::GroupShape shape = haste::group_shape(D, dtype);
    const int per = haste::kThreads / shape.tpr;
    const haste::Gradient g{static_cast<const char*>(dy), lddy, key, at, first,
                            reinterpret_cast<float*>(base + p.parts), static_cast<char*>(dw), V, D,
                            haste::window_of(N), p.windows, (float)scale, shape.tpr,
                            std::min(16 * 64 / shape.tpr, 128)};  // (narrow rows: many groups)
    // (a single window holds no token more often than it is long)
    const int windows = p.windows > 1 ? (int)p.windows : 0;
#define HASTE_EMB(DT, VEC)                                                                           \
    do {                                                                                             \
        auto kernel = shape.columns == 1   ? haste::emb_grad_kernel<DT, VEC, 1>                      \
                      : shape.columns == 2 ? haste::emb_grad_kernel<DT, VEC, 2>                      \
                                           : haste::emb_grad_kernel<DT, VEC, 3>;                     \
        haste::in_launches(V, shape.tpr, [&](int64_t v0, int64_t n) {                                \
            const int first_windows = v0 == 0 ? windows : 0;                                         \
            const int64_t stride = haste::ceil_div(n, per);                                          \
            kernel<<<dim3((unsigned)(first_windows + stride)), dim3(haste::kThreads), 0, st>>>(      \
                g, first_windows, v0, n, stride);                                                    \
        });                                                                                          \
        if (windows)                                                                                 \
            haste::emb_join_kernel<DT, VEC>                                                          \
                <<<dim3((unsigned)p.windows), dim3(haste::kThreads), 0, st>>>(g);                    \
    } while (0)
    HASTE_EMB_TYPES(HASTE_EMB);
#undef HASTE_EMB
    HASTE_CHECK_LAUNCH(fn);
    return HASTE_OK;
}
