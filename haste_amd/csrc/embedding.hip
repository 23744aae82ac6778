// Embedding lookup with scaling, y[n] = s W[t_n], and the table's gradient by sorted tokens,
// dW[v] = s sum_{n: t_n = v} dy[n], summed in fp32 in the order of n (no float atomics).
// Both are bound by HBM; the gradient's table is written once, rows without a token among it.
#include <algorithm>

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
// counts each tile's digits, turns the counts into first places (bins in order, tiles in order
// within a bin), and moves.  Tokens that take no gradient are keyed V, behind all others.
constexpr int kTile = 2048, kMaxBins = 1024;

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
    uint32_t* counts;              // [bins][tiles]
    int64_t N;
    int tiles, shift, bins;
};

__global__ __launch_bounds__(kThreads) void sort_count_kernel(SortPass p) {
    __shared__ uint32_t hist[kMaxBins];
    for (int b = threadIdx.x; b < p.bins; b += kThreads) hist[b] = 0;
    __syncthreads();
    const int64_t i0 = (int64_t)blockIdx.x * kTile;
    for (int k = threadIdx.x; k < kTile && i0 + k < p.N; k += kThreads) {
        const uint32_t key =
            p.tokens ? sort_key(p.tokens, p.wide, i0 + k, p.V, p.padding) : p.key_in[i0 + k];
        atomicAdd(&hist[(key >> p.shift) & (p.bins - 1)], 1u);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < p.bins; b += kThreads)
        p.counts[(int64_t)b * p.tiles + blockIdx.x] = hist[b];
}

// counts [n] to the sums of those before, one workgroup.
__global__ __launch_bounds__(1024) void sort_scan_kernel(uint32_t* counts, int64_t n) {
    __shared__ uint32_t wave_sum[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t base = 0;
    for (int64_t i0 = 0; i0 < n; i0 += 4096) {
        const int64_t i = i0 + threadIdx.x * 4;
        uint32_t c[4], s = 0;
        for (int k = 0; k < 4; ++k) {
            c[k] = i + k < n ? counts[i + k] : 0;
            s += c[k];
        }
        uint32_t in = s;
        for (int o = 1; o < 64; o *= 2) {
            const uint32_t x = __shfl_up(in, o);
            if (lane >= o) in += x;
        }
        if (lane == 63) wave_sum[wave] = in;
        __syncthreads();
        uint32_t before = base, all = 0;
        for (int w = 0; w < 16; ++w) {
            before += w < wave ? wave_sum[w] : 0;
            all += wave_sum[w];
        }
        uint32_t at = before + in - s;
        for (int k = 0; k < 4; ++k) {
            if (i + k < n) counts[i + k] = at;
            at += c[k];
        }
        base += all;
        __syncthreads();
    }
}

__global__ __launch_bounds__(kThreads) void sort_move_kernel(SortPass p) {
    constexpr int kWaves = kThreads / 64, kPer = kTile / kWaves;
    __shared__ uint32_t next[kWaves][kMaxBins];  // counts of the waves' parts, then their next places
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int b = threadIdx.x; b < kWaves * kMaxBins; b += kThreads) (&next[0][0])[b] = 0;
    __syncthreads();
    const int64_t i0 = (int64_t)blockIdx.x * kTile + wave * kPer;
    uint32_t key[kPer / 64];
#pragma unroll
    for (int k = 0; k < kPer / 64; ++k) {
        const int64_t i = i0 + k * 64 + lane;
        key[k] = 0;
        if (i < p.N) {
            key[k] = p.tokens ? sort_key(p.tokens, p.wide, i, p.V, p.padding) : p.key_in[i];
            atomicAdd(&next[wave][(key[k] >> p.shift) & (p.bins - 1)], 1u);
        }
    }
    __syncthreads();
    for (int b = threadIdx.x; b < p.bins; b += kThreads) {
        uint32_t at = p.counts[(int64_t)b * p.tiles + blockIdx.x];
        for (int w = 0; w < kWaves; ++w) {
            const uint32_t c = next[w][b];
            next[w][b] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kPer / 64; ++k) {
        const int64_t i = i0 + k * 64 + lane;
        const bool in = i < p.N;
        const uint32_t d = (key[k] >> p.shift) & (p.bins - 1);
        // the wave's lanes with the same digit
        uint64_t same = __ballot(in);
        for (int b = 1; b < p.bins; b *= 2) {
            const uint64_t set = __ballot((d & b) != 0);
            same &= (d & b) ? set : ~set;
        }
        if (in) {
            const uint32_t rank = __popcll(same & (((uint64_t)1 << lane) - 1));
            const uint32_t at = next[wave][d] + rank;
            p.key_out[at] = key[k];
            p.at_out[at] = p.at_in ? p.at_in[i] : (uint32_t)i;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        // (the last of them moves the place on, after all have read it)
        if (in && (same >> lane) == 1) next[wave][d] += __popcll(same);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// first[v] = first sorted place whose key is at least v, for v = 0 .. V.
__global__ __launch_bounds__(kThreads) void emb_first_kernel(const uint32_t* key, int64_t N, int64_t V,
                                                             uint32_t* first) {
    const int64_t v = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (v > V) return;
    int64_t lo = 0, hi = N;
    while (lo < hi) {
        const int64_t mid = (lo + hi) / 2;
        if (key[mid] < (uint32_t)v) lo = mid + 1;
        else hi = mid;
    }
    first[v] = (uint32_t)lo;
}

// -------------------------------------------------------------- gradient ----
// A token met at most `window` times is summed by one group of threads.  The sorted places of one met
// more often are cut where multiples of `window` lie; the parts are summed each for itself and
// joined in order by a second launch.  A window has parts of at most two such tokens: of the one at
// its first place (slot 0), and of another at its last (slot 1).
template <int DT, int V>
__device__ __forceinline__ void add_rows(const char* dy, int64_t lddy, const uint32_t* at, int64_t b,
                                         int64_t e, int64_t col, float* sum) {
#pragma unroll 8
    for (int64_t i = b; i < e; ++i) {
        float f[V];
        const char* row = dy + (int64_t)at[i] * lddy * kElemBytes<DT>;
        if constexpr (V == 1) f[0] = load_elem<DT>(row, col);
        else unpack<DT, V>(load<DT, V>(row, col), f);
#pragma unroll
        for (int k = 0; k < V; ++k) sum[k] += f[k];
    }
}
template <int DT, int V>
__device__ __forceinline__ void put_row(char* dw, int64_t v, int64_t D, int64_t col, float* f,
                                        float scale) {
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] *= scale;
    char* row = dw + v * D * kElemBytes<DT>;
    if constexpr (V == 1) store_elem<DT>(row, col, f[0]);
    else store<DT, V>(row, col, pack<DT, V>(f));
}

template <int DT, int V>
__global__ __launch_bounds__(kThreads) void emb_grad_kernel(const char* dy, int64_t lddy,
                                                            const uint32_t* at, const uint32_t* first,
                                                            char* dw, int64_t rows, int64_t D,
                                                            int64_t window, float scale, int tpr) {
    const int64_t v = (int64_t)blockIdx.x * (kThreads / tpr) + threadIdx.x / tpr;
    if (v >= rows) return;
    const int64_t b = first[v], e = first[v + 1];
    if (e - b > window) return;
    for (int64_t i = (int64_t)(threadIdx.x % tpr) * V; i < D; i += tpr * V) {
        const int64_t col = min(i, D - V);
        float sum[V] = {};
        add_rows<DT, V>(dy, lddy, at, b, e, col, sum);
        put_row<DT, V>(dw, v, D, col, sum, scale);
    }
}

template <int DT, int V>
__global__ __launch_bounds__(kThreads) void emb_windows_kernel(const char* dy, int64_t lddy,
                                                               const uint32_t* key, const uint32_t* at,
                                                               const uint32_t* first, float* parts,
                                                               int64_t rows, int64_t D, int64_t window,
                                                               int tpr) {
    const int64_t w = (int64_t)blockIdx.x * (kThreads / tpr) + threadIdx.x / tpr;
    const int64_t live = first[rows], from = w * window, to = min(live, from + window);
    for (int slot = 0; slot < 2 && from < live; ++slot) {
        const int64_t v = key[slot ? to - 1 : from];
        const int64_t b0 = first[v], e0 = first[v + 1];
        if (e0 - b0 <= window || (slot && b0 <= from)) continue;
        for (int64_t i = (int64_t)(threadIdx.x % tpr) * V; i < D; i += tpr * V) {
            const int64_t col = min(i, D - V);
            float sum[V] = {};
            add_rows<DT, V>(dy, lddy, at, max(b0, from), min(e0, to), col, sum);
            float* p = parts + (2 * w + slot) * D + col;
#pragma unroll
            for (int k = 0; k < V; ++k) p[k] = sum[k];
        }
    }
}

// A workgroup to a window: the token that starts in it, if it is one of those.
constexpr int kJoinThreads = 1024;
template <int DT, int V>
__global__ __launch_bounds__(kJoinThreads) void emb_join_kernel(const float* parts,
                                                                const uint32_t* key,
                                                                const uint32_t* first, char* dw,
                                                                int64_t rows, int64_t D,
                                                                int64_t window, float scale, int tpr) {
    __shared__ float share[kJoinThreads * V];
    const int64_t w = blockIdx.x;
    const int64_t live = first[rows], from = w * window, to = min(live, from + window);
    const int groups = kJoinThreads / tpr, group = threadIdx.x / tpr;
    for (int slot = 0; slot < 2 && from < live; ++slot) {
        const int64_t v = key[slot ? to - 1 : from];
        const int64_t b0 = first[v], e0 = first[v + 1];
        if (e0 - b0 <= window || (slot ? b0 <= from : b0 < from)) continue;
        const int64_t n = (e0 - 1) / window - w + 1;  // parts, cut evenly among the groups
        const int64_t x0 = n * group / groups, x1 = n * (group + 1) / groups;
        for (int64_t i0 = 0; i0 < D; i0 += tpr * V) {
            const int64_t i = i0 + (int64_t)(threadIdx.x % tpr) * V, col = min(i, D - V);
            float sum[V] = {};
#pragma unroll 4
            for (int64_t x = x0; x < x1; ++x) {
                const float* p = parts + (2 * (w + x) + (x == 0 ? slot : 0)) * D + col;
#pragma unroll
                for (int k = 0; k < V; ++k) sum[k] += p[k];
            }
#pragma unroll
            for (int k = 0; k < V; ++k) share[threadIdx.x * V + k] = sum[k];
            __syncthreads();
            if (group == 0 && i < D) {
                for (int g = 1; g < groups; ++g)
#pragma unroll
                    for (int k = 0; k < V; ++k) sum[k] += share[(g * tpr + threadIdx.x) * V + k];
                put_row<DT, V>(dw, v, D, col, sum, scale);
            }
            __syncthreads();
        }
    }
}

// ------------------------------------------------------------------ host ----
// Places to a window: 2048 windows at most.
int64_t window_of(int64_t N) { return std::max<int64_t>(64, ceil_div(N, 2048)); }

struct Plan {
    int passes, bits;
    int64_t tiles, windows;
    int64_t key[2], at[2], counts, first, parts, bytes;  // places in the workspace
};
Plan plan(int64_t N, int64_t V, int64_t D) {
    Plan p;
    int bits = 1;
    while ((V >> bits) != 0) ++bits;
    p.passes = (bits + 9) / 10;
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
    p.counts = take(4 * (p.tiles << p.bits));
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

#define HASTE_TRY(expr)                  \
    do {                                 \
        const int rc_ = (expr);          \
        if (rc_ != HASTE_OK) return rc_; \
    } while (0)

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
    for (int k = 0; k < p.passes && N > 0; ++k) {
        haste::SortPass s{};
        if (k == 0) s.tokens = tokens;
        s.wide = token_bits == 64;
        s.V = V;
        s.padding = padding;
        s.key_in = key;
        s.at_in = k ? at : nullptr;
        key = s.key_out = words(p.key[(k + 1) % 2]);
        at = s.at_out = words(p.at[(k + 1) % 2]);
        s.counts = words(p.counts);
        s.N = N;
        s.tiles = (int)p.tiles;
        s.shift = k * p.bits;
        s.bins = 1 << p.bits;
        const dim3 grid((unsigned)p.tiles), block(haste::kThreads);
        haste::sort_count_kernel<<<grid, block, 0, st>>>(s);
        haste::sort_scan_kernel<<<dim3(1), dim3(1024), 0, st>>>(s.counts, p.tiles << p.bits);
        haste::sort_move_kernel<<<grid, block, 0, st>>>(s);
    }
    haste::emb_first_kernel<<<dim3((unsigned)haste::ceil_div(V + 1, haste::kThreads)),
                              dim3(haste::kThreads), 0, st>>>(key, N, V, first);
    const int tpr = haste::threads_of(D, dtype), per = haste::kThreads / tpr;
    const int64_t window = haste::window_of(N);
    float* parts = reinterpret_cast<float*>(base + p.parts);
    const char* dyc = static_cast<const char*>(dy);
    char* dwc = static_cast<char*>(dw);
    const int64_t size = haste::elem_bytes(dtype);
#define HASTE_EMB(DT, VEC)                                                                           \
    do {                                                                                             \
        haste::in_launches(V, tpr, [&](int64_t v0, int64_t n) {                                      \
            haste::emb_grad_kernel<DT, VEC><<<dim3((unsigned)haste::ceil_div(n, per)),               \
                                              dim3(haste::kThreads), 0, st>>>(                       \
                dyc, lddy, at, first + v0, dwc + v0 * D * size, n, D, window, (float)scale, tpr);    \
        });                                                                                          \
        if (p.windows > 1) {                                                                         \
            haste::emb_windows_kernel<DT, VEC><<<dim3((unsigned)haste::ceil_div(p.windows, per)),    \
                                                 dim3(haste::kThreads), 0, st>>>(                    \
                dyc, lddy, key, at, first, parts, V, D, window, tpr);                                \
            haste::emb_join_kernel<DT, VEC><<<dim3((unsigned)p.windows), dim3(haste::kJoinThreads),  \
                                              0, st>>>(parts, key, first, dwc, V, D, window,         \
                                                       (float)scale, tpr);                           \
        }                                                                                            \
    } while (0)
    HASTE_EMB_TYPES(HASTE_EMB);
#undef HASTE_EMB
    HASTE_CHECK_LAUNCH(fn);
    return HASTE_OK;
}
