// Layer norm over rows, forward and backward: with n = (h - mean) / sqrt(var + eps), y = n w + b and
//   dx = (a - mean(a) - n mean(a n)) / sqrt(var + eps) + dh,  a = dy w;   dw = sum dy n, db = sum dy.
// Bound by HBM (8 and 14 operations an element): rows stay in registers between their passes, and the
// backward makes one pass for dx, dw and db.  2^26 bf16 elements in rows of 768: forward 42 us, 6.4
// TB/s, backward 78 us, 5.1 TB/s (a copy reaches 4.8-5.4); rows of 512 5.7, of 8192 4.5.
#include <algorithm>
#include <type_traits>

#include "elements.hpp"

namespace haste {
namespace {

constexpr int kRowThreads = 256;

// The sum of v over the workgroup, in every thread.  `part` [kRowThreads / 64] is free again
// after the next barrier.
__device__ __forceinline__ float group_sum(float v, float* part) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
    for (int k = 0; k < kRowThreads / 64; ++k) v += part[k];
    return v;
}

// Rows are met V elements (16 bytes) at a time.  Where V does not divide D, the thread of the last
// ones takes the row's last V elements instead, of which it shares the first `skip` with another
// thread (which computes the same values) and leaves them out of sums; with skip >= V it has none
// of its own.
constexpr int row_vec(int32_t dtype) { return dtype == HASTE_DTYPE_F32 ? 4 : 8; }
struct Slot {
    int64_t at;  // first element
    int skip;
};
template <int V>
__device__ __forceinline__ Slot last_slot(int64_t e, int64_t D) {
    const int64_t at = min(e, D - V);
    return Slot{at, (int)(e - at)};
}

// ---------------------------------------------------------------- any width ----
// For rows shorter than a slot (V = 1) or past what registers hold: a workgroup to a row, which
// is read again from cache for each of its passes.
template <int DT, int V>
__device__ __forceinline__ void get(const void* p, int64_t i, float* f) {
    if constexpr (V == 1) f[0] = load_elem<DT>(p, i);
    else unpack<DT, V>(load<DT, V>(p, i), f);
}
template <int DT, int V>
__device__ __forceinline__ void put(void* p, int64_t i, const float* f) {
    if constexpr (V == 1) store_elem<DT>(p, i, f[0]);
    else store<DT, V>(p, i, pack<DT, V>(f));
}

template <int DT, int WT, int V>
__global__ __launch_bounds__(kRowThreads) void ln_fwd_any_kernel(
    const char* x, int64_t ldx, const char* res, int64_t ldres, const void* w, const void* b,
    char* y, char* h, float* stats, int64_t D, float eps) {
    __shared__ float part[kRowThreads / 64];
    constexpr int S = kElemBytes<DT>;
    const int64_t row = blockIdx.x;
    x += row * ldx * S;
    y += row * D * S;
    if (res) {
        res += row * ldres * S;
        h += row * D * S;
    }
    auto rows = [&](int64_t at, float* f) __attribute__((always_inline)) {
        get<DT, V>(x, at, f);
        if (!res) return;
        float g[V];
        get<DT, V>(res, at, g);
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = round_elem<DT>(f[e] + g[e]);
    };
    float s = 0.f, f[V], g[V];
    for (int64_t i = threadIdx.x * V; i < D; i += kRowThreads * V) {
        const Slot t = last_slot<V>(i, D);
        rows(t.at, f);
#pragma unroll
        for (int e = 0; e < V; ++e) s += e >= t.skip ? f[e] : 0.f;
    }
    const float mean = group_sum(s, part) / (float)D;
    s = 0.f;
    for (int64_t i = threadIdx.x * V; i < D; i += kRowThreads * V) {
        const Slot t = last_slot<V>(i, D);
        rows(t.at, f);
#pragma unroll
        for (int e = 0; e < V; ++e) s += e >= t.skip ? (f[e] - mean) * (f[e] - mean) : 0.f;
    }
    const float rstd = 1.f / sqrtf(group_sum(s, part) / (float)D + eps);
    for (int64_t i = threadIdx.x * V; i < D; i += kRowThreads * V) {
        const int64_t at = last_slot<V>(i, D).at;
        rows(at, f);
        if (res) put<DT, V>(h, at, f);
        get<WT, V>(w, at, g);
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = (f[e] - mean) * rstd * g[e];
        if (b) {
            get<WT, V>(b, at, g);
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] += g[e];
        }
        put<DT, V>(y, at, f);
    }
    if (stats && threadIdx.x == 0) {
        stats[2 * row] = mean;
        stats[2 * row + 1] = rstd;
    }
}

template <int DT, int WT, int V>
__global__ __launch_bounds__(kRowThreads) void ln_dx_any_kernel(
    const char* dy, int64_t lddy, const char* dh, int64_t lddh, const char* h, int64_t ldh,
    const void* w, const float* stats, char* dx, int64_t D) {
    __shared__ float part[kRowThreads / 64];
    constexpr int S = kElemBytes<DT>;
    const int64_t row = blockIdx.x;
    dy += row * lddy * S;
    h += row * ldh * S;
    dx += row * D * S;
    if (dh) dh += row * lddh * S;
    const float mean = stats[2 * row], rstd = stats[2 * row + 1];
    float s1 = 0.f, s2 = 0.f, a[V], n[V], g[V];
    auto rows = [&](int64_t at) __attribute__((always_inline)) {
        get<DT, V>(dy, at, a);
        get<DT, V>(h, at, n);
        get<WT, V>(w, at, g);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            a[e] *= g[e];
            n[e] = (n[e] - mean) * rstd;
        }
    };
    for (int64_t i = threadIdx.x * V; i < D; i += kRowThreads * V) {
        const Slot t = last_slot<V>(i, D);
        rows(t.at);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            s1 += e >= t.skip ? a[e] : 0.f;
            s2 += e >= t.skip ? a[e] * n[e] : 0.f;
        }
    }
    const float c1 = group_sum(s1, part) / (float)D, c2 = group_sum(s2, part) / (float)D;
    for (int64_t i = threadIdx.x * V; i < D; i += kRowThreads * V) {
        const int64_t at = last_slot<V>(i, D).at;
        rows(at);
#pragma unroll
        for (int e = 0; e < V; ++e) a[e] = rstd * (a[e] - c1 - n[e] * c2);
        if (dh) {
            get<DT, V>(dh, at, g);
#pragma unroll
            for (int e = 0; e < V; ++e) a[e] += g[e];
        }
        put<DT, V>(dx, at, a);
    }
}

// sums[blockIdx.y] = dw and db of every gridDim.y-th 16 rows: 16 V columns to a workgroup, from
// column c0 on.
constexpr int kAnyRows = 16;
template <int DT, int V>
__global__ __launch_bounds__(kRowThreads) void ln_dw_any_kernel(const char* dy, int64_t lddy,
                                                                const char* h, int64_t ldh,
                                                                const float* stats, float* sums,
                                                                int64_t N, int64_t D, int64_t c0) {
    __shared__ float part[2 * V][kRowThreads];
    constexpr int S = kElemBytes<DT>;
    const int x = threadIdx.x & 15, y = threadIdx.x >> 4;
    const int64_t i = c0 + ((int64_t)blockIdx.x * 16 + x) * V;
    const Slot t = last_slot<V>(i, D);
    float sw[V] = {}, sb[V] = {}, a[V], n[V];
    if (i < D)
        for (int64_t r = (int64_t)blockIdx.y * kAnyRows + y; r < N; r += gridDim.y * kAnyRows) {
            get<DT, V>(dy + r * lddy * S, t.at, a);
            get<DT, V>(h + r * ldh * S, t.at, n);
            const float mean = stats[2 * r], rstd = stats[2 * r + 1];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                sw[e] += a[e] * ((n[e] - mean) * rstd);
                sb[e] += a[e];
            }
        }
#pragma unroll
    for (int e = 0; e < V; ++e) {
        part[e][threadIdx.x] = sw[e];
        part[V + e][threadIdx.x] = sb[e];
    }
    __syncthreads();
    if (y || i >= D) return;
    sums += (int64_t)blockIdx.y * 2 * D;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        if (e < t.skip) continue;
        for (int k = 1; k < kRowThreads / 16; ++k) {
            sw[e] += part[e][k * 16 + x];
            sb[e] += part[V + e][k * 16 + x];
        }
        sums[t.at + e] = sw[e];
        sums[D + t.at + e] = sb[e];
    }
}

// ------------------------------------------------------- rows in registers ----
// `tpr` threads (a power of two) hold a row in C slots: thread t has elements
// V (c tpr + t) + 0..V-1 of it in slot c.  Only the last slot can pass the row's end.
template <int V>
__device__ __forceinline__ Slot row_slot(int c, int C, int tpr, int lane, int64_t D) {
    const int64_t e = V * ((int64_t)c * tpr + lane);
    return c < C - 1 ? Slot{e, 0} : last_slot<V>(e, D);
}

template <int C>
__device__ __forceinline__ float dpp_add(float x) {
    return x + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), C, 0xF, 0xF, true));
}
// The sum over groups of min(tpr, 64) lanes, in all of them: neighbours, pairs, quads mirrored
// within 8 and 16 lanes, then rows and halves of the wave swapped.
__device__ __forceinline__ float lanes_sum(float x, int tpr) {
    if (tpr >= 2) x = dpp_add<0xB1>(x);
    if (tpr >= 4) x = dpp_add<0x4E>(x);
    if (tpr >= 8) x = dpp_add<0x141>(x);
    if (tpr >= 16) x = dpp_add<0x140>(x);
    if (tpr >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x),
                                                        false, false);
        x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if (tpr >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x),
                                                        false, false);
        x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return x;
}

// Sums of a and b over the row's threads, in all of them.  Rows of several waves meet in
// part[2][2 * 16], whose halves take turns (`turn`): one barrier a sum.
__device__ __forceinline__ void row_sums(float& a, float& b, int tpr, float (*part)[32], int& turn) {
    a = lanes_sum(a, tpr);
    b = lanes_sum(b, tpr);
    if (tpr <= 64) return;
    const int wave = threadIdx.x >> 6, waves = tpr >> 6;
    float* p = part[turn];
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) {
        p[wave] = a;
        p[16 + wave] = b;
    }
    __syncthreads();
    const int first = wave & ~(waves - 1);
    a = b = 0.f;
    for (int k = 0; k < waves; ++k) {
        a += p[first + k];
        b += p[16 + first + k];
    }
}

// NT: rows past the last-level cache are read and written non-temporally, all but h, which the
// backward reads.  (y and dx that fit it stay there for whoever reads them next.)
template <int DT, int WT, int C, bool NT>
__global__ __launch_bounds__(1024) void ln_fwd_kernel(
    const char* __restrict__ x, int64_t ldx, const char* __restrict__ res, int64_t ldres,
    const void* __restrict__ w, const void* __restrict__ b, char* __restrict__ y,
    char* __restrict__ h, float* __restrict__ stats, int64_t N, int64_t D, float eps, int tpr) {
    __shared__ float part[2][32];
    constexpr int S = kElemBytes<DT>, V = row_vec(DT);
    const int lane = threadIdx.x & (tpr - 1), group = threadIdx.x / tpr;
    const int64_t want = (int64_t)blockIdx.x * (blockDim.x / tpr) + group;
    const int64_t row = min(want, N - 1);
    const bool live = want < N;
    int turn = 0;
    x += row * ldx * S;
    if (res) res += row * ldres * S;
    Elems<DT, V> raw[C], add[C];
#pragma unroll
    for (int c = 0; c < C; ++c) raw[c] = load<DT, V, NT>(x, row_slot<V>(c, C, tpr, lane, D).at);
    if (res) {
#pragma unroll
        for (int c = 0; c < C; ++c) add[c] = load<DT, V, NT>(res, row_slot<V>(c, C, tpr, lane, D).at);
    }
    float f[C][V], s = 0.f, none = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const Slot at = row_slot<V>(c, C, tpr, lane, D);
        unpack<DT, V>(raw[c], f[c]);
        if (res) {
            float g[V];
            unpack<DT, V>(add[c], g);
#pragma unroll
            for (int e = 0; e < V; ++e) f[c][e] += g[e];
            const Elems<DT, V> sum = pack<DT, V>(f[c]);
            if (live && at.skip < V) store<DT, V>(h + row * D * S, at.at, sum);
            unpack<DT, V>(sum, f[c]);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) s += c < C - 1 || e >= at.skip ? f[c][e] : 0.f;
    }
    row_sums(s, none, tpr, part, turn);
    const float mean = s / (float)D;
    s = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int skip = row_slot<V>(c, C, tpr, lane, D).skip;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            f[c][e] -= mean;
            s += c < C - 1 || e >= skip ? f[c][e] * f[c][e] : 0.f;
        }
    }
    row_sums(s, none, tpr, part, turn);
    const float rstd = 1.f / sqrtf(s / (float)D + eps);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const Slot at = row_slot<V>(c, C, tpr, lane, D);
        float g[V];
        unpack<WT, V>(load<WT, V>(w, at.at), g);
#pragma unroll
        for (int e = 0; e < V; ++e) f[c][e] = f[c][e] * rstd * g[e];
        if (b) {
            unpack<WT, V>(load<WT, V>(b, at.at), g);
#pragma unroll
            for (int e = 0; e < V; ++e) f[c][e] += g[e];
        }
        if (live && at.skip < V) store<DT, V, NT>(y + row * D * S, at.at, pack<DT, V>(f[c]));
    }
    if (stats && lane == 0 && live) {
        stats[2 * row] = mean;
        stats[2 * row + 1] = rstd;
    }
}

constexpr int kBwdThreads = 512;
constexpr int kWideThreads = 1024;  // (rows of fp32 past 8192)
constexpr int kBwdBlocks = 512;  // partial sums of dw and db: one pair of rows a workgroup

template <int DT, int C>
struct BwdRow {
    static constexpr int V = row_vec(DT);
    Elems<DT, V> dy[C], h[C], dh[C];
    float mean, rstd;
};

// Every group of tpr threads takes each (gridDim groups)-th row: one read of dy, h and dh, their
// last and non-temporal, gives dx, and what the row adds to dw and db stays in registers until
// the end.  The next row's loads are under way while a row is reduced, but with T = kWideThreads.
template <int DT, int WT, int C, bool NT, int T>
__global__ __launch_bounds__(T) void ln_bwd_kernel(
    const char* __restrict__ dy, int64_t lddy, const char* __restrict__ dh, int64_t lddh,
    const char* __restrict__ h, int64_t ldh, const void* __restrict__ w,
    const float* __restrict__ stats, char* __restrict__ dx, float* __restrict__ sums, int64_t N,
    int64_t D, int tpr) {
    extern __shared__ float lds[];
    __shared__ float part[2][32];
    constexpr int S = kElemBytes<DT>, V = row_vec(DT);
    const int lane = threadIdx.x & (tpr - 1), group = threadIdx.x / tpr;
    const int groups = T / tpr;
    const int64_t step = (int64_t)gridDim.x * groups;
    int turn = 0;
    Elems<WT, V> gamma[C];
    float aw[C][V], ab[C][V];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        gamma[c] = load<WT, V>(w, row_slot<V>(c, C, tpr, lane, D).at);
#pragma unroll
        for (int e = 0; e < V; ++e) aw[c][e] = ab[c][e] = 0.f;
    }
    auto fetch = [&](BwdRow<DT, C>& r, int64_t want) __attribute__((always_inline)) {
        const int64_t row = min(want, N - 1);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int64_t at = row_slot<V>(c, C, tpr, lane, D).at;
            r.dy[c] = load<DT, V, true>(dy + row * lddy * S, at);
            r.h[c] = load<DT, V, true>(h + row * ldh * S, at);
            if (dh) r.dh[c] = load<DT, V, true>(dh + row * lddh * S, at);
        }
        r.mean = stats[2 * row];
        r.rstd = stats[2 * row + 1];
    };
    // (all groups make the same number of turns: rows_sums may hold a barrier)
    const int64_t turns = (N + step - 1) / step;
    int64_t row = (int64_t)blockIdx.x * groups + group;
    constexpr bool AHEAD = T == kBwdThreads;
    BwdRow<DT, C> next;
    if (AHEAD) fetch(next, row);
    for (int64_t k = 0; k < turns; ++k, row += step) {
        if (!AHEAD) fetch(next, row);
        const BwdRow<DT, C> r = next;
        if (AHEAD && k + 1 < turns) fetch(next, row + step);
        const bool live = row < N;
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int skip = row_slot<V>(c, C, tpr, lane, D).skip;
            float d[V], n[V], g[V];
            unpack<DT, V>(r.dy[c], d);
            unpack<DT, V>(r.h[c], n);
            unpack<WT, V>(gamma[c], g);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                n[e] = (n[e] - r.mean) * r.rstd;
                const bool own = live && (c < C - 1 || e >= skip);
                const float a = d[e] * g[e];
                s1 += own ? a : 0.f;
                s2 += own ? a * n[e] : 0.f;
                aw[c][e] += own ? d[e] * n[e] : 0.f;
                ab[c][e] += own ? d[e] : 0.f;
            }
        }
        if (!dx) continue;
        row_sums(s1, s2, tpr, part, turn);
        const float c1 = s1 / (float)D, c2 = s2 / (float)D;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const Slot at = row_slot<V>(c, C, tpr, lane, D);
            float d[V], n[V], g[V];
            unpack<DT, V>(r.dy[c], d);
            unpack<DT, V>(r.h[c], n);
            unpack<WT, V>(gamma[c], g);
#pragma unroll
            for (int e = 0; e < V; ++e)
                d[e] = r.rstd * (d[e] * g[e] - c1 - (n[e] - r.mean) * r.rstd * c2);
            if (dh) {
                float q[V];
                unpack<DT, V>(r.dh[c], q);
#pragma unroll
                for (int e = 0; e < V; ++e) d[e] += q[e];
            }
            if (live && at.skip < V) store<DT, V, NT>(dx + row * D * S, at.at, pack<DT, V>(d));
        }
    }
    if (!sums) return;
    // the groups' sums, halved until the first has them all
    for (int half = groups / 2; half; half /= 2) {
        __syncthreads();
        float* p = lds + (group & (half - 1)) * (2 * V * C * tpr) + lane;
        if (group >= half && group < 2 * half) {
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    p[(2 * V * c + e) * tpr] = aw[c][e];
                    p[(2 * V * c + V + e) * tpr] = ab[c][e];
                }
        }
        __syncthreads();
        if (group < half) {
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    aw[c][e] += p[(2 * V * c + e) * tpr];
                    ab[c][e] += p[(2 * V * c + V + e) * tpr];
                }
        }
    }
    if (group) return;
    float* out = sums + (int64_t)blockIdx.x * 2 * D;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const Slot at = row_slot<V>(c, C, tpr, lane, D);
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (c < C - 1 || e >= at.skip) {
                out[at.at + e] = aw[c][e];
                out[D + at.at + e] = ab[c][e];
            }
    }
}

// dw (blockIdx.y 0) and db (1) from the workgroups' sums: 64 columns a workgroup, from column c0
// on, 16 sums of each side by side, joined in order.
template <int WT>
__global__ __launch_bounds__(1024) void ln_sums_kernel(const float* __restrict__ sums, int blocks,
                                                       void* dw, void* db, int64_t D, int64_t c0) {
    __shared__ float part[16][64];
    const int x = threadIdx.x & 63, k = threadIdx.x >> 6;
    const int64_t c = c0 + (int64_t)blockIdx.x * 64 + x;
    void* out = blockIdx.y ? db : dw;
    float s = 0.f;
    if (c < D) {
        const float* p = sums + blockIdx.y * D + c;
#pragma unroll 8
        for (int b = k; b < blocks; b += 16) s += p[(int64_t)b * 2 * D];
    }
    part[k][x] = s;
    __syncthreads();
    if (k || c >= D || !out) return;
    for (int j = 1; j < 16; ++j) s += part[j][x];
    store_elem<WT>(out, c, s);
}

// How the threads hold rows of D elements: the fewest threads left over in up to `slots` slots of
// `most` threads; among those the most threads up to `wide`, and never several slots of under
// `narrow` threads, whose accesses would touch only part of their lines (2^26 elements of fp32 in
// rows of 16 with one thread to a row 445 us, with four 108; rows of 100 with eight threads 231,
// with 16 128).  The forward takes several slots where it can (rows of 512 in bf16: 43 us with
// four, 52 with one, whose threads have one load under way), the backward, which has the next
// row's loads under way, one (70 and 73).  C == 0: rows that do not fit, or shorter than a slot.
struct RowShape {
    int tpr, C;
};
RowShape row_shape(int64_t D, int32_t dtype, int most, int slots, int narrow, int wide) {
    const int64_t V = row_vec(dtype);
    RowShape best{0, 0};
    int64_t over = 0;
    if (D < V) return best;
    for (int tpr = 1; tpr <= most; tpr *= 2) {
        const int64_t C = ceil_div(D, V * tpr);
        if (C > slots || (tpr < narrow && C > 1)) continue;
        const int64_t o = C * V * tpr - D;
        if (best.C == 0 || o < over || (o == over && tpr <= wide)) {
            best = RowShape{tpr, (int)C};
            over = o;
        }
    }
    return best;
}
RowShape fwd_shape(int64_t D, int32_t dtype) { return row_shape(D, dtype, 1024, 4, 16, 0); }
// (the registers of a backward slot: 56 with 16-bit rows and 40 with fp32 ones, of 256)
constexpr int bwd_slots(int32_t dtype) { return dtype == HASTE_DTYPE_F32 ? 4 : 3; }
// Wider fp32 rows take 1024 threads, with half the registers and no loads ahead of their row: rows
// of 12,000, 2^26 elements, 295 -> 162 us; of 16,384 (33 registers spilled) 321 -> 210.  With
// 16-bit rows, whose slots hold twice the elements, the any-width passes are as fast.
constexpr bool wide(int32_t dtype, int C) { return dtype == HASTE_DTYPE_F32 && C >= 3; }
RowShape bwd_shape(int64_t D, int32_t dtype) {
    const int64_t C = ceil_div(D, (int64_t)kWideThreads * row_vec(dtype));
    if (C <= 4 && wide(dtype, (int)C)) return RowShape{kWideThreads, (int)C};
    return row_shape(D, dtype, kBwdThreads, bwd_slots(dtype), 8, 64);
}

// Whether a matrix of rows is no more in the last-level cache when it is met again: half of it,
// since others are read beside it.  (65,536 rows of 4096 in bf16: 788 -> 700 us.)
bool past_cache(int64_t N, int64_t D, int32_t dtype) {
    return N * D * elem_bytes(dtype) > kMallBytes / 2;
}

// The partial sums of dw and db.
int bwd_blocks(int64_t N, const RowShape& r) {
    const int64_t rows = r.C ? std::max(kBwdThreads / r.tpr, 1) : 4 * kAnyRows;
    const int64_t most = r.C ? kBwdBlocks : 64;
    return (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(N, rows), most));
}

int ln_types(const char* fn, int32_t dtype, int32_t w_dtype) {
    HASTE_CHECK_ARG(elem_dtype(dtype), "%s: rows must be bf16, fp16 or fp32 (dtype code %d)", fn,
                    (int)dtype);
    HASTE_CHECK_ARG(w_dtype == dtype || w_dtype == HASTE_DTYPE_F32,
                    "%s: weights must be of the rows' dtype or fp32 (dtype code %d)", fn,
                    (int)w_dtype);
    return HASTE_OK;
}

// A matrix of rows `ld` apart that is read.
int ln_rows(const char* fn, const char* what, const void* p, int64_t ld, int64_t D, int32_t dtype) {
    HASTE_CHECK_ARG(p != nullptr, "%s: %s is NULL", fn, what);
    HASTE_CHECK_ARG(elem_aligned(p, dtype), "%s: %s is not aligned to its elements", fn, what);
    HASTE_CHECK_ARG(ld == 0 || ld >= D, "%s: row pitch of %s is short (%lld < %lld)", fn, what,
                    (long long)ld, (long long)D);
    return HASTE_OK;
}

// f(first, count) over launches of `count` rows or columns, `per` to a workgroup of `threads`: an axis
// of a launch takes fewer than 2^32 threads.
template <typename F>
void in_launches(int64_t count, int64_t per, int threads, F f) {
    const int64_t most = (((int64_t)1 << 32) - 1) / threads * per;
    for (int64_t i = 0; i < count; i += most) f(i, std::min(most, count - i));
}

// f with C as a constant.
template <typename F>
void with_slots(int C, F f) {
    if (C == 1) f(std::integral_constant<int, 1>());
    else if (C == 2) f(std::integral_constant<int, 2>());
    else if (C == 3) f(std::integral_constant<int, 3>());
    else f(std::integral_constant<int, 4>());
}

// `call` with DT and WT for the types of a call.
#define HASTE_LN_TYPES(call)                                                                 \
    do {                                                                                     \
        if (dtype == HASTE_DTYPE_F32) call(HASTE_DTYPE_F32, HASTE_DTYPE_F32);                \
        else if (dtype == HASTE_DTYPE_BF16 && w_dtype == dtype)                              \
            call(HASTE_DTYPE_BF16, HASTE_DTYPE_BF16);                                        \
        else if (dtype == HASTE_DTYPE_BF16) call(HASTE_DTYPE_BF16, HASTE_DTYPE_F32);         \
        else if (w_dtype == dtype) call(HASTE_DTYPE_F16, HASTE_DTYPE_F16);                   \
        else call(HASTE_DTYPE_F16, HASTE_DTYPE_F32);                                         \
    } while (0)

}  // namespace
}  // namespace haste

extern "C" int haste_layer_norm(const void* x, int64_t ldx, const void* res, int64_t ldres,
                                const void* w, const void* b, void* y, void* h, float* stats,
                                int64_t N, int64_t D, double eps, int32_t dtype, int32_t w_dtype,
                                void* stream) {
    const char* fn = "haste_layer_norm";
    HASTE_CHECK_ARG(N >= 0 && D > 0, "%s: bad sizes N=%lld D=%lld", fn, (long long)N, (long long)D);
    HASTE_CHECK_ARG(N < (int64_t)1 << 31 && D < (int64_t)1 << 31, "%s: matrix too large", fn);
    HASTE_CHECK_ARG(eps >= 0.0, "%s: eps must be >= 0", fn);
    HASTE_TRY(haste::ln_types(fn, dtype, w_dtype));
    if (N == 0) return HASTE_OK;
    HASTE_TRY(haste::ln_rows(fn, "x", x, ldx, D, dtype));
    if (res) {
        HASTE_TRY(haste::ln_rows(fn, "res", res, ldres, D, dtype));
        HASTE_TRY(haste::ln_rows(fn, "h", h, D, D, dtype));
    }
    HASTE_TRY(haste::ln_rows(fn, "w", w, D, D, w_dtype));
    HASTE_CHECK_ARG(haste::elem_aligned(b, w_dtype), "%s: b is not aligned to its elements", fn);
    HASTE_TRY(haste::ln_rows(fn, "y", y, D, D, dtype));
    HASTE_CHECK_ARG(haste::elem_aligned(stats, HASTE_DTYPE_F32), "%s: stats is misaligned", fn);
    const haste::RowShape r = haste::fwd_shape(D, dtype);
    const int threads = std::max(r.tpr, 256), rows = r.C ? threads / r.tpr : 1;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool nt = haste::past_cache(N, D, dtype);
    haste::in_launches(N, rows, threads, [&](int64_t r0, int64_t n) {
        const dim3 grid((unsigned)haste::ceil_div(n, (int64_t)rows));
        const int64_t size = haste::elem_bytes(dtype);
        const char *xc = static_cast<const char*>(x) + r0 * ldx * size,
                   *rc = res ? static_cast<const char*>(res) + r0 * ldres * size : nullptr;
        char *yc = static_cast<char*>(y) + r0 * D * size,
             *hc = res ? static_cast<char*>(h) + r0 * D * size : nullptr;
        float* sc = stats ? stats + 2 * r0 : nullptr;
        auto any = [&](auto kernel) {
            kernel<<<grid, dim3(haste::kRowThreads), 0, st>>>(xc, ldx, rc, ldres, w, b, yc, hc, sc, D,
                                                              (float)eps);
        };
#define HASTE_LN_FWD(DT, WT)                                                                       \
    do {                                                                                           \
        auto slots = [&](auto c) {                                                                 \
            constexpr int C = decltype(c)::value;                                                  \
            if (nt)                                                                                \
                haste::ln_fwd_kernel<DT, WT, C, true><<<grid, dim3(threads), 0, st>>>(             \
                    xc, ldx, rc, ldres, w, b, yc, hc, sc, n, D, (float)eps, r.tpr);                \
            else                                                                                   \
                haste::ln_fwd_kernel<DT, WT, C, false><<<grid, dim3(threads), 0, st>>>(            \
                    xc, ldx, rc, ldres, w, b, yc, hc, sc, n, D, (float)eps, r.tpr);                \
        };                                                                                         \
        if (r.C)                                                                                   \
            haste::with_slots(r.C, slots);                                                         \
        else                                                                                       \
            any(D < haste::row_vec(DT) ? haste::ln_fwd_any_kernel<DT, WT, 1>                       \
                                       : haste::ln_fwd_any_kernel<DT, WT, haste::row_vec(DT)>);    \
    } while (0)
        HASTE_LN_TYPES(HASTE_LN_FWD);
#undef HASTE_LN_FWD
    });
    HASTE_CHECK_LAUNCH(fn);
    return HASTE_OK;
}

extern "C" int64_t haste_layer_norm_bwd_workspace_size(int64_t N, int64_t D) {
    if (N < 0 || D < 0) return HASTE_ERR_INVALID_ARG;
    // (the larger of the two shapes that the rows' dtypes may take)
    int most = 1;
    for (int32_t dt : {HASTE_DTYPE_BF16, HASTE_DTYPE_F32})
        most = std::max(most, haste::bwd_blocks(N, haste::bwd_shape(D, dt)));
    return most * 2 * std::max<int64_t>(D, 8) * (int64_t)sizeof(float);
}

extern "C" int haste_layer_norm_bwd(const void* dy, int64_t lddy, const void* dh, int64_t lddh,
                                    const void* h, int64_t ldh, const void* w, const float* stats,
                                    void* dx, void* dw, void* db, void* ws, int64_t ws_bytes,
                                    int64_t N, int64_t D, int32_t dtype, int32_t w_dtype,
                                    void* stream) {
    const char* fn = "haste_layer_norm_bwd";
    HASTE_CHECK_ARG(N >= 0 && D > 0, "%s: bad sizes N=%lld D=%lld", fn, (long long)N, (long long)D);
    HASTE_CHECK_ARG(N < (int64_t)1 << 31 && D < (int64_t)1 << 31, "%s: matrix too large", fn);
    HASTE_TRY(haste::ln_types(fn, dtype, w_dtype));
    if (N > 0) {
        HASTE_TRY(haste::ln_rows(fn, "dy", dy, lddy, D, dtype));
        if (dh) HASTE_TRY(haste::ln_rows(fn, "dh", dh, lddh, D, dtype));
        HASTE_TRY(haste::ln_rows(fn, "h", h, ldh, D, dtype));
        HASTE_TRY(haste::ln_rows(fn, "w", w, D, D, w_dtype));
        HASTE_CHECK_ARG(stats != nullptr && haste::elem_aligned(stats, HASTE_DTYPE_F32),
                        "%s: stats is NULL or misaligned", fn);
        HASTE_CHECK_ARG(haste::elem_aligned(dx, dtype), "%s: dx is not aligned to its elements", fn);
    }
    HASTE_CHECK_ARG(haste::elem_aligned(dw, w_dtype) && haste::elem_aligned(db, w_dtype),
                    "%s: dw or db is not aligned to its elements", fn);
    if (dw || db) {
        const int64_t need = haste_layer_norm_bwd_workspace_size(N, D);
        HASTE_CHECK_ARG(ws != nullptr && haste::aligned16(ws), "%s: workspace is NULL or misaligned",
                        fn);
        if (ws_bytes < need) {
            haste::set_error("%s: workspace too small (%lld < %lld bytes)", fn, (long long)ws_bytes,
                             (long long)need);
            return HASTE_ERR_WORKSPACE;
        }
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    const haste::RowShape r = haste::bwd_shape(D, dtype);
    const int blocks = haste::bwd_blocks(N, r);
    const bool nt = haste::past_cache(N, D, dtype);
    const char *dyc = static_cast<const char*>(dy), *dhc = static_cast<const char*>(dh),
               *hc = static_cast<const char*>(h);
    float* sums = dw || db ? static_cast<float*>(ws) : nullptr;
    auto any_dx = [&](auto kernel) {
        haste::in_launches(N, 1, haste::kRowThreads, [&](int64_t r0, int64_t n) {
            const int64_t size = haste::elem_bytes(dtype);
            kernel<<<dim3((unsigned)n), dim3(haste::kRowThreads), 0, st>>>(
                dyc + r0 * lddy * size, lddy, dhc ? dhc + r0 * lddh * size : nullptr, lddh,
                hc + r0 * ldh * size, ldh, w, stats + 2 * r0,
                static_cast<char*>(dx) + r0 * D * size, D);
        });
    };
    auto any_dw = [&](auto kernel, int V) {
        haste::in_launches(D, 16 * V, haste::kRowThreads, [&](int64_t c0, int64_t n) {
            kernel<<<dim3((unsigned)haste::ceil_div(n, (int64_t)16 * V), blocks),
                     dim3(haste::kRowThreads), 0, st>>>(dyc, lddy, hc, ldh, stats, sums, N, D, c0);
        });
    };
    auto join = [&](auto kernel) {
        haste::in_launches(D, 64, 1024, [&](int64_t c0, int64_t n) {
            kernel<<<dim3((unsigned)haste::ceil_div(n, 64), 2), dim3(1024), 0, st>>>(sums, blocks, dw,
                                                                                   db, D, c0);
        });
    };
#define HASTE_LN_BWD(DT, WT)                                                                     \
    do {                                                                                         \
        auto slots = [&](auto c) {                                                               \
            constexpr int C = std::min(decltype(c)::value, haste::bwd_slots(DT));                \
            const size_t lds = r.tpr >= haste::kBwdThreads || !sums                              \
                                   ? 0                                                           \
                                   : sizeof(float) * haste::row_vec(DT) * C * haste::kBwdThreads; \
            auto kernel = nt ? haste::ln_bwd_kernel<DT, WT, C, true, haste::kBwdThreads>         \
                             : haste::ln_bwd_kernel<DT, WT, C, false, haste::kBwdThreads>;       \
            if constexpr (haste::wide(DT, C))                                                    \
                if (r.tpr == haste::kWideThreads)                                                \
                    kernel = nt ? haste::ln_bwd_kernel<DT, WT, C, true, haste::kWideThreads>     \
                                : haste::ln_bwd_kernel<DT, WT, C, false, haste::kWideThreads>;   \
            kernel<<<dim3(blocks), dim3(std::max(r.tpr, haste::kBwdThreads)), lds, st>>>(        \
                dyc, lddy, dhc, lddh, hc, ldh, w, stats, static_cast<char*>(dx), sums, N, D,     \
                r.tpr);                                                                          \
        };                                                                                       \
        if (N > 0 && r.C) {                                                                      \
            haste::with_slots(r.C, slots);                                                       \
        } else {                                                                                 \
            constexpr int V = haste::row_vec(DT);                                                \
            if (N > 0 && dx)                                                                     \
                any_dx(D < V ? haste::ln_dx_any_kernel<DT, WT, 1>                                \
                             : haste::ln_dx_any_kernel<DT, WT, V>);                              \
            if (sums && D < V)                                                                   \
                any_dw(haste::ln_dw_any_kernel<DT, 1>, 1);                                       \
            else if (sums)                                                                       \
                any_dw(haste::ln_dw_any_kernel<DT, V>, V);                                       \
        }                                                                                        \
        if (sums) join(haste::ln_sums_kernel<WT>);                                               \
    } while (0)
    HASTE_LN_TYPES(HASTE_LN_BWD);
#undef HASTE_LN_BWD
    HASTE_CHECK_LAUNCH(fn);
    return HASTE_OK;
}
