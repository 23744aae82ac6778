// Log probabilities of given labels under rows of logits, the rows' entropy and their likeliest labels:
//   m = max z, s = sum e^(z - m), log p = (z - m) - log s, H = log s - sum e^(z - m) (z - m) / s
// and the logits' gradient dz = p (-sum_l g_l - g_H (log p + H)) + sum_{l: label l = j} g_l.
// One pass over the logits forward and one backward: a thread keeps the running maximum and sums of its
// part of a row, a wave the largest K keys of its part.  Measured on bf16 logits: 512 rows of 670,091 forward
// 150 us (686 MB, 4.6 TB/s) and backward 228 us (1.4 GB, 6.0 TB/s, in part from the last-level cache), bound
// by HBM; 512 rows of 131,073 with ten labels 31 us (139 MB, 4.5 TB/s), some 6 of them to find the labels.  One
// row of 131,073: 8 us, and 5 us to join its parts, latency.
#include <algorithm>

#include "elements.hpp"

namespace haste {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxTop = 128;
constexpr float kGone = -150.f;  // e^x is 0 below

// ------------------------------------------------------------- softmax sums ----
// s = sum e^(z - m), t = sum e^(z - m) (z - m).  Before the first finite logit m is the lowest
// fp32 value, not -infinity, so that z - m is a number for every z but +infinity and NaN.
struct Sums {
    float m, s, t;
};
__device__ __forceinline__ Sums no_sums() { return Sums{-3.402823466e38f, 0.f, 0.f}; }
__device__ __forceinline__ void rescale(Sums& a, float m) {
    const float d = fmaxf(a.m - m, kGone), f = __builtin_amdgcn_exp2f(d * kLog2e);
    a.t = (a.t + a.s * d) * f;
    a.s *= f;
    a.m = m;
}
// What terms of maximum m are taken relative to: 2^(z log2 e - r) takes one operation where e^(z - m) takes
// two, with r = m log2 e rounded; `off`, the rounding, is made good in the sums.  Far from zero the
// rounding is too large for that, and (z - m) log2 e is taken.
constexpr float kLn2 = 0.69314718056f;
struct Reference {
    float r, off, scale;  // off = m log2 e - r, scale = 2^-off
    bool far;             // (of any lane)
};
__device__ __forceinline__ Reference reference(float m) {
    Reference ref{m * kLog2e, 0.f, 1.f, (bool)__any(!(fabsf(m) < 1024.f))};
    if (!ref.far) {
        ref.off = __builtin_fmaf(m, kLog2e, -ref.r);
        ref.scale = __builtin_fmaf(-kLn2, ref.off, 1.f);
    }
    return ref;
}
__device__ __forceinline__ Sums join(Sums a, Sums b) {
    const float m = fmaxf(a.m, b.m);
    rescale(a, m);
    rescale(b, m);
    return Sums{m, a.s + b.s, a.t + b.t};
}

// ------------------------------------------------------------ largest K keys ----
// A label's key: its logit's order, then the lower label first.  0 is no label's.  NaN is largest.
typedef unsigned long long Key;
__device__ __forceinline__ uint32_t order_of(float z) {
    const uint32_t u = z == 0.f ? 0u : __float_as_uint(z);
    return z != z ? 0xFFFFFFFFu : u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ Key key_of(float z, uint32_t label) {
    return (Key)order_of(z) << 32 | (0xFFFFFFFFu - label);
}
__device__ __forceinline__ float value_of(Key k) {
    const uint32_t u = (uint32_t)(k >> 32);
    return __uint_as_float(u == 0xFFFFFFFFu ? 0x7FC00000u
                                            : u ^ ((u >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ uint32_t label_of(Key k) { return 0xFFFFFFFFu - (uint32_t)k; }

__device__ __forceinline__ uint32_t lane_value(uint32_t v, int lane) {
    return (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}

// A wave's list of candidates in LDS, of 64 R keys.  Whenever fewer than 64 places are free it is cut to
// its largest K, in order, and the K-th is what a key has to exceed from then on; `shared` holds the
// largest such bound of the workgroup.
template <int R>
struct Candidates {
    Key* buf;
    Key* shared;
    int K, count, lane;
    Key bound;
    // Every key goes to the place that the number of larger ones gives: fewer steps that wait for one
    // another than a sorting network has, and as many as there are keys.
    __device__ __forceinline__ void cut() {
        Key k[R];
        int rank[R];
        wave_sync();
#pragma unroll
        for (int r = 0; r < R; ++r) {
            k[r] = r * 64 + lane < count ? buf[r * 64 + lane] : 0;
            rank[r] = 0;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int n = min(64, count - r * 64);
            for (int j = 0; j < n; ++j) {
                const Key o = (Key)lane_value((uint32_t)(k[r] >> 32), j) << 32 | lane_value((uint32_t)k[r], j);
#pragma unroll
                for (int q = 0; q < R; ++q) rank[q] += o > k[q] ? 1 : 0;
            }
        }
        wave_sync();
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (r * 64 + lane < count) {
                if (rank[r] < K) buf[rank[r]] = k[r];
            } else if (r * 64 + lane < K) {
                buf[r * 64 + lane] = 0;
            }
        wave_sync();
        if (count >= K) {
            count = K;
            bound = max(bound, buf[K - 1]);
            if (lane == 0) atomicMax(shared, bound);
        }
    }
    // The keys of the wave's lanes; 0 for none.
    __device__ __forceinline__ void add(Key key) {
        const bool pass = key > bound;
        const uint64_t mask = __ballot(pass);
        if (!mask) return;
        if (pass) buf[count + __popcll(mask & (((uint64_t)1 << lane) - 1))] = key;
        count += __popcll(mask);
        if (count > 64 * (R - 1)) cut();
    }
};

// The K-th largest of the workgroup's values, one to a thread (u; `share` has room for them), by halving: a
// key that every label of such an order exceeds.  Orders are taken to the bits that the logits' type has.
// Every thread calls.
template <int DT>
__device__ __forceinline__ Key bound_of(uint32_t u, uint32_t* share, int K) {
    constexpr int bits = DT == HASTE_DTYPE_F32 ? 32 : DT == HASTE_DTYPE_BF16 ? 16 : 19;
    share[threadIdx.x] = u;
    __syncthreads();
    uint32_t x[kWaves], least = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) x[w] = share[w * 64 + (threadIdx.x & 63)];
#pragma unroll
    for (int b = 31; b >= 32 - bits; --b) {
        const uint32_t more = least | 1u << b;
        int reach = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) reach += __popcll(__ballot(x[w] >= more));
        least = reach >= K ? more : least;
    }
    return (Key)least << 32;
}

// A thread's windows of steps, at most.  More re-read less and keep more: with four workgroups to a CU 512 x
// 131,073 with the 100 likeliest took 59 us, with 4 windows 63; 4096 x 20,000 with 10 53 us, with 16 windows 60.
constexpr int kWindows = 8;
constexpr int buffer_keys(int R) { return R ? 64 * R : 1; }

// The workgroup's sums and largest keys from its waves' in wave 0's list.
template <int R>
struct Shared {
    Sums sums[kWaves];
    int count[kWaves];
    Key bound;
    Key buf[kWaves][buffer_keys(R)];
};

template <int R>
__device__ __forceinline__ void join_waves(Shared<R>& sh, Sums& a, Candidates<R ? R : 2>& c) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int o = 32; o; o >>= 1) {
        Sums b;
        b.m = __shfl_xor(a.m, o);
        b.s = __shfl_xor(a.s, o);
        b.t = __shfl_xor(a.t, o);
        a = join(a, b);
    }
    if (lane == 0) {
        sh.sums[wave] = a;
        if (R) sh.count[wave] = c.count;
    }
    __syncthreads();
    a = sh.sums[0];
    for (int w = 1; w < kWaves; ++w) a = join(a, sh.sums[w]);
    if constexpr (R > 0) {
        if (wave == 0) {
            // (the key that is the bound may be in another wave's list)
            c.bound = sh.bound ? sh.bound - 1 : 0;
            for (int w = 1; w < kWaves; ++w)
                for (int i = 0; i < sh.count[w]; i += 64)
                    c.add(i + lane < sh.count[w] ? sh.buf[w][i + lane] : 0);
            c.cut();
        }
        __syncthreads();
    }
}

struct Out {
    float *stats, *log_probs, *entropy, *top;
    int64_t* top_labels;
};

template <int DT>
__device__ __forceinline__ void write_row(const void* z, const void* labels, bool wide, int64_t L,
                                          int64_t O, int K, int64_t row, const Sums& a,
                                          const Key* keys, const Out& out) {
    // (a row without a finite logit has no distribution: NaN)
    const float log_s = a.s > 0.f ? logf(a.s) : __uint_as_float(0x7FC00000u);
    if (threadIdx.x == 0) {
        if (out.stats) {
            out.stats[2 * row] = a.m;
            out.stats[2 * row + 1] = a.s > 0.f ? a.s : __uint_as_float(0x7FC00000u);
        }
        if (out.entropy) out.entropy[row] = log_s - a.t / a.s;
    }
    for (int64_t l = threadIdx.x; l < L; l += kThreads) {
        const int64_t i = row * L + l;
        const int64_t j = wide ? static_cast<const int64_t*>(labels)[i]
                               : (int64_t)static_cast<const int32_t*>(labels)[i];
        out.log_probs[i] = j >= 0 && j < O ? (load_elem<DT>(z, j) - a.m) - log_s : 0.f;
    }
    for (int k = threadIdx.x; k < K; k += kThreads) {
        out.top[row * K + k] = (value_of(keys[k]) - a.m) - log_s;
        out.top_labels[row * K + k] = label_of(keys[k]);
    }
}

// Part `blockIdx.x % S` of row `blockIdx.x / S`.  Vectors lie on 16-byte boundaries; the row's first
// and last may have elements of other rows in them, which are not read.
template <int DT, int R>
__global__ __launch_bounds__(kThreads) void lp_kernel(const char* z, int64_t ldz, const void* labels,
                                                      int wide, int64_t L, int64_t O, int K, int S,
                                                      int64_t per, Out out, Sums* part,
                                                      Key* part_keys, int64_t row0) {
    constexpr int SZ = kElemBytes<DT>, V = 16 / SZ;
    typedef Elems<DT, V> Vec;
    __shared__ Shared<R> sh;
    // a thread's largest logit of each window of its steps (as orders), and those that are read again
    __shared__ uint32_t seen[R ? kWindows : 1][R ? kThreads : 1], share[R ? kThreads : 1];
    __shared__ uint16_t list[R ? kWaves : 1][R ? 64 * kWindows : 1];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t row = row0 + blockIdx.x / S;
    const int c = blockIdx.x % S;
    const char* p = z + row * ldz * SZ;
    const int off = (int)((reinterpret_cast<uintptr_t>(p) & 15) / SZ);
    const int64_t nv = (off + O + V - 1) / V;
    const int64_t v1 = min(nv, (c + 1) * per);
    Sums a = no_sums();
    Candidates<R ? R : 2> top{sh.buf[wave], &sh.bound, K, 0, lane, 0};
    // Lane's vector v; what is not the part's is -infinity.
    auto fetch = [&](int64_t v) __attribute__((always_inline)) {
        const int64_t e0 = v * V - off;
        constexpr uint32_t none = DT == HASTE_DTYPE_F32    ? 0xFF800000u
                                  : DT == HASTE_DTYPE_BF16 ? 0xFF80FF80u
                                                           : 0xFC00FC00u;
        Vec q;
#pragma unroll
        for (int i = 0; i < 4; ++i) q.q[i] = none;
        if (v >= v1) return q;
        if (e0 >= 0 && e0 + V <= O) return load<DT, V>(p, e0);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if (e0 + e < 0 || e0 + e >= O) continue;
            if constexpr (DT == HASTE_DTYPE_F32) {
                q.q[e] = reinterpret_cast<const uint32_t*>(p)[e0 + e];
            } else {
                const uint32_t h = reinterpret_cast<const uint16_t*>(p)[e0 + e];
                q.q[e / 2] = (e & 1) ? (q.q[e / 2] & 0xFFFFu) | h << 16 : (q.q[e / 2] & 0xFFFF0000u) | h;
            }
        }
        return q;
    };
    constexpr int U = 2;
    const int64_t v0 = c * per + wave * 64, stride = U * kThreads,
                  steps = v0 < v1 ? (v1 - v0 + stride - 1) / stride : 0;
    const int length = (int)((steps + kWindows - 1) / kWindows);  // steps to a window
    float all = -__builtin_inff(), most = all;  // the largest of the lane's logits, and of the window's
    int window = 0, left = length;
    auto close = [&]() __attribute__((always_inline)) {
        all = fmaxf(all, most);
        if constexpr (R > 0) {
            seen[window++][threadIdx.x] = order_of(most);
            most = -__builtin_inff();
            left = length;
        }
    };
    Reference ref = reference(a.m);
    auto step = [&](const Vec (&q)[U]) __attribute__((always_inline)) {
        float f[U * V];
#pragma unroll
        for (int u = 0; u < U; ++u) unpack<DT, V>(q[u], f + u * V);
        float top_of_step = f[0];
#pragma unroll
        for (int e = 1; e < U * V; ++e) top_of_step = fmaxf(top_of_step, f[e]);
        most = fmaxf(most, top_of_step);
        // (terms up to e^2 lose nothing, and a new maximum by more is rare)
        if (__any(top_of_step > a.m + 2.f)) {
            rescale(a, fmaxf(a.m, top_of_step));
            ref = reference(a.m);
        }
        float s = 0.f, t = 0.f;
        if (!ref.far) {
#pragma unroll
            for (int e = 0; e < U * V; ++e) {
                const float w = __builtin_fmaf(f[e], kLog2e, -ref.r), x = __builtin_amdgcn_exp2f(w);
                s += x;
                t = __builtin_fmaf(x, fmaxf(w, kGone), t);
            }
        } else {
#pragma unroll
            for (int e = 0; e < U * V; ++e) {
                const float w = (f[e] - a.m) * kLog2e, x = __builtin_amdgcn_exp2f(w);
                s += x;
                t = __builtin_fmaf(x, fmaxf(w, kGone), t);
            }
        }
        a.s = __builtin_fmaf(s, ref.scale, a.s);
        a.t = __builtin_fmaf(__builtin_fmaf(-ref.off, s, t), ref.scale * kLn2, a.t);
        if (R > 0 && --left == 0) close();
    };
    // two vectors a step, the next two on their way; steps up to in1 have whole vectors only
    const int64_t whole = min(v1, (off + O) / V);  // (vectors behind it are not whole)
    const int64_t in1 = max((int64_t)0, (whole - v0 - (U - 1) * kThreads - 64 + stride) / stride);
    Vec q[U], next[U];
    auto edge = [&](int64_t i) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = fetch(v0 + i * stride + u * kThreads + lane);
    };
    int64_t i = 0;
    if (v0 * V < off && steps > 0) {
        edge(i++);
        step(q);
    }
    if (i < in1) {
        const char* at = p + ((v0 + i * stride + lane) * V - off) * SZ;
#pragma unroll
        for (int u = 0; u < U; ++u) next[u] = load<DT, V>(at, (int64_t)u * kThreads * V);
        for (; i < in1; ++i) {
#pragma unroll
            for (int u = 0; u < U; ++u) q[u] = next[u];
            at += i + 1 < in1 ? stride * 16 : 0;  // (the last step's are read again)
#pragma unroll
            for (int u = 0; u < U; ++u) next[u] = load<DT, V>(at, (int64_t)u * kThreads * V);
            step(q);
        }
    }
    for (; i < steps; ++i) {
        edge(i);
        step(q);
    }
    if (R == 0 || left < length) close();
    rescale(a, fmaxf(a.m, all));
    if constexpr (R > 0) {
        // K of the threads reach the K-th largest of their maxima, so K labels do, and no label under it is
        // among the K likeliest.  Only the threads' windows that reach it are read again: a few.
        if (threadIdx.x == 0) sh.bound = 0;
        // (a NaN hides from the maxima, but not from the sum; it is not what bounds, since +infinity makes the
        // sum one too)
        const bool hidden = a.s != a.s;
        top.bound = bound_of<DT>(order_of(all), share, K);
        if (lane == 0) atomicMax(&sh.bound, top.bound);
        int found = 0;
        for (int w = 0; w < window; ++w) {
            const bool in = hidden || seen[w][threadIdx.x] >= (uint32_t)(top.bound >> 32);
            const uint64_t mask = __ballot(in);
            if (in) list[wave][found + __popcll(mask & (((uint64_t)1 << lane) - 1))] = w * 64 + lane;
            found += __popcll(mask);
        }
        wave_sync();
        // (two vectors of a lane at a time: their loads do not wait for one another)
        constexpr int B = 2;
        const int vectors = length * U, items = found * vectors;
        for (int i0 = 0; i0 < items; i0 += 64 * B) {
            const int n = items - i0 > 64 ? 2 : 1;
            Vec w[B];
            int64_t v[B];
#pragma unroll
            for (int k = 0; k < B; ++k) {
                if (k >= n) break;
                const uint32_t i = i0 + k * 64 + lane, x = min(i / vectors, (uint32_t)found - 1);
                const int at = list[wave][x];
                v[k] = i < (uint32_t)items
                           ? v0 + ((int64_t)(at >> 6) * vectors + i % vectors) * kThreads + (at & 63)
                           : v1;
                w[k] = fetch(v[k]);
            }
#pragma unroll
            for (int k = 0; k < B; ++k) {
                if (k >= n) break;
                float f[V];
                unpack<DT, V>(w[k], f);
                const float least = value_of(top.bound);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    if (!__any(!(f[e] < least))) continue;
                    const int64_t j = v[k] * V - off + e;
                    top.add(v[k] < v1 && j >= 0 && j < O ? key_of(f[e], (uint32_t)j) : 0);
                }
            }
        }
    }
    join_waves<R>(sh, a, top);
    if (S == 1) {
        write_row<DT>(p, labels, wide, L, O, K, row, a, sh.buf[0], out);
        return;
    }
    if (threadIdx.x == 0) part[row * S + c] = a;
    for (int k = threadIdx.x; k < K; k += kThreads)
        part_keys[(row * S + c) * K + k] = sh.buf[0][k];
}

// A row's parts joined.
template <int DT, int R>
__global__ __launch_bounds__(kThreads) void lp_join_kernel(const char* z, int64_t ldz,
                                                           const void* labels, int wide, int64_t L,
                                                           int64_t O, int K, int S, Out out,
                                                           const Sums* part, const Key* part_keys,
                                                           int64_t row0) {
    __shared__ Shared<R> sh;
    __shared__ uint32_t share[R ? kThreads : 1];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t row = row0 + blockIdx.x;
    Sums a = no_sums();
    for (int i = threadIdx.x; i < S; i += kThreads) a = join(a, part[row * S + i]);
    Candidates<R ? R : 2> top{sh.buf[wave], &sh.bound, K, 0, lane, 0};
    if constexpr (R > 0) {
        if (threadIdx.x == 0) sh.bound = 0;
        const int64_t n = (int64_t)S * K;
        uint32_t most = 0;
        for (int64_t i = threadIdx.x; i < n; i += kThreads)
            most = max(most, (uint32_t)(part_keys[row * n + i] >> 32));
        top.bound = bound_of<DT>(most, share, K);  // (as in the parts)
        if (lane == 0) atomicMax(&sh.bound, top.bound);
        for (int64_t i = wave * 64; i < n; i += kThreads)
            top.add(i + lane < n ? part_keys[row * n + i + lane] : 0);
    }
    join_waves<R>(sh, a, top);
    write_row<DT>(z + row * ldz * kElemBytes<DT>, labels, wide, L, O, K, row, a, sh.buf[0], out);
}

// Elements [blockIdx.x % S * per, ...) of a row.  The labels' own elements are written again, with what
// their labels add, after every thread's stores are done.
template <int DT>
__global__ __launch_bounds__(kThreads) void lp_bwd_kernel(const char* z, int64_t ldz,
                                                          const void* labels, int wide, int64_t L,
                                                          const float* stats, const float* entropy,
                                                          const float* dlp, const float* dent,
                                                          char* dz, int64_t lddz, int64_t O, int S,
                                                          int64_t per, int64_t row0) {
    constexpr int SZ = kElemBytes<DT>, V = 16 / SZ;
    const int64_t row = row0 + blockIdx.x / S, from = blockIdx.x % S * per, to = min(O, from + per);
    z += row * ldz * SZ;
    dz += row * lddz * SZ;
    const float m = stats[2 * row], s = stats[2 * row + 1], H = entropy[row];
    const float log_s = logf(s), inv = 1.f / s;
    const float ge = dent ? dent[row] : 0.f;
    auto label = [&](int64_t l) __attribute__((always_inline)) {
        const int64_t i = row * L + l;
        return wide ? static_cast<const int64_t*>(labels)[i]
                    : (int64_t)static_cast<const int32_t*>(labels)[i];
    };
    float sum = 0.f;
    if (dlp)
        for (int64_t l = 0; l < L; ++l) {
            const int64_t j = label(l);
            if (j >= 0 && j < O) sum += dlp[row * L + l];
        }
    const float c0 = -sum - ge * H;
    // (16-bit gradients have no use for the last bits of e^d.  The instruction gives 0 for what is under 2^-126,
    // where bf16 has values yet once the factor, up to some hundreds, is in: it takes 2^24 e^d.)
    auto base = [&](float x) __attribute__((always_inline)) {
        const float d = x - m, by = __builtin_fmaf(-ge, fmaxf(d, kGone) - log_s, c0);
        if constexpr (DT == HASTE_DTYPE_F32) return expf(d) * inv * by;
        return __builtin_amdgcn_exp2f(__builtin_fmaf(d, kLog2e, 24.f)) * inv * by * 0x1p-24f;
    };
    for (int64_t e0 = from + threadIdx.x * V; e0 < to; e0 += kThreads * V) {
        float f[V];
        unpack<DT, V>(load_part<DT, V>(z, e0, to - e0), f);
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = base(f[e]);
        store_part<DT, V>(dz, e0, pack<DT, V>(f), to - e0);
    }
    if (!dlp) return;
    __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
    __syncthreads();
    for (int64_t l = threadIdx.x; l < L; l += kThreads) {
        const int64_t j = label(l);
        if (j < from || j >= to) continue;
        bool first = true;
        for (int64_t k = 0; k < l; ++k) first &= label(k) != j;
        if (!first) continue;
        float g = 0.f;
        for (int64_t k = l; k < L; ++k) g += label(k) == j ? dlp[row * L + k] : 0.f;
        store_elem<DT>(dz, j, base(load_elem<DT>(z, j)) + g);
    }
}

// How a row is cut: `per` 16-byte vectors to a part, whole steps of a workgroup's.  Two workgroups to a CU (512
// rows of 131,073 with ten labels: 30.5 us, with four 36.4, with eight 42; 1000 rows without: 48 and 58), in as
// many parts as there are steps; but a row of up to 8 steps is not cut where there is one for each CU, since
// joining parts takes a launch more (5 to 8 us).
constexpr int64_t kStep = 2 * kThreads;
struct Cut {
    int64_t per;
    int parts;
};
Cut cut_of(int64_t B, int64_t O, int32_t dtype) {
    const int64_t vectors = ceil_div(O, 16 / elem_bytes(dtype)) + 1, steps = ceil_div(vectors, kStep);
    if (B >= 256 && steps <= 8) return Cut{steps * kStep, 1};
    const int64_t parts = std::min<int64_t>({ceil_div(512, std::max<int64_t>(B, 1)), steps, 256});
    const int64_t per = ceil_div(steps, parts);
    return Cut{per * kStep, (int)ceil_div(steps, per)};
}

int lp_check(const char* fn, const void* z, int64_t ldz, const void* labels, int32_t label_bits,
             int64_t L, int64_t B, int64_t O, int32_t dtype) {
    HASTE_CHECK_ARG(B >= 0 && O > 0 && L >= 0, "%s: bad sizes B=%lld O=%lld L=%lld", fn, (long long)B,
                    (long long)O, (long long)L);
    HASTE_CHECK_ARG(B < (int64_t)1 << 31 && O < (int64_t)1 << 31 && L < (int64_t)1 << 31,
                    "%s: too large", fn);
    HASTE_CHECK_ARG(elem_dtype(dtype), "%s: logits must be bf16, f16 or f32", fn);
    HASTE_CHECK_ARG(label_bits == 32 || label_bits == 64, "%s: labels have 32 or 64 bits", fn);
    if (B == 0) return HASTE_OK;
    HASTE_CHECK_ARG(z != nullptr && elem_aligned(z, dtype), "%s: logits are NULL or misaligned", fn);
    HASTE_CHECK_ARG(ldz == 0 || ldz >= O, "%s: row pitch of the logits is short (%lld < %lld)", fn,
                    (long long)ldz, (long long)O);
    HASTE_CHECK_ARG(L == 0 || (labels != nullptr &&
                               reinterpret_cast<uintptr_t>(labels) % (label_bits / 8) == 0),
                    "%s: labels are NULL or misaligned", fn);
    return HASTE_OK;
}

// f(first row, rows) over launches of fewer than 2^32 threads.
template <typename F>
void in_launches(int64_t B, int64_t S, F f) {
    const int64_t most = (((int64_t)1 << 32) - 1) / (kThreads * S);
    for (int64_t i = 0; i < B; i += most) f(i, std::min(most, B - i));
}

#define HASTE_LP_TYPES(call)                                                                  \
    do {                                                                                      \
        if (dtype == HASTE_DTYPE_F32) call(HASTE_DTYPE_F32);                                  \
        else if (dtype == HASTE_DTYPE_BF16) call(HASTE_DTYPE_BF16);                           \
        else call(HASTE_DTYPE_F16);                                                           \
    } while (0)

int64_t lp_workspace(int64_t B, int64_t O, int64_t K) {
    int64_t S = 1;
    for (int32_t dtype : {HASTE_DTYPE_BF16, HASTE_DTYPE_F32}) S = std::max<int64_t>(S, cut_of(B, O, dtype).parts);
    return S == 1 ? 0 : ceil_div(B * S * (int64_t)sizeof(Sums), 16) * 16 + B * S * K * 8;
}

}  // namespace
}  // namespace haste

extern "C" int64_t haste_label_log_probs_workspace_size(int64_t B, int64_t O, int32_t K) {
    if (B < 0 || O <= 0 || K < 0 || K > haste::kMaxTop || B >= (int64_t)1 << 31 ||
        O >= (int64_t)1 << 31)
        return HASTE_ERR_INVALID_ARG;
    return haste::lp_workspace(B, O, K);
}

extern "C" int haste_label_log_probs(const void* z, int64_t ldz, const void* labels,
                                     int32_t label_bits, int64_t L, float* stats, float* log_probs,
                                     float* entropy, float* top, int64_t* top_labels, int64_t B,
                                     int64_t O, int32_t K, int32_t dtype, void* ws, int64_t ws_bytes,
                                     void* stream) {
    const char* fn = "haste_label_log_probs";
    const int rc = haste::lp_check(fn, z, ldz, labels, label_bits, L, B, O, dtype);
    if (rc != HASTE_OK) return rc;
    HASTE_CHECK_ARG(K >= 0 && K <= haste::kMaxTop && K <= O, "%s: top must be 0 to min(%d, O) (got %d)",
                    fn, haste::kMaxTop, (int)K);
    if (B == 0) return HASTE_OK;
    HASTE_CHECK_ARG(haste::elem_aligned(stats, HASTE_DTYPE_F32) &&
                        haste::elem_aligned(entropy, HASTE_DTYPE_F32),
                    "%s: stats or entropy is misaligned", fn);
    HASTE_CHECK_ARG(L == 0 || (log_probs != nullptr && haste::elem_aligned(log_probs, HASTE_DTYPE_F32)),
                    "%s: log_probs is NULL or misaligned", fn);
    HASTE_CHECK_ARG(K == 0 || (top != nullptr && top_labels != nullptr &&
                               haste::elem_aligned(top, HASTE_DTYPE_F32) &&
                               reinterpret_cast<uintptr_t>(top_labels) % 8 == 0),
                    "%s: top or top_labels is NULL or misaligned", fn);
    const haste::Cut cut = haste::cut_of(B, O, dtype);
    const int S = cut.parts;
    if (S > 1) {
        const int64_t need = haste::lp_workspace(B, O, K);
        HASTE_CHECK_ARG(ws != nullptr && haste::aligned16(ws), "%s: workspace is NULL or misaligned",
                        fn);
        if (ws_bytes < need) {
            haste::set_error("%s: workspace too small (%lld < %lld bytes)", fn, (long long)ws_bytes,
                             (long long)need);
            return HASTE_ERR_WORKSPACE;
        }
    }
    auto* part = static_cast<haste::Sums*>(ws);
    auto* keys = reinterpret_cast<haste::Key*>(
        static_cast<char*>(ws) + haste::ceil_div(B * S * (int64_t)sizeof(haste::Sums), 16) * 16);
    const haste::Out out{stats, log_probs, entropy, top, top_labels};
    hipStream_t st = static_cast<hipStream_t>(stream);
    const char* zc = static_cast<const char*>(z);
    const int wide = label_bits == 64;
    haste::in_launches(B, S, [&](int64_t r0, int64_t n) {
#define HASTE_LP(DT)                                                                               \
    do {                                                                                           \
        auto kernel = K == 0    ? haste::lp_kernel<DT, 0>                                          \
                      : K <= 32 ? haste::lp_kernel<DT, 2>                                          \
                                : haste::lp_kernel<DT, 4>;                                         \
        auto join = K == 0    ? haste::lp_join_kernel<DT, 0>                                       \
                    : K <= 32 ? haste::lp_join_kernel<DT, 2>                                       \
                              : haste::lp_join_kernel<DT, 4>;                                      \
        kernel<<<dim3((unsigned)(n * S)), dim3(haste::kThreads), 0, st>>>(                         \
            zc, ldz, labels, wide, L, O, K, S, cut.per, out, part, keys, r0);                          \
        if (S > 1)                                                                                 \
            join<<<dim3((unsigned)n), dim3(haste::kThreads), 0, st>>>(zc, ldz, labels, wide, L, O, \
                                                                      K, S, out, part, keys, r0);  \
    } while (0)
        HASTE_LP_TYPES(HASTE_LP);
#undef HASTE_LP
    });
    HASTE_CHECK_LAUNCH(fn);
    return HASTE_OK;
}

extern "C" int haste_label_log_probs_bwd(const void* z, int64_t ldz, const void* labels,
                                         int32_t label_bits, int64_t L, const float* stats,
                                         const float* entropy, const float* dlp, const float* dent,
                                         void* dz, int64_t lddz, int64_t B, int64_t O,
                                         int32_t dtype, void* stream) {
    const char* fn = "haste_label_log_probs_bwd";
    const int rc = haste::lp_check(fn, z, ldz, labels, label_bits, dlp ? L : 0, B, O, dtype);
    if (rc != HASTE_OK) return rc;
    // (a row's labels are compared with one another)
    HASTE_CHECK_ARG(!dlp || L <= HASTE_MAX_GRAD_LABELS, "%s: at most %d labels a row (got %lld)", fn,
                    HASTE_MAX_GRAD_LABELS, (long long)L);
    if (B == 0) return HASTE_OK;
    HASTE_CHECK_ARG(stats != nullptr && entropy != nullptr &&
                        haste::elem_aligned(stats, HASTE_DTYPE_F32) &&
                        haste::elem_aligned(entropy, HASTE_DTYPE_F32),
                    "%s: stats or entropy is NULL or misaligned", fn);
    HASTE_CHECK_ARG(haste::elem_aligned(dlp, HASTE_DTYPE_F32) &&
                        haste::elem_aligned(dent, HASTE_DTYPE_F32),
                    "%s: a gradient is misaligned", fn);
    HASTE_CHECK_ARG(dz != nullptr && haste::elem_aligned(dz, dtype) && lddz >= O,
                    "%s: dz is NULL or misaligned, or its row pitch is short", fn);
    // (four vectors to a thread)
    const int64_t V = 16 / haste::elem_bytes(dtype), most = haste::kThreads * V * 4;
    const int64_t S = haste::ceil_div(O, most);
    hipStream_t st = static_cast<hipStream_t>(stream);
    haste::in_launches(B, S, [&](int64_t r0, int64_t n) {
#define HASTE_LP(DT)                                                                             \
    haste::lp_bwd_kernel<DT><<<dim3((unsigned)(n * S)), dim3(haste::kThreads), 0, st>>>(         \
        static_cast<const char*>(z), ldz, labels, label_bits == 64, L, stats, entropy, dlp,     \
        dent, static_cast<char*>(dz), lddz, O, (int)S, most, r0)
        HASTE_LP_TYPES(HASTE_LP);
#undef HASTE_LP
    });
    HASTE_CHECK_LAUNCH(fn);
    return HASTE_OK;
}
