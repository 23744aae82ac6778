// What the products of the gated feed-forward block do with their sums, for all types:
//   forward   g = x Wg^T, u = x Wu^T, h = act(g) u;  y = h Wd^T
//   backward  dh = dy Wd, dg = dh u act'(g), du = dh act(g);  dx = dg Wg + du Wu,
//             dWg = dg^T x, dWu = du^T x, dWd = dy^T h
// The epilogues of h and of dg and du are bound by what they move, 8 and 10 bytes an element for 16-bit
// matrices (65,536 x 2048: 1.07 GB and 1.34 GB, 220 and 270 us of HBM, in part under the products).
#pragma once

#include <type_traits>

#include "elements.hpp"

namespace haste {

// act(g) and act'(g).  16-bit results have no use for the last bits of the exponential's.
template <bool PRECISE>
__device__ __forceinline__ float sigmoid(float x) {
    if (PRECISE) return 1.f / (1.f + expf(-x));
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
}
template <int ACT, bool PRECISE>
__device__ __forceinline__ void activation(float g, float* a, float* slope) {
    if constexpr (ACT == HASTE_ACT_SILU) {
        const float s = sigmoid<PRECISE>(g);
        *a = g * s;
        *slope = s * __builtin_fmaf(g, 1.f - s, 1.f);
    } else if constexpr (ACT == HASTE_ACT_GELU) {
        float cdf, e;  // the normal distribution at g, e^(-g^2 / 2)
        if constexpr (PRECISE) {
            cdf = 0.5f * erfcf(-0.70710678118654752f * g);
            e = expf(-0.5f * g * g);
        } else {
            // erfc(x) e^(x^2), x = |g| / sqrt 2, as a polynomial in t = 1 / (1 + x / 2): a least-squares fit
            // with weights driven to equal errors, 1.5e-6 of its value up to x = 9.5 (e^(-x^2) is 0 in fp32
            // behind).  A fifth of erfcf's operations, which took 5 of 15 us at 509 rows.
            const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.35355339059f, fabsf(g), 1.f));
            float q = 0.08912339f;
            q = __builtin_fmaf(q, t, -0.35997868f);
            q = __builtin_fmaf(q, t, 0.393769f);
            q = __builtin_fmaf(q, t, 0.03466602f);
            q = __builtin_fmaf(q, t, 0.28271684f);
            q = __builtin_fmaf(q, t, 0.27735418f);
            q = __builtin_fmaf(q, t, 0.28234804f);
            e = __builtin_amdgcn_exp2f(-0.72134752044448170f * g * g);
            const float tail = 0.5f * q * t * e;
            cdf = g < 0.f ? tail : 1.f - tail;
        }
        *a = g * cdf;
        *slope = __builtin_fmaf(g * 0.39894228040143268f, e, cdf);
    } else {
        // 0.5 (1 + tanh(t)) = sigmoid(2 t), t = sqrt(2 / pi) (g + 0.044715 g^3)
        const float t2 = 1.5957691216057308f * g * __builtin_fmaf(0.044715f * g, g, 1.f);
        const float s = sigmoid<PRECISE>(t2);
        *a = g * s;
        const float d = 1.5957691216057308f * __builtin_fmaf(3 * 0.044715f * g, g, 1.f);
        *slope = __builtin_fmaf(g * s, (1.f - s) * d, s);
    }
}

// f with the activation as a constant.
template <typename F>
__device__ __forceinline__ void with_activation(int act, F f) {
    if (act == HASTE_ACT_SILU) f(std::integral_constant<int, HASTE_ACT_SILU>());
    else if (act == HASTE_ACT_GELU) f(std::integral_constant<int, HASTE_ACT_GELU>());
    else f(std::integral_constant<int, HASTE_ACT_GELU_TANH>());
}

// 4 F columns side by side, the first `count` of them.
template <int DT, int F>
__device__ __forceinline__ void put_columns(void* p, int64_t at, const f32x4 (&v)[F], int64_t count) {
    constexpr int V = DT == HASTE_DTYPE_F32 || F == 1 ? 4 : 8;
#pragma unroll
    for (int k = 0; k < 4 * F; k += V) {
        float f[V];
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = v[(k + e) / 4][e % 4];
        store_part<DT, V>(p, at + k, pack<DT, V>(f), count - k);
    }
}

// fp32 as three bf16 parts, the rest rounded to nearest each time (gemm.hpp).  What is not finite is its
// own first part; what would round to infinity is cut instead.
__device__ __forceinline__ void split_f32(float a, uint32_t (&u)[3]) {
    u[0] = f32_to_bf16_rne(a);
    const uint32_t bits = __float_as_uint(a);
    const bool finite = (bits & 0x7F800000u) != 0x7F800000u;
    if (finite && (u[0] & 0x7FFFu) == 0x7F80u) u[0] = bits >> 16;
    const float r = finite ? a - bf16_bits_to_f32(u[0]) : 0.f;
    u[1] = f32_to_bf16_rne(r);
    u[2] = f32_to_bf16_rne(r - bf16_bits_to_f32(u[1]));
}
// 4 F columns of a matrix that is an operand of the next product: of its type, or three parts.
template <int DT, int F>
__device__ __forceinline__ void put_operand(void* p, int64_t plane, int64_t at, const f32x4 (&v)[F]) {
    if constexpr (DT == HASTE_DTYPE_F32) {
        uint32_t w[3][2 * F];
#pragma unroll
        for (int k = 0; k < 2 * F; ++k) {
            uint32_t lo[3], hi[3];
            split_f32(v[k / 2][k % 2 * 2], lo);
            split_f32(v[k / 2][k % 2 * 2 + 1], hi);
#pragma unroll
            for (int i = 0; i < 3; ++i) w[i][k] = lo[i] | hi[i] << 16;
        }
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            char* to = static_cast<char*>(p) + i * plane + at * 2;
#pragma unroll
            for (int k = 0; k < 2 * F; k += 2)
                *reinterpret_cast<u32x2*>(to + 4 * k) = u32x2{w[i][k], w[i][k + 1]};
        }
    } else {
        put_columns<DT, F>(p, at, v, 4 * F);
    }
}

// What the forward keeps for the backward, s = u act'(g) and a = act(g): fp32, or for 16-bit matrices its
// upper 24 bits (15 of mantissa), rounded to nearest.  16 bits would add two roundings of the type's
// to the gradients, which have two that cannot be helped (dg and du as the matrix instructions take
// them, and their own): 3.1e-3 off in norm for bf16 instead of 2.3e-3.
//
// Blocks of 16 rows x 64 columns, laid out for whole lines a load of a wave: 16-byte pieces of 8
// columns' upper 16 bits (fp32: of 4 columns), rows side by side, then 16-byte pieces of 16 columns' next 8
// bits; s, then a.
template <int DT>
constexpr int kKeptBlock = 16 * 64 * (DT == HASTE_DTYPE_F32 ? 4 : 3);
struct KeptPlace {
    void* p;
    int64_t blocks;  // to a row of blocks
    template <int DT>
    __device__ __forceinline__ char* block(int64_t m, int n) const {
        return static_cast<char*>(p) + ((m >> 4) * blocks + (n >> 6)) * (2 * kKeptBlock<DT>);
    }
};
// 4 F columns from n (a multiple of 4 F) of row m, F at most 2.
template <int DT, int F>
__device__ __forceinline__ void put_kept(char* block, int64_t m, int n, const f32x4 (&v)[F]) {
    static_assert(F <= 2, "a piece at most");
    const int r = (int)(m & 15), c = n & 63;
    if constexpr (DT == HASTE_DTYPE_F32) {
#pragma unroll
        for (int k = 0; k < F; ++k)
            *reinterpret_cast<f32x4*>(block + ((c / 4 + k) * 16 + r) * 16) = v[k];
    } else {
        uint32_t hi[2 * F], lo[F];
#pragma unroll
        for (int k = 0; k < F; ++k) {
            uint32_t b[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) b[e] = __float_as_uint(v[k][e]) + 0x80u;
            hi[2 * k] = __builtin_amdgcn_perm(b[1], b[0], 0x07060302u);
            hi[2 * k + 1] = __builtin_amdgcn_perm(b[3], b[2], 0x07060302u);
            lo[k] = __builtin_amdgcn_perm(b[1], b[0], 0x0C0C0501u) |
                    __builtin_amdgcn_perm(b[3], b[2], 0x05010C0Cu);
        }
        char* to_hi = block + ((c / 8) * 16 + r) * 16 + (c & 7) * 2;
        char* to_lo = block + 2048 + ((c / 16) * 16 + r) * 16 + (c & 15);
        if constexpr (F == 2) {
            *reinterpret_cast<u32x4*>(to_hi) = u32x4{hi[0], hi[1], hi[2], hi[3]};
            *reinterpret_cast<u32x2*>(to_lo) = u32x2{lo[0], lo[1]};
        } else {
            *reinterpret_cast<u32x2*>(to_hi) = u32x2{hi[0], hi[1]};
            *reinterpret_cast<uint32_t*>(to_lo) = lo[0];
        }
    }
}
// Sixteen columns from n (a multiple of 16).
template <int DT>
struct Kept {
    u32x4 w[DT == HASTE_DTYPE_F32 ? 4 : 3];
};
template <int DT>
__device__ __forceinline__ Kept<DT> load_kept(const char* block, int64_t m, int n) {
    const int r = (int)(m & 15), c = n & 63;
    Kept<DT> k;
    if constexpr (DT == HASTE_DTYPE_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            k.w[i] = *reinterpret_cast<const u32x4*>(block + ((c / 4 + i) * 16 + r) * 16);
    } else {
        k.w[0] = *reinterpret_cast<const u32x4*>(block + ((c / 8) * 16 + r) * 16);
        k.w[1] = *reinterpret_cast<const u32x4*>(block + ((c / 8 + 1) * 16 + r) * 16);
        k.w[2] = *reinterpret_cast<const u32x4*>(block + 2048 + ((c / 16) * 16 + r) * 16);
    }
    return k;
}
// Columns 4 j .. 4 j + 3 of them.
template <int DT>
__device__ __forceinline__ f32x4 kept_columns(const Kept<DT>& k, int j) {
    if constexpr (DT == HASTE_DTYPE_F32) return __builtin_bit_cast(f32x4, k.w[j]);
    const uint32_t h0 = k.w[j / 2][j % 2 * 2], h1 = k.w[j / 2][j % 2 * 2 + 1], lo = k.w[2][j];
    return f32x4{__uint_as_float(__builtin_amdgcn_perm(h0, lo, 0x0504000Cu)),
                 __uint_as_float(__builtin_amdgcn_perm(h0, lo, 0x0706010Cu)),
                 __uint_as_float(__builtin_amdgcn_perm(h1, lo, 0x0504020Cu)),
                 __uint_as_float(__builtin_amdgcn_perm(h1, lo, 0x0706030Cu))};
}

// Columns n and on, those from H on as zeros.  They come out of products with zeros, but a row with an infinity
// makes those NaN, and the next product would take that to all of the row.
template <int F>
__device__ __forceinline__ void zero_from(f32x4 (&v)[F], int n, int H) {
    if (n + 4 * F <= H) return;
#pragma unroll
    for (int k = 0; k < F; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[k][e] = n + 4 * k + e < H ? v[k][e] : 0.f;
}

// Columns n (a multiple of 4 F) and on of row m: h, and s and a where the backward will want them.  Rows of
// h are ld apart, a multiple of 16 that holds them; columns from H on come out as zeros.
struct GatedOut {
    KeptPlace kept;
    void* h;
    int64_t ld, plane;
    int H;
    template <int DT, int ACT, int F>
    __device__ __forceinline__ void put(int64_t m, int n, const f32x4 (&vg)[F], const f32x4 (&vu)[F]) const {
        f32x4 vh[F], vs[F], va[F];
#pragma unroll
        for (int k = 0; k < F; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float a, s;
                activation<ACT, DT == HASTE_DTYPE_F32>(vg[k][e], &a, &s);
                va[k][e] = a;
                vs[k][e] = s * vu[k][e];
                vh[k][e] = a * vu[k][e];
            }
        zero_from<F>(vh, n, H);
        put_operand<DT, F>(h, plane, m * ld + n, vh);
        if (!kept.p) return;
        char* block = kept.template block<DT>(m, n);
        put_kept<DT, F>(block, m, n, vs);
        put_kept<DT, F>(block + kKeptBlock<DT>, m, n, va);
    }
};
// dg and du from dh and what the forward kept.
struct GatedGrad {
    KeptPlace kept;
    void *dg, *du;
    int64_t ld, plane;
    int H;
    template <int DT, int F>
    __device__ __forceinline__ void put(int64_t m, int n, const f32x4 (&dh)[F], const Kept<DT>& s,
                                        const Kept<DT>& a) const {
        f32x4 v[F];
#pragma unroll
        for (int k = 0; k < F; ++k) v[k] = dh[k] * kept_columns<DT>(s, k);
        zero_from<F>(v, n, H);
        put_operand<DT, F>(dg, plane, m * ld + n, v);
#pragma unroll
        for (int k = 0; k < F; ++k) v[k] = dh[k] * kept_columns<DT>(a, k);
        zero_from<F>(v, n, H);
        put_operand<DT, F>(du, plane, m * ld + n, v);
    }
};

// A product's result: C's rows, or where K is split fp32 parts [split][product][M][ceil16(N)].
struct PlainOut {
    void* c[2];
    int64_t ld;
    float* parts;
    int M, N, batches;
    __host__ __device__ int64_t pitch() const { return (N + 15) / 16 * 16; }
    template <int DT, int F>
    __device__ __forceinline__ void put(int split, int batch, int64_t m, int n, const f32x4 (&v)[F]) const {
        if (parts)
            put_columns<HASTE_DTYPE_F32, F>(parts,
                                            (((int64_t)split * batches + batch) * M + m) * pitch() + n, v, 4 * F);
        else
            put_columns<DT, F>(c[batch], m * ld + n, v, N - n);
    }
};

// The parts of a split product, summed in order.
template <int DT>
__global__ __launch_bounds__(256) void sum_parts_kernel(PlainOut o, int splits) {
    const int64_t pitch4 = o.pitch() / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)o.batches * o.M * pitch4) return;
    const f32x4* p = reinterpret_cast<const f32x4*>(o.parts);
    const int64_t step = (int64_t)o.batches * o.M * pitch4;
    f32x4 s[1] = {p[i]};
    for (int k = 1; k < splits; ++k) s[0] += p[i + k * step];
    const int64_t row = i / pitch4, n = i % pitch4 * 4;
    const float f[4] = {s[0][0], s[0][1], s[0][2], s[0][3]};
    store_part<DT, 4>(o.c[row / o.M], row % o.M * o.ld + n, pack<DT, 4>(f), o.N - n);
}

}  // namespace haste
