// What the products of the gated feed-forward block do with their sums, for all types:
//   forward   g = x Wg^T, u = x Wu^T, h = act(g) u;  y = h Wd^T
//   backward  dh = dy Wd, dg = dh u act'(g), du = dh act(g);  dx = dg Wg + du Wu,
//             dWg = dg^T x, dWu = du^T x, dWd = dy^T h
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
        const float cdf = 0.5f * erfcf(-0.70710678118654752f * g);
        *a = g * cdf;
        const float e = PRECISE ? expf(-0.5f * g * g)
                                : __builtin_amdgcn_exp2f(-0.72134752044448170f * g * g);
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

template <int DT>
__device__ __forceinline__ void put4(void* p, int64_t at, f32x4 v, int64_t count) {
    const float f[4] = {v[0], v[1], v[2], v[3]};
    store_part<DT, 4>(p, at, pack<DT, 4>(f), count);
}
template <int DT>
__device__ __forceinline__ f32x4 get4(const void* p, int64_t at) {
    float f[4];
    unpack<DT, 4>(load<DT, 4>(p, at), f);
    return f32x4{f[0], f[1], f[2], f[3]};
}

// Four columns from n of row m: h, and g and u where the backward will want them.  Rows of g, u and h are
// ld apart, a multiple of 8 (16-bit) that holds them; columns past the extent come out as zeros.
struct GatedOut {
    void *g, *u, *h;
    int64_t ld;
    template <int DT, int ACT>
    __device__ __forceinline__ void put(int64_t m, int n, f32x4 vg, f32x4 vu) const {
        const int64_t at = m * ld + n, left = ld - n;
        f32x4 vh;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float a, slope;
            activation<ACT, DT == HASTE_DTYPE_F32>(vg[e], &a, &slope);
            vh[e] = a * vu[e];
        }
        if (g) {
            put4<DT>(g, at, vg, left);
            put4<DT>(u, at, vu, left);
        }
        put4<DT>(h, at, vh, left);
    }
};
// dg and du from dh and the forward's g and u.
struct GatedGrad {
    const void *g, *u;
    void *dg, *du;
    int64_t ld;
    template <int DT, int ACT>
    __device__ __forceinline__ void put(int64_t m, int n, f32x4 dh) const {
        const int64_t at = m * ld + n;
        const f32x4 vg = get4<DT>(g, at), vu = get4<DT>(u, at);
        f32x4 a, b;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float act, slope;
            activation<ACT, DT == HASTE_DTYPE_F32>(vg[e], &act, &slope);
            a[e] = dh[e] * vu[e] * slope;
            b[e] = dh[e] * act;
        }
        put4<DT>(dg, at, a, 4);
        put4<DT>(du, at, b, 4);
    }
};

// A product's result: C's rows, or where K is split fp32 parts [split][product][M][ceil4(N)].
struct PlainOut {
    void* c[2];
    int64_t ld;
    float* parts;
    int M, N, batches;
    template <int DT>
    __device__ __forceinline__ void put(int split, int batch, int64_t m, int n, f32x4 v) const {
        if (parts) {
            const int64_t pitch = (N + 3) / 4 * 4;
            *reinterpret_cast<f32x4*>(parts + (((int64_t)split * batches + batch) * M + m) * pitch + n) = v;
        } else {
            put4<DT>(c[batch], m * ld + n, v, N - n);
        }
    }
};

// The parts of a split product, summed in order.
template <int DT>
__global__ __launch_bounds__(256) void sum_parts_kernel(PlainOut o, int splits) {
    const int64_t pitch4 = (o.N + 3) / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)o.batches * o.M * pitch4) return;
    const f32x4* p = reinterpret_cast<const f32x4*>(o.parts);
    const int64_t step = (int64_t)o.batches * o.M * pitch4;
    f32x4 s = p[i];
    for (int k = 1; k < splits; ++k) s += p[i + k * step];
    const int64_t row = i / pitch4, n = i % pitch4 * 4;
    put4<DT>(o.c[row / o.M], row % o.M * o.ld + n, s, o.N - n);
}

}  // namespace haste
