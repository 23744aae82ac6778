// The norm of many gradients, and AdamW steps of many tensors with states in 32 or in 8 bits.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "elements.hpp"

namespace haste {
namespace {

constexpr int kBlock = 128;    // elements of an 8-bit state that share a scale
constexpr int kMaxSegs = 64;   // tensors of one launch: a lane to each when a wave looks its own up,
                               // and their table stays within 4 KB of kernel arguments
constexpr int kThreads = 256;
constexpr int kPiece = kThreads * 8;  // elements of a workgroup (two such pieces take the same)

struct AdamSeg {
    void* w;
    const void* g;
    void* m;
    void* v;
    uint8_t* ms;
    uint8_t* vs;
    uint64_t n_stream;  // elements, and the tensor's stream << 40
};
struct AdamBatch {
    uint32_t blk0[kMaxSegs];  // first workgroup of each tensor
    AdamSeg s[kMaxSegs];
    int32_t count;
};
struct AdamArgs {
    float b1, c1, b2, c2;  // beta1, 1 - beta1, beta2, 1 - beta2
    float lr_wd, lr, rcorr, eps;  // lr wd, lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t)
    uint32_t k0, k1;
    int32_t do_sr;
    uint32_t blk0;  // first workgroup of the launch among those of its tensors
    const float* grad_scale;
};

// 200 tensors fill 4 KB of kernel arguments.
constexpr int kMaxGrads = 200;
struct GradBatch {
    uint32_t piece0[kMaxGrads];   // first piece of each tensor
    const void* g[kMaxGrads];
    uint64_t n_dtype[kMaxGrads];  // elements, and the dtype << 56
    int32_t count, pieces;
};

// The tensor that workgroup `blk` belongs to: every lane compares one start.
__device__ __forceinline__ int find_seg(const AdamBatch& b, uint32_t blk) {
    const int lane = threadIdx.x & 63;
    const bool at = lane < b.count && b.blk0[lane] <= blk;
    return __builtin_amdgcn_readfirstlane(__popcll(__ballot(at)) - 1);
}

// The four words of Philox4x32-10 (philox_w0's function).
__device__ __forceinline__ u32x4 philox_words(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t k0,
                                              uint32_t k1) {
    uint32_t c3 = 0u;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
        c0 = __builtin_amdgcn_bitop3_b32((uint32_t)(p1 >> 32), c1, k0, 0x96);
        c2 = __builtin_amdgcn_bitop3_b32((uint32_t)(p0 >> 32), c3, k1, 0x96);
        c1 = (uint32_t)p1;
        c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return u32x4{c0, c1, c2, c3};
}

// w as fp16, rounded by the 16 bits r: |w| in units of its spacing (10 mantissa bits, smallest
// normal 2^-14) plus the upper 13 bits of r over 2^13, cut to a whole number.
__device__ __forceinline__ uint32_t sr_f16(float w, uint32_t r) {
    const uint32_t e = max(__float_as_uint(w) & 0x7F800000u, (uint32_t)(127 - 14) << 23);
    const float unit = __uint_as_float(e - (10u << 23));
    const float t = floorf(fabsf(w) * __uint_as_float((264u << 23) - e) + (float)(r >> 3) * 0x1p-13f);
    return f32_to_f16_rne(fabsf(w) < 65536.f ? copysignf(t * unit, w) : w);
}

template <int C>
__device__ __forceinline__ uint32_t dpp_max(uint32_t x) {
    return max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, C, 0xF, 0xF, true));
}
// The maximum over the 16 lanes of a row, in all of them (rotations by 8, 4, 2 and 1).
__device__ __forceinline__ uint32_t row_max(uint32_t x) {
    return dpp_max<0x121>(dpp_max<0x122>(dpp_max<0x124>(dpp_max<0x128>(x))));
}

constexpr uint32_t kInfBits = 0x7F800000u;

// The largest |x| of a row as a bit pattern, at or above kInfBits where not all are finite: of |x| as
// whole numbers, whose order is theirs with infinities and NaN above, or by v_maximum3_f32, which
// takes |x| and passes NaN on.  FINITE leaves those out.
template <bool FINITE>
__device__ __forceinline__ uint32_t row_top(const float* x) {
    uint32_t top = 0;
    if constexpr (FINITE) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t a = __float_as_uint(x[e]) & 0x7FFFFFFFu;
            top = max(top, a >= kInfBits ? 0u : a);
        }
    } else {
        float t = fabsf(x[0]);
#pragma unroll
        for (int e = 1; e < 8; ++e) t = __builtin_elementwise_maximum(t, fabsf(x[e]));
        top = __float_as_uint(t) & 0x7FFFFFFFu;
    }
    return row_max(top);
}

// The E8M0 code of the power of two that puts what has these bits in [128, 256).
__device__ __forceinline__ uint32_t scale_code(uint32_t top) {
    return (uint32_t)max((int)(top >> 23) - 7, 1);
}

__device__ __forceinline__ float pow2_code(uint32_t code) { return __uint_as_float(code << 23); }

// Eight m and u as e4m3 codes under the scales of cm and cu, m[e] rounded up by the upper half of
// r[e] and u[e] by that of its quad's next: v_cvt_sr_fp8_f32 adds the seed's upper 20 bits to what
// it cuts off, subnormals included, and makes NaN of what is not finite.  u > 0 (a root: 2^-63 at
// least) does not become 0.
__device__ __forceinline__ void cut_e4m3(const float* m, const float* u, uint32_t cm, uint32_t cu,
                                         const uint32_t* r, bool finite, u32x2& m8, u32x2& u8) {
    const float im = pow2_code(254u - cm), iu = pow2_code(254u - cu);
    int out[4] = {0, 0, 0, 0};
    float sm[8], su[8];
    int seed[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        sm[e] = m[e] * im;
        su[e] = __builtin_amdgcn_fmed3f(u[e] * iu, 0x1p-9f, u[e] * 0x1p100f);
        seed[e] = (int)(r[e] & 0xFFFF0000u);
    }
    if (!finite) {  // the median of a NaN is not one
#pragma unroll
        for (int e = 0; e < 8; ++e) su[e] = u[e] == u[e] ? su[e] : u[e];
    }
#define HASTE_CUT(E)                                                                          \
    out[0] = __builtin_amdgcn_cvt_sr_fp8_f32(sm[E], seed[E], out[0], E);                      \
    out[1] = __builtin_amdgcn_cvt_sr_fp8_f32(sm[4 + E], seed[4 + E], out[1], E);              \
    out[2] = __builtin_amdgcn_cvt_sr_fp8_f32(su[E], seed[(E + 1) & 3], out[2], E);            \
    out[3] = __builtin_amdgcn_cvt_sr_fp8_f32(su[4 + E], seed[4 + ((E + 1) & 3)], out[3], E)
    HASTE_CUT(0);
    HASTE_CUT(1);
    HASTE_CUT(2);
    HASTE_CUT(3);
#undef HASTE_CUT
    m8 = u32x2{(uint32_t)out[0], (uint32_t)out[1]};
    u8 = u32x2{(uint32_t)out[2], (uint32_t)out[3]};
}

__device__ __forceinline__ void from_e4m3(u32x2 c, float* f) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[h], false);
        const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[h], true);
        f[4 * h] = lo[0];
        f[4 * h + 1] = lo[1];
        f[4 * h + 2] = hi[0];
        f[4 * h + 3] = hi[1];
    }
}

// w' = w - t, t = lr wd w + lr m / (u rcorr + eps), u = sqrt(v'): lr wd keeps its own 24 bits, where
// a factor 1 - lr wd would keep what is left of them beside 1 (7 for lr wd = 1e-5).  The hardware's
// root and reciprocal are within 1 ulp and take what is below 2^-126 for 0.  An infinite w counts
// in t as the largest finite one, so that w - t stays infinite (inf - inf and inf * 0 are not).
__device__ __forceinline__ float adam_change(float w, float m, float u, const AdamArgs& a) {
    w = __builtin_amdgcn_fmed3f(w, -__FLT_MAX__, __FLT_MAX__);
    return __builtin_fmaf(w, a.lr_wd, a.lr * m * __builtin_amdgcn_rcpf(u * a.rcorr + a.eps));
}

// Four differences w - t cut towards zero, as a draw added to their lower bits needs them: rounded
// to the nearest, one value in 2^18 would go the other way than the exact difference, by a whole
// place of 16 bits.  Mode bits 0-1 are fp32's rounding: 3 towards zero, 0 to the nearest.  The
// nearest's rest tested for its sign instead takes 5 instructions a weight: 670 M weights with 8-bit
// states 1314 us, 1299 so, 1292 with no cut.
__device__ __forceinline__ void sub4_towards_zero(float* w, const float* t) {
    asm("s_setreg_imm32_b32 hwreg(HW_REG_MODE, 0, 2), 3\n\t"
        "v_sub_f32 %0, %0, %4\n\t"
        "v_sub_f32 %1, %1, %5\n\t"
        "v_sub_f32 %2, %2, %6\n\t"
        "v_sub_f32 %3, %3, %7\n\t"
        "s_setreg_imm32_b32 hwreg(HW_REG_MODE, 0, 2), 0"
        : "+&v"(w[0]), "+&v"(w[1]), "+&v"(w[2]), "+&v"(w[3])  // (written before all of t is read)
        : "v"(t[0]), "v"(t[1]), "v"(t[2]), "v"(t[3]));
}

// CHECK: w may be a NaN with payload bits in its lower half, which adding to could carry over.
template <int WT, bool CHECK = true>
__device__ __forceinline__ uint32_t sr_pair(float lo, float hi, uint32_t r_lo, uint32_t r_hi) {
    r_lo &= 0xFFFFu;
    r_hi &= 0xFFFFu;
    if constexpr (WT == HASTE_DTYPE_BF16 && !CHECK)
        return __builtin_amdgcn_perm(__float_as_uint(hi) + r_hi, __float_as_uint(lo) + r_lo,
                                     0x07060302u);
    return WT == HASTE_DTYPE_BF16 ? sr_bf16(lo, r_lo) | sr_bf16(hi, r_hi) << 16
                                  : sr_f16(lo, r_lo) | sr_f16(hi, r_hi) << 16;
}

// 32-bit states: a thread has two runs of four elements, half a workgroup's apart, so that every
// 16-byte access of fp32 is next to its neighbour lane's and lines are met whole.  A Philox call
// serves eight elements, which two threads make each for itself.
template <int WT, int GT>
struct AdamElems32 {
    static constexpr int kRun = kThreads * 4;
    Elems<WT, 4> w[2];
    Elems<GT, 4> g[2];
    Elems<HASTE_DTYPE_F32, 4> m[2], v[2];

    // FULL: all of the workgroup's elements are the tensor's; else those below n are.
    template <bool FULL>
    __device__ __forceinline__ void fetch(const AdamSeg& s, int64_t piece, int64_t n) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int64_t i = piece + k * kRun + threadIdx.x * 4;
            if constexpr (FULL) {
                w[k] = load<WT, 4, true>(s.w, i);
                g[k] = load<GT, 4, true>(s.g, i);
                m[k] = load<HASTE_DTYPE_F32, 4, true>(s.m, i);
                v[k] = load<HASTE_DTYPE_F32, 4, true>(s.v, i);
            } else {
                w[k] = load_part<WT, 4>(s.w, i, n - i);
                g[k] = load_part<GT, 4>(s.g, i, n - i);
                m[k] = load_part<HASTE_DTYPE_F32, 4>(s.m, i, n - i);
                v[k] = load_part<HASTE_DTYPE_F32, 4>(s.v, i, n - i);
            }
        }
    }

    template <bool FULL>
    __device__ __forceinline__ void step(const AdamSeg& s, const AdamArgs& a, float gs,
                                         int64_t piece, int64_t n) const {
        const uint32_t stream = (uint32_t)(s.n_stream >> 40);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int64_t i = piece + k * kRun + threadIdx.x * 4;
            float wf[4], gf[4], mf[4], vf[4], tf[4];
            unpack<WT, 4>(w[k], wf);
            unpack<GT, 4>(g[k], gf);
            unpack<HASTE_DTYPE_F32, 4>(m[k], mf);
            unpack<HASTE_DTYPE_F32, 4>(v[k], vf);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                gf[e] *= gs;
                mf[e] = a.b1 * mf[e] + a.c1 * gf[e];
                vf[e] = a.b2 * vf[e] + a.c2 * gf[e] * gf[e];
                tf[e] = adam_change(wf[e], mf[e], __builtin_amdgcn_sqrtf(vf[e]), a);
            }
            Elems<WT, 4> out;
            if (WT != HASTE_DTYPE_F32 && a.do_sr) {
                sub4_towards_zero(wf, tf);
                const uint64_t c = (uint64_t)i / 8;
                const u32x4 q = philox_words((uint32_t)c, (uint32_t)(c >> 32), stream, a.k0, a.k1);
                const uint32_t r0 = i & 4 ? q[2] : q[0], r1 = i & 4 ? q[3] : q[1];
                out.q[0] = sr_pair<WT>(wf[0], wf[1], r0, r0 >> 16);
                out.q[1] = sr_pair<WT>(wf[2], wf[3], r1, r1 >> 16);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) wf[e] -= tf[e];
                out = pack<WT, 4>(wf);
            }
            const Elems<HASTE_DTYPE_F32, 4> mo = pack<HASTE_DTYPE_F32, 4>(mf),
                                          vo = pack<HASTE_DTYPE_F32, 4>(vf);
            if constexpr (FULL) {
                store<WT, 4, true>(s.w, i, out);
                store<HASTE_DTYPE_F32, 4, true>(s.m, i, mo);
                store<HASTE_DTYPE_F32, 4, true>(s.v, i, vo);
            } else {
                store_part<WT, 4>(s.w, i, out, n - i);
                store_part<HASTE_DTYPE_F32, 4>(s.m, i, mo, n - i);
                store_part<HASTE_DTYPE_F32, 4>(s.v, i, vo, n - i);
            }
        }
    }
};

// The root of x to the nearest: the estimate s is within 1 ulp, and kept unless x is past the middle
// between it and a neighbour.
__device__ __forceinline__ float root(float x) {
    const float s = __builtin_amdgcn_sqrtf(x);
    const float lo = __uint_as_float(__float_as_uint(s) - 1u),
                hi = __uint_as_float(__float_as_uint(s) + 1u);
    const float up = __builtin_fmaf(-hi, s, x) > 0.f ? hi : s;
    return __builtin_fmaf(-lo, s, x) <= 0.f ? lo : up;
}

// m' and v' of 8-bit states (u = sqrt(v)), each operation rounded for itself: a rounding more or less
// moves a block's scale where its largest value meets a power of two, as m' does wherever m and g
// are the same one (bf16 gradients and e4m3 codes have few mantissas).
__device__ __forceinline__ void moments8(float* m, float* u, const float* g, float fm, float su,
                                         const AdamArgs& a) {
#pragma clang fp contract(off)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        m[e] = m[e] * fm + g[e] * a.c1;
        u[e] *= su;
        u[e] = u[e] * u[e] * a.b2 + g[e] * g[e] * a.c2;
    }
}

// 8-bit states: a thread has eight elements, so 16 lanes (one DPP row) a block of 128, whose
// maxima need no LDS.  The states are padded to whole blocks.
template <int WT, int GT>
struct AdamElems8 {
    Elems<WT, 8> w;
    Elems<GT, 8> g;
    u32x2 m, u;
    uint32_t ms, us;

    template <bool FULL>
    __device__ __forceinline__ void fetch(const AdamSeg& s, int64_t piece, int64_t n) {
        const int64_t i = piece + threadIdx.x * 8;
        if constexpr (FULL) {
            w = load<WT, 8, WT != HASTE_DTYPE_F32>(s.w, i);
            g = load<GT, 8, GT != HASTE_DTYPE_F32>(s.g, i);
        } else {
            w = load_part<WT, 8>(s.w, i, n - i);
            g = load_part<GT, 8>(s.g, i, n - i);
        }
        m = u = u32x2{0, 0};
        ms = us = 127;
        if (FULL || i < n) {
            const u32x2* mp = reinterpret_cast<const u32x2*>(static_cast<uint8_t*>(s.m) + i);
            const u32x2* up = reinterpret_cast<const u32x2*>(static_cast<uint8_t*>(s.v) + i);
            m = __builtin_nontemporal_load(mp);
            u = __builtin_nontemporal_load(up);
            ms = s.ms[i / kBlock];
            us = s.vs[i / kBlock];
        }
    }

    template <bool FULL>
    __device__ __forceinline__ void step(const AdamSeg& s, const AdamArgs& a, float gs,
                                         int64_t piece, int64_t n) const {
        const int64_t i = piece + threadIdx.x * 8;
        float wf[8], gf[8], mf[8], uf[8], tf[8];
        unpack<WT, 8>(w, wf);
        unpack<GT, 8>(g, gf);
        from_e4m3(m, mf);
        from_e4m3(u, uf);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (!FULL && i + e >= n) mf[e] = uf[e] = 0.f;
            gf[e] *= gs;
        }
        moments8(mf, uf, gf, a.b1 * pow2_code(ms), pow2_code(us), a);
        uint32_t tm = row_top<false>(mf), tv = row_top<false>(uf);
        const bool finite = !__any(max(tm, tv) >= kInfBits);
        if (!finite) {
            tm = row_top<true>(mf);
            tv = row_top<true>(uf);
        }
        // (the largest root's scale needs it to the last place, the roots themselves do not)
        const uint32_t cm = scale_code(tm),
                       cu = scale_code(__float_as_uint(root(__uint_as_float(tv))));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            uf[e] = __builtin_amdgcn_sqrtf(uf[e]);
            tf[e] = adam_change(wf[e], mf[e], uf[e], a);
        }
        const uint32_t stream = (uint32_t)(s.n_stream >> 40);
        const uint64_t c = (uint64_t)i / 4;
        const u32x4 q0 = philox_words((uint32_t)c, (uint32_t)(c >> 32), stream, a.k0, a.k1);
        const u32x4 q1 = philox_words((uint32_t)c + 1, (uint32_t)(c >> 32), stream, a.k0, a.k1);
        const uint32_t r[8] = {q0[0], q0[1], q0[2], q0[3], q1[0], q1[1], q1[2], q1[3]};
        Elems<WT, 8> out;
        if (WT != HASTE_DTYPE_F32 && a.do_sr) {
            sub4_towards_zero(wf, tf);
            sub4_towards_zero(wf + 4, tf + 4);
            // (where m and u are finite only a NaN of w itself is left, whose payload is w's)
            if (finite) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    out.q[e] = sr_pair<WT, false>(wf[2 * e], wf[2 * e + 1], r[2 * e], r[2 * e + 1]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    out.q[e] = sr_pair<WT>(wf[2 * e], wf[2 * e + 1], r[2 * e], r[2 * e + 1]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) wf[e] -= tf[e];
            out = pack<WT, 8>(wf);
        }
        if constexpr (FULL) store<WT, 8, WT != HASTE_DTYPE_F32>(s.w, i, out);
        else store_part<WT, 8>(s.w, i, out, n - i);
        u32x2 mo, uo;
        cut_e4m3(mf, uf, cm, cu, r, finite, mo, uo);
        if (FULL || (i & ~(int64_t)(kBlock - 1)) < n) {
            u32x2* mp = reinterpret_cast<u32x2*>(static_cast<uint8_t*>(s.m) + i);
            u32x2* up = reinterpret_cast<u32x2*>(static_cast<uint8_t*>(s.v) + i);
            __builtin_nontemporal_store(mo, mp);
            __builtin_nontemporal_store(uo, up);
            if ((threadIdx.x & 15) == 0) {
                s.ms[i / kBlock] = (uint8_t)cm;
                s.vs[i / kBlock] = (uint8_t)cu;
            }
        }
    }
};

// Every byte is met once, and HBM bounds it.  32-bit states: 91 M bf16 weights of 195 tensors take
// 298 us for 2.0 GB, 6.7 TB/s with the gradients that the norm before has left in the last-level
// cache.  8-bit states: 670 M weights take 1051 us for 6.7 GB, 6.4 TB/s, at 49 vector instructions
// an element (10 of them Philox), which keep the vector units 88 % busy; at 55 it took 1068.  All
// accesses are non-temporal (but 8-wide ones of fp32, of which each touches half a line), so that
// what is met once and dirty lines do not drive those gradients out: with the norm, 8-bit
// 221 -> 188 us and 1497 -> 1350, 32-bit 424 -> 345.
template <int WT, int GT, bool Q8>
__global__ __launch_bounds__(kThreads) void adamw_kernel(const AdamBatch b, const AdamArgs a) {
    using Elems = std::conditional_t<Q8, AdamElems8<WT, GT>, AdamElems32<WT, GT>>;
    float gs = 1.f;
    if (a.grad_scale) {
        gs = *a.grad_scale;
        if (gs != gs) return;
    }
    const uint32_t blk = a.blk0 + blockIdx.x;
    const int t = find_seg(b, blk);
    const AdamSeg& s = b.s[t];
    const int64_t n = (int64_t)(s.n_stream & 0xFFFFFFFFFFull);
    const int64_t i0 = (int64_t)(blk - b.blk0[t]) * kPiece;
    Elems x;
    if (i0 + kPiece <= n) {
        x.template fetch<true>(s, i0, n);
        x.template step<true>(s, a, gs, i0, n);
    } else {
        x.template fetch<false>(s, i0, n);
        x.template step<false>(s, a, gs, i0, n);
    }
}

constexpr int kNormThreads = 256;
constexpr int kNormLoads = 8;                                  // 16-byte (fp32: 32) loads in flight
constexpr int kNormPiece = kNormThreads * 8 * kNormLoads;      // elements of a piece
constexpr int kNormParts = 1024;                               // workgroups of a launch, 4 to a CU

__device__ __forceinline__ double wave_sum(double v) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// This thread's share of the squares of elements i0 .. i0 + kNormPiece of n, in fp64.
template <int DT>
__device__ __forceinline__ double piece_squares64(const void* g, int64_t i0, int64_t n) {
    double sum = 0.0;
    float f[8];
    for (int k = 0; k < kNormLoads; ++k) {
        const int64_t at = i0 + threadIdx.x * 8 + k * (kNormThreads * 8);
        if (at >= n) break;
        unpack<DT, 8>(load_part<DT, 8>(g, at, n - at), f);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += (double)f[e] * f[e];
    }
    return sum;
}

// The same in fp32, four sums side by side, unless that overflows or is so small that squares may
// have lost bits below 2^-149 (64 such losses are at most 2^-44 of a sum from 2^-100 on).
template <int DT>
__device__ __forceinline__ double piece_squares(const void* g, int64_t i0, int64_t n) {
    float sum[4] = {0.f, 0.f, 0.f, 0.f}, f[8];
    uint32_t any = 0;
    auto add = [&](const Elems<DT, 8>& x) __attribute__((always_inline)) {
        unpack<DT, 8>(x, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e & 3] += f[e] * f[e];
#pragma unroll
        for (uint32_t q : x.q) any |= q;
    };
    const int64_t i = i0 + threadIdx.x * 8;
    if (i0 + kNormPiece <= n) {
        Elems<DT, 8> x[kNormLoads];
#pragma unroll
        for (int k = 0; k < kNormLoads; ++k) x[k] = load<DT, 8>(g, i + k * (kNormThreads * 8));
#pragma unroll
        for (int k = 0; k < kNormLoads; ++k) add(x[k]);
    } else {
        for (int k = 0; k < kNormLoads; ++k) {
            const int64_t at = i + k * (kNormThreads * 8);
            if (at >= n) break;
            add(load_part<DT, 8>(g, at, n - at));
        }
    }
    const float s = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    if (any == 0 || (s >= 0x1p-100f && s < INFINITY)) return s;
    return piece_squares64<DT>(g, i0, n);
}

// part[workgroup] = the sum of squares of every gridDim-th piece, the launch's last pieces first:
// the first tensors' gradients are then what the last-level cache holds when a step reads them
// again from the start.  Bound by HBM: 1.34 GB of bf16 in 223 us, 6.0 TB/s; 182 MB of 195
// tensors in 32 us, in one launch (in four of 64 tensors each 60 us).
__global__ __launch_bounds__(kNormThreads) void grad_norm_kernel(const GradBatch b, double* part) {
    __shared__ double sums[kNormThreads / 64];
    __shared__ uint32_t piece0[kMaxGrads];
    for (int k = threadIdx.x; k < b.count; k += kNormThreads) piece0[k] = b.piece0[k];
    __syncthreads();
    const int lane = threadIdx.x & 63;
    double total = 0.0;
    for (int p = b.pieces - 1 - (int)blockIdx.x; p >= 0; p -= (int)gridDim.x) {
        int t = -1;
        for (int k = 0; k < b.count; k += 64)
            t += __popcll(__ballot(k + lane < b.count && piece0[k + lane] <= (uint32_t)p));
        t = __builtin_amdgcn_readfirstlane(t);
        const void* g = b.g[t];
        const int64_t n = (int64_t)(b.n_dtype[t] & 0xFFFFFFFFFFFFFFull);
        const int dtype = (int)(b.n_dtype[t] >> 56);
        const int64_t i0 = (int64_t)((uint32_t)p - b.piece0[t]) * kNormPiece;
        total += dtype == HASTE_DTYPE_BF16  ? piece_squares<HASTE_DTYPE_BF16>(g, i0, n)
                 : dtype == HASTE_DTYPE_F16 ? piece_squares<HASTE_DTYPE_F16>(g, i0, n)
                                            : piece_squares<HASTE_DTYPE_F32>(g, i0, n);
    }
    total = wave_sum(total);
    if (lane == 0) sums[threadIdx.x >> 6] = total;
    __syncthreads();
    if (threadIdx.x) return;
    for (int k = 1; k < kNormThreads / 64; ++k) total += sums[k];
    part[blockIdx.x] = total;
}

constexpr int kFinalThreads = 1024;
__global__ __launch_bounds__(kFinalThreads) void grad_norm_final_kernel(const double* part,
                                                                        int64_t parts,
                                                                        float max_norm, float* out) {
    __shared__ double sums[kFinalThreads / 64];
    double total = 0.0;
    for (int64_t i = threadIdx.x; i < parts; i += kFinalThreads) total += part[i];
    total = wave_sum(total);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = total;
    __syncthreads();
    if (threadIdx.x) return;
    for (int k = 1; k < kFinalThreads / 64; ++k) total += sums[k];
    const float norm = (float)sqrt(total);
    out[0] = norm;
    out[1] = norm < INFINITY ? fminf(1.f, max_norm / (norm + 1e-6f)) : NAN;
}

constexpr int64_t kMostBlocks = (((int64_t)1 << 32) - 1) / kThreads;  // (a launch takes 2^32 - 1 threads)

template <int WT, int GT, bool Q8>
int launch_adamw(const haste_adamw_tensor* ts, int count, AdamArgs a, hipStream_t st) {
    for (int base = 0; base < count;) {
        AdamBatch b;
        b.count = 0;
        int64_t blocks = 0;
        for (; base < count && b.count < kMaxSegs; ++base) {
            const haste_adamw_tensor& t = ts[base];
            if (t.n == 0) continue;
            b.blk0[b.count] = (uint32_t)blocks;
            b.s[b.count++] = AdamSeg{t.w, t.g, t.m, t.v, t.m_scale, t.v_scale,
                                     (uint64_t)t.n | (uint64_t)t.stream << 40};
            blocks += ceil_div(t.n, (int64_t)kPiece);
            HASTE_CHECK_ARG(blocks < (int64_t)1 << 31, "haste_adamw_step: tensors too large");
        }
        if (b.count == 0) break;
        for (int64_t at = 0; at < blocks; at += kMostBlocks) {
            a.blk0 = (uint32_t)at;
            const unsigned grid = (unsigned)std::min(blocks - at, kMostBlocks);
            adamw_kernel<WT, GT, Q8><<<dim3(grid), dim3(kThreads), 0, st>>>(b, a);
            HASTE_CHECK_LAUNCH("haste_adamw_step");
        }
    }
    return HASTE_OK;
}

}  // namespace
}  // namespace haste

extern "C" int haste_adamw_step(const haste_adamw_tensor* tensors, int32_t count, int32_t w_dtype,
                                int32_t g_dtype, int32_t state_bits, double lr, double beta1,
                                double beta2, double eps, double wd, int64_t step, int32_t do_sr,
                                uint64_t seed, const float* grad_scale, void* stream) {
    const char* fn = "haste_adamw_step";
    HASTE_CHECK_ARG(count >= 0 && (count == 0 || tensors != nullptr), "%s: bad tensor list", fn);
    HASTE_CHECK_ARG(haste::elem_dtype(w_dtype) && haste::elem_dtype(g_dtype),
                    "%s: weights and gradients must be bf16, fp16 or fp32 (dtype codes %d, %d)", fn,
                    (int)w_dtype, (int)g_dtype);
    HASTE_CHECK_ARG(state_bits == 8 || state_bits == 32, "%s: states must have 8 or 32 bits (got %d)",
                    fn, (int)state_bits);
    HASTE_CHECK_ARG(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0,
                    "%s: betas must be in [0, 1) and eps >= 0", fn);
    HASTE_CHECK_ARG(step >= 1, "%s: step must be >= 1 (got %lld)", fn, (long long)step);
    HASTE_CHECK_ARG((reinterpret_cast<uintptr_t>(grad_scale) & 3u) == 0, "%s: grad_scale misaligned",
                    fn);
    const bool q8 = state_bits == 8;
    for (int k = 0; k < count; ++k) {
        const haste_adamw_tensor& t = tensors[k];
        HASTE_CHECK_ARG(t.n >= 0 && t.n < (int64_t)1 << 40,
                        "%s: tensor %d: n must be >= 0 and below 2^40", fn, k);
        HASTE_CHECK_ARG(t.stream < 1u << 24, "%s: tensor %d: stream must be below 2^24", fn, k);
        if (t.n == 0) continue;
        HASTE_CHECK_ARG(t.w && t.g && t.m && t.v && (!q8 || (t.m_scale && t.v_scale)),
                        "%s: tensor %d: null pointer", fn, k);
        const uintptr_t st = reinterpret_cast<uintptr_t>(t.m) | reinterpret_cast<uintptr_t>(t.v);
        HASTE_CHECK_ARG(haste::elem_aligned(t.w, w_dtype) && haste::elem_aligned(t.g, g_dtype) &&
                            (st & (q8 ? 7u : 15u)) == 0,
                        "%s: tensor %d is misaligned", fn, k);
    }
    haste::AdamArgs a{};
    a.b1 = (float)beta1;
    a.c1 = (float)(1.0 - beta1);
    a.b2 = (float)beta2;
    a.c2 = (float)(1.0 - beta2);
    a.lr_wd = (float)(lr * wd);
    a.lr = (float)(lr / (1.0 - std::pow(beta1, (double)step)));
    a.rcorr = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step)));
    a.eps = (float)eps;
    a.k0 = (uint32_t)seed;
    a.k1 = (uint32_t)(seed >> 32);
    a.do_sr = do_sr != 0;
    a.grad_scale = grad_scale;
    hipStream_t st = static_cast<hipStream_t>(stream);
#define HASTE_ADAMW(WT, GT)                                                                 \
    if (w_dtype == WT && g_dtype == GT)                                                     \
        return q8 ? haste::launch_adamw<WT, GT, true>(tensors, count, a, st)                \
                  : haste::launch_adamw<WT, GT, false>(tensors, count, a, st)
    HASTE_ADAMW(HASTE_DTYPE_BF16, HASTE_DTYPE_BF16);
    HASTE_ADAMW(HASTE_DTYPE_BF16, HASTE_DTYPE_F16);
    HASTE_ADAMW(HASTE_DTYPE_BF16, HASTE_DTYPE_F32);
    HASTE_ADAMW(HASTE_DTYPE_F16, HASTE_DTYPE_BF16);
    HASTE_ADAMW(HASTE_DTYPE_F16, HASTE_DTYPE_F16);
    HASTE_ADAMW(HASTE_DTYPE_F16, HASTE_DTYPE_F32);
    HASTE_ADAMW(HASTE_DTYPE_F32, HASTE_DTYPE_BF16);
    HASTE_ADAMW(HASTE_DTYPE_F32, HASTE_DTYPE_F16);
    HASTE_ADAMW(HASTE_DTYPE_F32, HASTE_DTYPE_F32);
#undef HASTE_ADAMW
    return HASTE_ERR_UNSUPPORTED;
}

extern "C" int64_t haste_grad_norm_workspace_size(int32_t count) {
    if (count < 0) return HASTE_ERR_INVALID_ARG;
    return haste::ceil_div(std::max(count, 1), haste::kMaxGrads) * haste::kNormParts *
           (int64_t)sizeof(double);
}

extern "C" int haste_grad_norm(const haste_grad_tensor* tensors, int32_t count, double max_norm,
                               float* out, void* ws, int64_t ws_bytes, void* stream) {
    const char* fn = "haste_grad_norm";
    HASTE_CHECK_ARG(count >= 0 && (count == 0 || tensors != nullptr), "%s: bad tensor list", fn);
    HASTE_CHECK_ARG(out != nullptr && (reinterpret_cast<uintptr_t>(out) & 3u) == 0,
                    "%s: out is NULL or misaligned", fn);
    HASTE_CHECK_ARG(max_norm >= 0.0, "%s: max_norm must be >= 0", fn);
    HASTE_CHECK_ARG(ws != nullptr && (reinterpret_cast<uintptr_t>(ws) & 7u) == 0,
                    "%s: workspace is NULL or misaligned", fn);
    if (ws_bytes < haste_grad_norm_workspace_size(count)) {
        haste::set_error("%s: workspace too small (%lld < %lld bytes)", fn, (long long)ws_bytes,
                         (long long)haste_grad_norm_workspace_size(count));
        return HASTE_ERR_WORKSPACE;
    }
    for (int k = 0; k < count; ++k) {
        const haste_grad_tensor& t = tensors[k];
        HASTE_CHECK_ARG(t.n >= 0 && t.n < (int64_t)1 << 44,
                        "%s: tensor %d: n must be >= 0 and below 2^44", fn, k);
        HASTE_CHECK_ARG(haste::elem_dtype(t.dtype),
                        "%s: tensor %d must be bf16, fp16 or fp32 (dtype code %d)", fn, k,
                        (int)t.dtype);
        HASTE_CHECK_ARG(t.n == 0 || (t.g && haste::elem_aligned(t.g, t.dtype)),
                        "%s: tensor %d is NULL or misaligned", fn, k);
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    double* part = static_cast<double*>(ws);
    int64_t parts = 0;
    for (int base = 0; base < count;) {
        haste::GradBatch b;
        b.count = 0;
        int64_t pieces = 0;
        for (; base < count && b.count < haste::kMaxGrads; ++base) {
            const haste_grad_tensor& t = tensors[base];
            if (t.n == 0) continue;
            b.piece0[b.count] = (uint32_t)pieces;
            b.g[b.count] = t.g;
            b.n_dtype[b.count++] = (uint64_t)t.n | (uint64_t)t.dtype << 56;
            pieces += haste::ceil_div(t.n, (int64_t)haste::kNormPiece);
            HASTE_CHECK_ARG(pieces < (int64_t)1 << 30, "%s: tensors too large", fn);
        }
        if (b.count == 0) break;
        b.pieces = (int32_t)pieces;
        const int64_t blocks = std::min<int64_t>(pieces, haste::kNormParts);
        haste::grad_norm_kernel<<<dim3((unsigned)blocks), dim3(haste::kNormThreads), 0, st>>>(
            b, part + parts);
        HASTE_CHECK_LAUNCH(fn);
        parts += blocks;
    }
    haste::grad_norm_final_kernel<<<dim3(1), dim3(haste::kFinalThreads), 0, st>>>(
        part, parts, (float)max_norm, out);
    HASTE_CHECK_LAUNCH(fn);
    return HASTE_OK;
}
