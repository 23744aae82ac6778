// Products of 16-bit matrices with fp32 sums, C[m, n] = sum_k A(m, k) B(n, k), as tiles of BM x BN for
// a workgroup of WM x WN waves, each of which holds FM x FN MFMA tiles of 16 x 16.
//
// fp32 matrices come as three bf16 parts, a = a0 + a1 + a2 (each the rest rounded to nearest, so that
// |a1| <= 2^-9 |a| and |a2| <= 2^-18 |a|), and their product as the six of the parts' products that are not
// under 2^-26 of it: a2 b0 + a0 b2 + a1 b1 + a1 b0 + a0 b1 + a0 b0, one behind the other along K.  Six
// bf16 products take less time than one on the fp32 matrix instructions, whose rate is a sixteenth.
//
// K goes in steps of 32 through four stages of LDS (three where two workgroups of 256 x 128 share it).  Loads
// write LDS straight from memory, all but one of the stages ahead; a wave reads the fragments of step k + 1
// while its MFMAs work on step k, so neither waits for the other, and one barrier a step is enough: the
// stage that is loaded into was last read two steps ago.
//
// Measured in bf16: 16384 x 4096 x 8192 at 1.12 to 1.21 PFLOP/s by operands' order, 65536 x 768 x 2048 at 0.89
// (y) to 1.0 (dWg, dWu).  The matrix units bound the large ones: fed without a pause they draw the card's
// power and its clock falls to 1.7 GHz; a library product of 8192^3 reaches 1.37.  No bank conflicts were
// counted in LDS.
//
// An operand is K-contiguous (element (r, k) at r * ld + k) or R-contiguous (at k * ld + r).  The
// first kind lies in LDS as rows of 32 k's (64 bytes) and is read 16 bytes a lane; the second as
// rows of BM (BN) r's and is read by ds_read_b64_tr_b16, which transposes 4 x 16 elements.  16-byte
// pieces (pairs of them) are permuted within their rows so that the lanes of a read meet all banks: the
// lanes' addresses in memory are permuted, since a load to LDS writes lane after lane.
#pragma once

#include <type_traits>

#include "elements.hpp"

namespace haste {

// Operand rows start on 16 bytes; columns past the extent up to the next multiple of 8 are zero (K) or
// unused (R).
struct GemmOperand {
    const char* base[2];
    int64_t ld;     // elements
    int64_t plane;  // bytes between the parts of an fp32 matrix
};

// PLAIN: one product.  DUAL: the left half of a tile's columns is B's base[0], the right half base[1],
// each of N columns.  SEGMENTS: K is [0, K) of base[0] of both operands, then [0, K) of base[1].
// BATCH: two products, of base[0] and base[1] of A, both with B's base[0].
enum class GemmMode { kPlain, kDual, kSegments, kBatch };

struct GemmArgs {
    GemmOperand a, b;
    int M, N, K;
    int tiles_m, tiles_n;
    int steps;   // steps of 32 of a segment
    int splits;  // the steps are cut evenly into so many parts
};

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

// 64 lanes x 16 bytes from memory to LDS at `lds` (wave-uniform), lane after lane.  Lanes at or past the
// resource's 2 GB write zeros.  Not the builtin: for it the compiler waits for every load in
// flight before each read of LDS.  Nothing waits for this but wait_loads().
__device__ __forceinline__ void load_lds16(const char* base, uint32_t voff, uint32_t lds) {
    const uint64_t p = reinterpret_cast<uint64_t>(base);
    const i32x4 rsrc = {__builtin_amdgcn_readfirstlane((int)(uint32_t)p),
                        __builtin_amdgcn_readfirstlane((int)((uint32_t)(p >> 32) & 0xFFFFu)), 0x7FFFFF00,
                        0x00020000};
    asm volatile(
        "s_mov_b32 m0, %0\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %1, %2, 0 offen lds"
        :
        : "s"(lds), "v"(voff), "s"(rsrc)
        : "memory");
}
// Until at most n such loads of the wave are in flight and its LDS reads are done, then for the workgroup.
template <int n>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(n) : "memory");
}

// The fp32 form's six products: which part of A and of B (two bits each).
constexpr uint32_t kPartsOfA = 2 | 0 << 2 | 1 << 4 | 1 << 6 | 0 << 8 | 0 << 10;
constexpr uint32_t kPartsOfB = 0 | 2 << 2 | 1 << 4 | 0 << 6 | 1 << 8 | 0 << 10;

// T: BF16, F16, or F32Parts.
struct F32Parts {
    static constexpr int code = HASTE_DTYPE_F32;
};

template <typename T, GemmMode MODE, bool AK, bool BK_, int FM_, int FN_, int WM_, int WN_,
          int STAGES>
struct GemmTile {
    static constexpr bool kParts = std::is_same<T, F32Parts>::value;
    static constexpr int kProducts = kParts ? 6 : 1;
    typedef typename std::conditional<kParts, BF16, T>::type M_;
    static constexpr int FM = FM_, FN = FN_, WM = WM_, WN = WN_, kWaves = WM * WN;
    static constexpr int BM = 16 * FM * WM, BN = 16 * FN * WN, KS = 32, kStages = STAGES;
    static constexpr int kThreads = 64 * kWaves;
    static constexpr int kABytes = BM * KS * 2, kBBytes = BN * KS * 2, kStage = kABytes + kBBytes;
    static constexpr int kLdsBytes = kStages * kStage;
    static constexpr int kALoads = BM / 16 / kWaves, kBLoads = BN / 16 / kWaves;
    static constexpr int kLoads = kALoads + kBLoads;
    static constexpr bool kDual = MODE == GemmMode::kDual;
    // columns of C to a tile
    static constexpr int kCols = kDual ? BN / 2 : BN;
    static_assert(BM / 16 % kWaves == 0 && BN / 16 % kWaves == 0, "loads do not divide");
    static_assert(kStages >= 3 && (kStages - 2) * kLoads < 63, "stages");

    f32x4 acc[FN][FM];
    int m0, n0;  // first row and column of the wave's part (DUAL: of either half)

    static __device__ __forceinline__ int stage_of(int kt) { return (int)((uint32_t)kt % kStages); }

    // Where a lane's 16 bytes of load j lie: row and k of their first element within the tile.
    template <bool KC, int R>
    static __device__ __forceinline__ void place(int j, int lane, int* r, int* k) {
        if constexpr (KC) {
            *r = j * 16 + lane / 4;
            *k = 8 * ((lane & 3) ^ ((*r >> 1) & 3));
        } else {
            constexpr int C = R / 8;  // pieces to a row
            const int i = j * 64 + lane, s = i % C;
            *k = i / C;
            const int f = ((*k & 3) | (*k >> 3 & 3) << 2) & (C / 2 - 1);
            *r = 8 * (2 * ((s / 2) ^ f) + (s & 1));
        }
    }

    // Fragment (16 rows from r0) of an operand's stage: lane l has row l % 16, k = 8 (l / 16) + 0..7.
    template <bool KC, int R>
    static __device__ __forceinline__ u32x4 fragment(const char* stage, int r0, int lane) {
        if constexpr (KC) {
            const int r = r0 + (lane & 15);
            return *reinterpret_cast<const u32x4*>(stage + r * 64 +
                                                   (((lane >> 4) ^ ((lane >> 1) & 3)) << 4));
        } else {
            constexpr int C = R / 8;
            const int i = lane & 15, q = lane >> 4;
            const int f = ((i >> 2) | q << 2) & (C / 2 - 1);
            const char* p = stage + (q * 8 + (i >> 2)) * (R * 2) + (((r0 >> 4) ^ f) << 5) + (i & 3) * 8;
            const u32x2 lo = lds_read_tr16(p), hi = lds_read_tr16(p + 4 * R * 2);
            return u32x4{lo[0], lo[1], hi[0], hi[1]};
        }
    }

    __device__ __forceinline__ void run(const GemmArgs& g, char* lds, int tm, int tn, int batch,
                                        int split) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
        const int wm = wave % WM, wn = wave / WM;
        m0 = tm * BM + wm * FM * 16;
        n0 = tn * kCols + wn * (kDual ? FN / 2 : FN) * 16;
        const int all = (MODE == GemmMode::kSegments ? 2 : 1) * kProducts * g.steps;
        const int k0 = __builtin_amdgcn_readfirstlane((int)((int64_t)all * split / g.splits)),
                  k1 = __builtin_amdgcn_readfirstlane((int)((int64_t)all * (split + 1) / g.splits));
        // bytes from a tile's first element
        uint32_t off[kLoads];
        int kpos[kLoads];
        const char *pa[2], *pb[2];
        const int64_t lda = g.a.ld * 2, ldb = g.b.ld * 2;
        const int64_t a0 = AK ? tm * BM * lda : tm * BM * 2, b0 = BK_ ? tn * kCols * ldb : tn * kCols * 2;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int from = MODE == GemmMode::kBatch ? batch : MODE == GemmMode::kPlain ? 0 : x;
            pa[x] = g.a.base[kDual ? 0 : from] + a0;
            pb[x] = g.b.base[MODE == GemmMode::kBatch ? 0 : from] + b0;
        }
#pragma unroll
        for (int j = 0; j < kALoads; ++j) {
            int r, k;
            place<AK, BM>(wave * kALoads + j, lane, &r, &k);
            off[j] = tm * BM + r < g.M ? (uint32_t)(AK ? r * lda + k * 2 : k * lda + r * 2) : kOOB;
            kpos[j] = k;
        }
#pragma unroll
        for (int j = 0; j < kBLoads; ++j) {
            int r, k;
            place<BK_, BN>(wave * kBLoads + j, lane, &r, &k);
            if (kDual) r = r % (BN / 2);
            off[kALoads + j] =
                tn * kCols + r < g.N ? (uint32_t)(BK_ ? r * ldb + k * 2 : k * ldb + r * 2) : kOOB;
            kpos[kALoads + j] = k;
        }
        const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
        // the next step to be loaded: step `k_in` of run `part` over K
        int part = __builtin_amdgcn_readfirstlane(k0 / max(g.steps, 1)), k_in = k0 - part * g.steps;
        auto issue = [&](int kt) __attribute__((always_inline)) {
            const bool second = MODE == GemmMode::kSegments && part >= kProducts;
            const int k = k_in * KS;
            const int left = kt < k1 ? g.K - k : 0;
            const uint32_t to = lds0 + stage_of(kt) * kStage;
            int64_t pa_off = AK ? (int64_t)k * 2 : k * lda, pb_off = BK_ ? (int64_t)k * 2 : k * ldb;
            if (kParts) {
                const int product = second ? part - kProducts : part;
                pa_off += (kPartsOfA >> (2 * product) & 3) * g.a.plane;
                pb_off += (kPartsOfB >> (2 * product) & 3) * g.b.plane;
            }
            const char* a = (second ? pa[1] : pa[0]) + pa_off;
            const char* b = (second ? pb[1] : pb[0]) + pb_off;
            const char* b2 = kDual ? pb[1] + pb_off : b;
            if (++k_in == g.steps) {
                k_in = 0;
                ++part;
            }
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                const bool is_a = j < kALoads;
                const int i = is_a ? wave * kALoads + j : wave * kBLoads + (j - kALoads);
                const char* p = is_a ? a : kDual && i * 16 >= BN / 2 ? b2 : b;
                load_lds16(p, kpos[j] < left ? off[j] : kOOB, to + (is_a ? 0 : kABytes) + i * 1024);
            }
        };
        u32x4 fa[2][FM], fb[2][FN];
        auto read = [&](int kt, int set) __attribute__((always_inline)) {
            const char* s = lds + stage_of(kt) * kStage;
#pragma unroll
            for (int f = 0; f < FN; ++f) {
                const int r = kDual ? (f / (FN / 2)) * (BN / 2) + (wn * (FN / 2) + f % (FN / 2)) * 16
                                    : (wn * FN + f) * 16;
                fb[set][f] = fragment<BK_, BN>(s + kABytes, r, lane);
            }
#pragma unroll
            for (int f = 0; f < FM; ++f) fa[set][f] = fragment<AK, BM>(s, (wm * FM + f) * 16, lane);
        };
        auto multiply = [&](int set) __attribute__((always_inline)) {
#pragma unroll
            for (int f = 0; f < FM; ++f)
#pragma unroll
                for (int h = 0; h < FN; ++h)
                    acc[h][f] = mfma16x16x32<M_>(fb[set][h], fa[set][f], acc[h][f]);
        };
#pragma unroll
        for (int h = 0; h < FN; ++h)
#pragma unroll
            for (int f = 0; f < FM; ++f) acc[h][f] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (k0 < k1) {
#pragma unroll
            for (int i = 0; i < kStages - 1; ++i) issue(k0 + i);
            wait_loads<(kStages - 2) * kLoads>();
            read(k0, 0);
            // (steps past the last are zeros: loaded as such, or not multiplied)
            auto step = [&](int kt, int set) __attribute__((always_inline)) {
                wait_loads<(kStages - 3) * kLoads>();
                issue(kt + kStages - 1);
                __builtin_amdgcn_sched_barrier(0);
                read(kt + 1, 1 - set);
                multiply(set);
                // each read behind a few MFMAs, all of them in the step's first part
                constexpr int reads = (AK ? FM : 2 * FM) + (BK_ ? FN : 2 * FN);
                constexpr int per = FM * FN * 3 / 4 / reads < 1 ? 1 : FM * FN * 3 / 4 / reads;
#pragma unroll
                for (int i = 0; i < reads; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x008, per, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            };
            for (int kt = k0; kt < k1; kt += 2) {
                step(kt, 0);
                step(kt + 1, 1);
            }
        }
        // (LDS is written until here)
        wait_loads<0>();
    }
};

// A lane holds columns 16 f + 4 q + 0..3 (q = lane / 16) of one row of C in v[f].  Exchanged among the
// four lanes of the row so that each has 4 F columns side by side, from the returned one on: a row's
// columns then leave in 16-byte stores of whole 64- or 128-byte lines.
template <int F>
__device__ __forceinline__ int gather_columns(f32x4 (&v)[F], int lane) {
    static_assert(F == 2 || F == 4, "two or four tiles");
    auto swap = [](f32x4& a, f32x4& b, auto op) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const auto r = op(__float_as_uint(a[e]), __float_as_uint(b[e]));
            a[e] = __uint_as_float(r[0]);
            b[e] = __uint_as_float(r[1]);
        }
    };
    // odd rows of 16 lanes of a with even rows of b; the upper 32 lanes of a with the lower of b
    auto by16 = [](uint32_t a, uint32_t b) __attribute__((always_inline)) {
        return __builtin_amdgcn_permlane16_swap(a, b, false, false);
    };
    auto by32 = [](uint32_t a, uint32_t b) __attribute__((always_inline)) {
        return __builtin_amdgcn_permlane32_swap(a, b, false, false);
    };
    const int q = lane >> 4;
    swap(v[0], v[1], by16);
    if constexpr (F == 2) {
        return 16 * (q & 1) + 8 * (q >> 1);
    } else {
        swap(v[2], v[3], by16);
        swap(v[0], v[2], by32);
        swap(v[1], v[3], by32);
        // (now v[0], v[1], v[2], v[3] are columns 0, 4, 8, 12 of the lane's sixteen)
        return 16 * q;
    }
}

// Workgroup -> (tile row, tile column, product, split): the tiles that one XCD works on at a time
// are eight rows by a few columns of one product, whose operands meet in its L2.
struct GemmPlace {
    int tm, tn, batch, split;
};
__device__ __forceinline__ bool gemm_place(const GemmArgs& g, int batches, GemmPlace* p) {
    // (32 bits: a launch has fewer than 2^31 workgroups)
    const uint32_t tiles = g.tiles_m * g.tiles_n, all = tiles * batches * g.splits;
    const uint32_t x = blockIdx.x % 8, k = blockIdx.x / 8, lo = all / 8, rem = all % 8;
    if (k >= lo + (x < rem ? 1 : 0)) return false;
    const uint32_t id = x * lo + min(x, rem) + k;  // (consecutive ones on one XCD)
    p->batch = (int)(id / (tiles * g.splits));
    const uint32_t in_batch = id % (tiles * g.splits);
    p->split = (int)(in_batch / tiles);
    const int t = (int)(in_batch % tiles), rows = 8;
    const int group = t / (rows * g.tiles_n), in = t % (rows * g.tiles_n);
    const int height = min(rows, g.tiles_m - group * rows);
    p->tm = group * rows + in % height;
    p->tn = in / height;
    return true;
}

}  // namespace haste
