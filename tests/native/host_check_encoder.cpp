// host_check_encoder.cpp -- drives the host-side code of the embedding, the gated feed-forward block
// and the label log probabilities (argument checks, workspace sizing, how products are cut) without
// a GPU, for the AddressSanitizer / UndefinedBehaviorSanitizer build of `make -C haste_amd
// sanitize_encoder` (host code only; no kernel is launched).  Prints "host_check_encoder OK" and exits
// 0 when every check held; a sanitizer report aborts the run.
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <limits>

#include "../../include/haste_ffi.h"

static int failures = 0;
#define EXPECT(cond)                                                                              \
    do {                                                                                          \
        if (!(cond)) {                                                                            \
            std::fprintf(stderr, "host_check_encoder: %s:%d: %s\n", __FILE__, __LINE__, #cond);   \
            ++failures;                                                                           \
        }                                                                                         \
    } while (0)

static void expect_rejected(int rc) {
    EXPECT(rc < 0);
    EXPECT(std::strlen(haste_last_error()) > 0);
}

// (an address that no check follows)
static char* at(uintptr_t a) { return reinterpret_cast<char*>(a); }
static const int64_t kSizes[] = {std::numeric_limits<int64_t>::min(), -1, 0, 1, 7, 64, 1000, 70000, 1 << 20,
                                 (int64_t)1 << 30, ((int64_t)1 << 31) - 1, (int64_t)1 << 31,
                                 std::numeric_limits<int64_t>::max()};

static void sizes() {
    for (int64_t a : kSizes)
        for (int64_t b : kSizes)
            for (int64_t c : kSizes) {
                const bool legal = a >= 0 && b > 0 && c > 0 && a < (int64_t)1 << 31 &&
                                   b < ((int64_t)1 << 31) - 1 && c < (int64_t)1 << 31;
                EXPECT((haste_embedding_bwd_workspace_size(a, b, c) > 0) == legal);
            }
    for (int64_t b : kSizes)
        for (int64_t o : kSizes)
            for (int32_t k : {-1, 0, 1, 128, 129}) {
                const bool legal = b >= 0 && o > 0 && b < (int64_t)1 << 31 && o < (int64_t)1 << 31 && k >= 0 &&
                                   k <= 128;
                EXPECT((haste_label_log_probs_workspace_size(b, o, k) >= 0) == legal);
            }
    for (int64_t n : kSizes)
        for (int64_t d : kSizes)
            for (int64_t h : kSizes)
                for (int32_t dt = -1; dt <= 3; ++dt)
                    for (int32_t flags = 0; flags < 4; ++flags) {
                        const bool legal = n >= 0 && n < (int64_t)1 << 30 && d > 0 && d <= 1 << 20 && h > 0 &&
                                           h <= 1 << 20 && dt >= 0 && dt <= 2 && n * d < (int64_t)1 << 34;
                        const int64_t size =
                            haste_gated_mlp_workspace_size(n, d, h, d, dt, flags & 1, flags >> 1);
                        EXPECT((size >= 0) == legal);
                        EXPECT((haste_gated_mlp_kept_size(n, h, dt) >= 0) ==
                               (n >= 0 && n < (int64_t)1 << 30 && h > 0 && h <= 1 << 20 && dt >= 0 && dt <= 2));
                    }
}

static void calls() {
    float* f = reinterpret_cast<float*>(at(64));
    int64_t* l = reinterpret_cast<int64_t*>(at(64));
    for (int32_t dt = -1; dt <= 5; ++dt) {
        // every pointer missing
        expect_rejected(haste_embedding(nullptr, 64, nullptr, 8, nullptr, 4, 10, 8, 1.0, dt, nullptr));
        expect_rejected(haste_embedding_bwd(nullptr, 64, nullptr, 8, nullptr, 4, 10, 8, 1.0, -1, dt, nullptr, 0,
                                            nullptr));
        expect_rejected(haste_gated_mlp(nullptr, 8, nullptr, 8, nullptr, 8, nullptr, 8, nullptr, nullptr,
                                        nullptr, 4, 8, 8, 8, 0, dt, nullptr, 0, nullptr));
        expect_rejected(haste_gated_mlp_bwd(nullptr, 8, nullptr, 8, nullptr, 8, nullptr, 8, nullptr, 8, nullptr,
                                            nullptr, nullptr, nullptr, nullptr, nullptr, 4, 8, 8, 8, dt,
                                            nullptr, 0, nullptr));
        expect_rejected(haste_label_log_probs(nullptr, 8, nullptr, 64, 1, nullptr, nullptr, nullptr, nullptr,
                                              nullptr, 4, 8, 1, dt, nullptr, 0, nullptr));
        expect_rejected(haste_label_log_probs_bwd(nullptr, 8, nullptr, 64, 1, nullptr, nullptr, nullptr,
                                                  nullptr, nullptr, 8, 4, 8, dt, nullptr));
    }
    // pitches and sizes at their limits, workspaces that are too small
    for (int64_t ld : kSizes) {
        if (ld != 0 && ld < 8)
            expect_rejected(haste_embedding(at(64), 64, at(64), ld, at(64), 4, 10, 8, 1.0, 0, nullptr));
        if (ld < 8 || ld > 1 << 22)
            expect_rejected(haste_gated_mlp(at(64), ld, at(64), 8, at(64), 8, at(64), 8, at(64), nullptr, at(64),
                                            400, 8, 8, 8, 0, 0, at(256), 1 << 30, nullptr));
        if (ld != 0 && ld < 8)
            expect_rejected(haste_label_log_probs(at(64), ld, nullptr, 64, 0, f, nullptr, f, nullptr, nullptr, 4,
                                                  8, 0, 0, nullptr, 0, nullptr));
    }
    expect_rejected(haste_embedding_bwd(at(64), 64, at(64), 8, at(64), 4, 10, 8, 1.0, -1, 0, at(64), 16, nullptr));
    expect_rejected(haste_label_log_probs(at(64), 131073, l, 64, 1, f, f, f, f, l, 1, 131073, 5, 0, at(64), 16,
                                          nullptr));
    expect_rejected(haste_gated_mlp_bwd(at(66), 8, at(66), 8, at(66), 8, at(66), 8, at(66), 8, at(64), at(64),
                                        at(64), at(64), at(64), at(64), 400, 8, 8, 8, 0, at(64), 16, nullptr));
    // nothing to do
    EXPECT(haste_embedding(nullptr, 32, nullptr, 8, nullptr, 0, 10, 8, 1.0, 0, nullptr) == HASTE_OK);
    EXPECT(haste_gated_mlp(nullptr, 8, nullptr, 8, nullptr, 8, nullptr, 8, nullptr, nullptr, nullptr, 0, 8, 8, 8,
                           2, 2, nullptr, 0, nullptr) == HASTE_OK);
    EXPECT(haste_label_log_probs(nullptr, 8, nullptr, 32, 0, nullptr, nullptr, nullptr, nullptr, nullptr, 0, 8, 8,
                                 1, nullptr, 0, nullptr) == HASTE_OK);
}

int main() {
    sizes();
    calls();
    if (failures) return 1;
    std::puts("host_check_encoder OK");
    return 0;
}
