// launches_check.cpp -- how workgroups are cut into launches (haste_amd/csrc/launches.hpp): all of them, in order,
// once, none of a launch's with 2^32 threads or more.  Prints "launches_check OK".
#include <cstdint>
#include <cstdio>
#include <initializer_list>

#include "../../haste_amd/csrc/launches.hpp"

int main() {
    int bad = 0;
    for (int threads : {64, 256, 512, 1024})
        for (int64_t n : {(int64_t)0, (int64_t)1, (int64_t)4096, ((int64_t)1 << 24) - 1, (int64_t)1 << 24,
                          ((int64_t)1 << 24) + 1, (int64_t)3 << 24, ((int64_t)1 << 32) - 1}) {
            int64_t next = 0;
            haste::in_launches_of(n, threads, [&](int64_t first, int64_t count) {
                bad += first != next || count <= 0 || count * threads >= (int64_t)1 << 32;
                next += count;
            });
            bad += next != n;
        }
    // a call's copies of more than 2^32 threads: two launches
    int launches = 0;
    haste::in_launches_of(((int64_t)1 << 24) + 512, 256, [&](int64_t, int64_t) { ++launches; });
    if (bad || launches != 2) return 1;
    std::puts("launches_check OK");
    return 0;
}
