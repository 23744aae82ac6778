// Launches of any number of workgroups.
#pragma once

#include <stdint.h>

#include <algorithm>

namespace haste {

// f(first, count) over launches of `count` of the workgroups, fewer than 2^32 threads each (more are refused).
template <typename F>
void in_launches_of(int64_t workgroups, int threads, F f) {
    const int64_t most = (((int64_t)1 << 32) - 1) / threads;
    for (int64_t i = 0; i < workgroups; i += most) f(i, std::min(most, workgroups - i));
}

}  // namespace haste
