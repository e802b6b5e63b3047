// How a number of workgroups is spread over launches.
#pragma once

#include <cstdint>

namespace auv {
namespace seq {

// HIP takes fewer than 2^32 threads along a dimension of a grid: 16,777,215 workgroups of 256, 4,194,303 of 1,024.  Calls
// launch(first workgroup, workgroups) for slices that keep to that, up to the first that fails, whose status it returns.
template <class Launch>
int in_slices(int64_t blocks, int64_t threads, Launch&& launch) {
    const int64_t most = 0xffffffffll / threads;
    for (int64_t first = 0; first < blocks; first += most) {
        const int rc = launch(first, blocks - first < most ? blocks - first : most);
        if (rc != 0) return rc;
    }
    return 0;
}

}  // namespace seq
}  // namespace auv
