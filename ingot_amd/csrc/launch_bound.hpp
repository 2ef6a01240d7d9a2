// How many workgroups one launch takes: the bounds of the decoder step's grids,
// in plain C++.
#pragma once

#include <cstdint>

namespace ingot {

// A launch takes fewer than 2^32 threads along an axis: 2^24 − 1 workgroups of the
// 256 that all of these kernels have.
constexpr int64_t kWorkgroupThreads = 256;
constexpr int64_t kLaunchWorkgroups = (((int64_t)1 << 32) - 1) / kWorkgroupThreads;

// Entries of a list that one launch takes at `blocks` workgroups an entry
// (1 <= blocks <= kLaunchWorkgroups).
constexpr int64_t entries_of_launch(int64_t blocks) { return kLaunchWorkgroups / blocks; }

}  // namespace ingot
