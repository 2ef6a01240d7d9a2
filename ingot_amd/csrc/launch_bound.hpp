// How many workgroups one launch takes: the bounds of the decoder step's grids,
// in plain C++.
#pragma once

#include <cstdint>

namespace ingot {

// A launch takes fewer than 2^32 threads along an axis: 2^24 − 1 workgroups of 256.
// Kernels with other workgroups (512 threads draw a token, 64 walk a tree, 512 in one
// workgroup plan shared prefixes) are bounded by their own number, or have fewer.
constexpr int64_t kWorkgroupThreads = 256;
constexpr int64_t kLaunchWorkgroups = (((int64_t)1 << 32) - 1) / kWorkgroupThreads;

// Entries of a list that one launch takes at `blocks` workgroups an entry
// (1 <= blocks <= kLaunchWorkgroups).
constexpr int64_t entries_of_launch(int64_t blocks) { return kLaunchWorkgroups / blocks; }

// n work items of a list with room for `room` (at most kLaunchWorkgroups) of them;
// more count as room + 1. A sum of counts is at most `room` where that of the items is,
// and then the same; and a hundred counts add up below 2^31, whatever the items.
constexpr int32_t counted(int64_t n, int32_t room) { return n <= room ? (int32_t)n : room + 1; }

}  // namespace ingot
