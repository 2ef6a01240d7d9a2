"""Counts of work items that stop at the room for them (ingot_amd/csrc/launch_bound.hpp), compiled here as plain C++."""
import os
import subprocess

import pytest

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ingot_amd", "csrc", "launch_bound.hpp")

# The sums of the plan of attention over shared prefixes: rounds of 512 spans, 8 waves of 64 lanes, each step checked
# against 31 bits and its verdict (does the span's work fit the room?) against sums in 64 bits.
PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
static int32_t add(int32_t a, int32_t b) {
    int32_t c;
    if (__builtin_add_overflow(a, b, &c)) { std::puts("wraps"); std::exit(1); }
    return c;
}
static int check(const std::vector<int64_t>& items, int32_t room) {
    using ingot::counted;
    int32_t base = 0;
    int64_t exact = 0;
    int kept = 0;
    for (size_t i0 = 0; i0 < items.size(); i0 += 512) {
        int32_t before = 0;
        for (size_t w0 = i0; w0 < i0 + 512; w0 += 64) {
            int32_t upto = 0;
            for (size_t i = w0; i < w0 + 64; ++i) {
                const int64_t n = i < items.size() ? items[i] : 0;
                const int32_t own = counted(n, room), item0 = add(base, add(before, upto));
                upto = add(upto, own);
                const bool fits = add(item0, own) <= room, should = exact + n <= room;
                if (fits != should || (fits && item0 != exact) || item0 < 0) { std::puts("differs"); return 1; }
                kept += fits && n;
                exact += n;
            }
            before = add(before, counted(upto, room));
        }
        base = counted(add(base, counted(before, room)), room);
    }
    std::printf("%d\n", kept);
    return 0;
}
int main() {
    const int32_t most = (int32_t)ingot::kLaunchWorkgroups;
    for (int32_t room : {0, 1, 1000, most}) {
        std::vector<std::vector<int64_t>> lists;
        lists.push_back(std::vector<int64_t>(1 << 18, (int64_t)1 << 15));  // 2^33 items
        lists.push_back(std::vector<int64_t>(70000, 1));
        lists.push_back(std::vector<int64_t>(5000, (int64_t)1 << 62 >> 20));
        lists.push_back(std::vector<int64_t>(2000, most));
        std::vector<int64_t> mixed;
        uint64_t x = 88172645463325252ull;
        for (int i = 0; i < 30000; ++i) {
            x ^= x << 13; x ^= x >> 7; x ^= x << 17;
            mixed.push_back(x % 7 ? (int64_t)(x >> 8) % 1200 : 0);
        }
        lists.push_back(mixed);
        for (const auto& l : lists)
            if (check(l, room)) return 1;
    }
    return 0;
}
"""


@pytest.fixture(scope="module")
def kept(tmp_path_factory):
    d = tmp_path_factory.mktemp("item_counts")
    src, exe = d / "counts.cpp", d / "counts"
    src.write_text(f'#include "{HEADER}"\n{PROGRAM}')
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
    return [int(x) for x in r.stdout.split()]


def test_sums_of_counts_stay_in_31_bits_and_say_what_fits(kept):
    """Lists whose items pass 2^31 (spans whose starts do not rise): what fits the room does so as in 64 bits, nothing wraps."""
    most = 2 ** 24 - 1
    assert kept[:5] == [0] * 5 and kept[5:8] == [0, 1, 0] and kept[11] == 1000
    assert kept[15] == most >> 15 and kept[16] == 70000 and kept[18] == 1
