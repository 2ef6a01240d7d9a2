"""The bounds of the decoder step's launches (ingot_amd/csrc/launch_bound.hpp), compiled here as plain C++."""
import os
import subprocess

import pytest

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ingot_amd", "csrc", "launch_bound.hpp")


@pytest.fixture(scope="module")
def entries(tmp_path_factory):
    """entries_of_launch of each of a list of workgroups an entry; the first line is a whole launch."""
    d = tmp_path_factory.mktemp("launch_bound")
    src, exe = d / "bound.cpp", d / "bound"
    src.write_text(f'#include <cstdio>\n#include <cstdlib>\n#include "{HEADER}"\n'
                   "int main(int n, char** v) {\n"
                   '    std::printf("%lld\\n", (long long)ingot::kLaunchWorkgroups);\n'
                   '    for (int i = 1; i < n; ++i) std::printf("%lld\\n", (long long)ingot::entries_of_launch(std::atoll(v[i])));\n'
                   "}\n")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", str(src), "-o", str(exe)], check=True)

    def of(blocks):
        out = subprocess.run([str(exe), *map(str, blocks)], check=True, capture_output=True, text=True).stdout.split()
        return int(out[0]), [int(x) for x in out[1:]]

    return of


def test_a_launch_stays_below_32_bits_of_threads(entries):
    """Pages of one to 2^22 workgroups (what the page operations accept): no launch of a split list has 2^32 threads,
    none is empty, and one more entry would not fit."""
    blocks = [1, 2, 3, 15, 16, 17, 255, 256, 1000, 4097, 1 << 20, (1 << 22) - 1, 1 << 22]
    whole, got = entries(blocks)
    assert whole * 256 < 1 << 32 <= (whole + 1) * 256
    for b, n in zip(blocks, got):
        assert n >= 1 and n * b * 256 < 1 << 32 <= (n + 1) * b * 256, b
