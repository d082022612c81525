"""What the experts' products compute about their tiles (csrc/expert_tiles.h), compiled for the host: the sizes at the limits are
too large to be run."""
import os
import subprocess

from alsparse_b200 import build


def run_on_host(tmp_path, main):
    (tmp_path / "main.cpp").write_text(main)
    exe = tmp_path / "main"
    subprocess.check_call(["/usr/bin/g++", "-std=c++17", "-O1", "-ftrapv", "-Wall", "-Werror", "-I", build.CSRC,
                           str(tmp_path / "main.cpp"), "-o", str(exe)])
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout
    return out.stdout


SHARES = r"""
#include <limits.h>
#include <stdio.h>
#include "expert_tiles.h"
using namespace asb;
// the tiles cover the rows, each at most `tile` of them and none of them empty
static bool good(int n, int tile, int unit) {
    const int tiles = (int)(((long long)n + tile - 1) / tile), share = equal_share(n, tiles, unit);
    const long long mean = ((long long)n + tiles - 1) / tiles;
    if (share != (mean + unit - 1) / unit * unit || share <= 0 || share > tile) return false;
    return (long long)(tiles - 1) * share < n && (long long)tiles * share >= n;
}
int main() {
    long long wrong = 0, seen = 0;
    const int tile[] = {32, 64, 128, 256}, unit[] = {16, 16, 16, 32}, most = INT_MAX - 4096;
    for (int i = 0; i < 4; i++) {
        for (int n = 1; n < 70000; n++, seen++) wrong += !good(n, tile[i], unit[i]);
        for (int n = most; n > most - 70000; n--, seen++) wrong += !good(n, tile[i], unit[i]);
        for (int n = most; n > 0; n -= 104729, seen++) wrong += !good(n, tile[i], unit[i]);
    }
    printf("%lld of %lld\n", wrong, seen);
    return wrong != 0;
}
"""


def test_rows_of_an_expert_in_equal_tiles(tmp_path):
    run_on_host(tmp_path, SHARES)
    kernel = open(os.path.join(build.CSRC, "expert_mm.cu")).read()
    assert "equal_share(" in kernel and "tiles - 1) / tiles" not in kernel
