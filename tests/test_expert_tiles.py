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


TURNS = r"""
#include <stdio.h>
#include <stdlib.h>
#include <vector>
#include "expert_tiles.h"
using namespace asb;
// Copies, products and the two clearing warps of a block as they meet the ends of experts; one of the four is held back for as long
// as another can go on.  A barrier is its number of completed phases; a wait for a parity ends when the phase it is in has the other.
static bool over(unsigned phases, unsigned parity) { return (phases & 1) != parity; }
static bool runs(int stages, int held, const std::vector<int> &stage) {
    const int ends = (int)stage.size();
    unsigned own[2 * kMmMostStages] = {}, ready[kMmMostStages] = {}, empty[kMmMostStages] = {};
    unsigned copy_phase[kMmMostStages] = {}, ready_phase = 0, own_phases[2] = {};
    int at[4] = {};  // copies, products, clearing warps 0 and 1: the end that each is at
    EndTurn copy_turn, clear_turn[2];
    const auto step = [&](int role) {
        if (at[role] == ends) return false;
        const int st = stage[at[role]];
        if (role == 0) {
            if (!over(empty[st], copy_phase[st] ^ 1)) return false;
            copy_phase[st] ^= 1;
            own[end_barrier(copy_turn.take(), st)]++;
        } else if (role == 1) {
            if (!over(ready[st], ready_phase >> st & 1)) return false;
            ready_phase ^= 1u << st;
            empty[st]++;
        } else {
            const int w = role - 2;
            EndTurn look = clear_turn[w];
            if (look.take() == w) {
                if (!over(own[end_barrier(w, st)], own_phases[w] >> st & 1)) return false;
                own_phases[w] ^= 1u << st;
                ready[st]++;
            }
            clear_turn[w] = look;
        }
        at[role]++;
        return true;
    };
    for (;;) {
        bool moved = false;
        const int first = rand() & 3;
        for (int i = 0; i < 4 && !moved; i++)
            if ((first + i) % 4 != held) moved = step((first + i) % 4);
        if (!moved && !step(held)) break;
    }
    return at[0] == ends && at[1] == ends && at[2] == ends && at[3] == ends;
}
int main() {
    long long wrong = 0, seen = 0;
    for (int stages = 1; stages <= kMmMostStages; stages++)
        for (int held = 0; held < 4; held++)
            for (int i = 0; i < 500; i++, seen++) {
                std::vector<int> stage(40);
                int st = 0;
                for (int &v : stage) v = (st += 1 + rand() % (2 * stages)) % stages;
                wrong += !runs(stages, held, stage);
            }
    printf("%lld of %lld\n", wrong, seen);
    return wrong != 0;
}
"""


def test_a_warp_that_is_held_back_misses_no_end(tmp_path):
    run_on_host(tmp_path, TURNS)
    kernel = open(os.path.join(build.CSRC, "expert_mm.cu")).read()
    assert kernel.count("turn.take()") == 2 and kernel.count("end_barrier(") == 2  # the copies and the clearing warps
