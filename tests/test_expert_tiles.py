"""What the experts' products compute about their tiles (csrc/expert_tiles.h), compiled for the host: the sizes at the limits are
too large to be run."""
import os
import re
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


LIMITS = r"""
#include <stdio.h>
#include <stdlib.h>
#include "expert_tiles.h"
using namespace asb;
// Tiles of a block one after the other, some with long sums that no end is cleared in, some of experts without rows: whoever waits
// for something of a tile waits longer than all that stands before it takes, at five times the time measured for a step and a tile.
int main() {
    long long wrong = 0;
    const int steps[] = {0, 0, 0, 1, 8, 300, 8192, 33554432};  // the last: an expert of 2^31 rows
    for (int i = 0; i < 100000; i++) {
        long long work = 0;
        double before_us = 0;
        for (int t = 0; t < 30; t++) {
            const int n = steps[rand() % 8];
            work += tile_work(n);
            before_us += 5 * (0.3 * n + 32);
            wrong += wait_limit_ns(work) < before_us * 1000.0 || wait_limit_ns(work) < 2000000000ull;
        }
    }
    // 524,288 rows of an expert, 221 tiles of 65,536 x 65,536 a pair, then one short expert with an end: 8192 steps each
    long long work = 0;
    for (int t = 0; t < 221 * 4; t++) work += tile_work(8192);
    wrong += wait_limit_ns(work + tile_work(1)) < 3000000000ull;
    printf("%lld\n", wrong);
    return wrong != 0;
}
"""


def test_a_wait_lasts_as_long_as_what_comes_before_it(tmp_path):
    run_on_host(tmp_path, LIMITS)
    kernel = open(os.path.join(build.CSRC, "expert_mm.cu")).read()
    body = kernel[kernel.index("    expert_mm_kernel("):kernel.index("typedef CUresult")]
    waits = re.findall(r"(?:warp|barrier)_wait(?:<true>)?\((.*)\)", body)
    assert len(waits) == 7 and all("s_stop, work)" in w for w in waits), waits
    roles = re.findall(r"mm_tile<FORM, PAIR>\(s, s_first, s_begin, t\);\n(.*)", body)
    assert len(roles) == 5 and all(r.strip() == "work += tile_work(q.steps);" for r in roles), roles


STAGES = r"""
#include <stdio.h>
// A ring as the copies walk it: what they wait for after their last step is the last use of every stage, and nothing else.
int main() {
    long long wrong = 0;
    for (int stages = 1; stages <= 8; stages++)
        for (int steps = 0; steps < 60; steps++) {
            int stage = 0, uses[8] = {};
            unsigned phase = 0;
            for (int k = 0; k < steps; k++) {
                uses[stage]++;
                if (++stage == stages) stage = 0, phase ^= 1;
            }
            for (int i = 0; i < stages; i++) {
                // done once the phase that `uses` products complete is over: phases 0 .. uses - 1; none was ever begun for 0 uses
                const unsigned parity = phase ^ 1;
                wrong += parity != ((unsigned)(uses[stage] - 1) & 1u);
                if (++stage == stages) stage = 0, phase ^= 1;
            }
        }
    printf("%lld\n", wrong);
    return wrong != 0;
}
"""


def test_a_block_waits_for_the_last_use_of_every_stage(tmp_path):
    run_on_host(tmp_path, STAGES)
    kernel = open(os.path.join(build.CSRC, "expert_mm.cu")).read()
    loops = re.findall(r"warp_wait\(&s_empty\[stage\], phase \^ 1, s_stop, work\)", kernel)
    ends = re.findall(r"if \(good\) last_uses\(s_empty, stage, phase, s.stages, s_stop, work\);\n    \} else if", kernel)
    assert len(loops) == len(ends) == 2  # copies by TMA, copies by warps
