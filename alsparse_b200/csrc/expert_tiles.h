// How the experts' products cut the rows of an expert into tiles, and in what turn the ends of experts are cleared.  Row counts go
// to 2^31 - 4097.
// Plain C++ as well, so that the arithmetic is tested on the host at the limits.
#pragma once

#include "index_bounds.h"

namespace asb {

// Rows of each but the last of `tiles` tiles that n > 0 rows are cut into: equal shares, rounded up to a multiple of `unit`.
// (n + tiles - 1 may pass an int where n does not.)
ASB_HD int equal_share(int n, int tiles, int unit) {
    return ((n - 1) / tiles / unit + 1) * unit;
}

constexpr int kMmMostStages = 8;

// The gradient's steps that end within an expert's rows are cleared by two warps in turn, counted in the order in which every warp
// of the block meets them.
struct EndTurn {
    int warp = 0;
    ASB_HD int take() {
        const int w = warp;
        warp ^= 1;
        return w;
    }
};
// Each of the two has barriers of its own, one a stage: a barrier has one warp that waits for it, and its next phase does not
// complete before that warp has seen the last.  (With one barrier a stage for both, a warp held back while it was not its turn
// could find two phases gone, which looks like none.)
ASB_HD int end_barrier(int warp, int stage) {
    return warp * kMmMostStages + stage;
}

// The limit of a wait.  What a wait may have to sit through is at most what its block has to do from its start to the end of the
// tile at hand: `work`, the sum of tile_work over those tiles.  Two seconds, and 10 us for each unit (a step of 64 terms takes
// 0.3 us, 2.5 us unaligned; a tile of the output 64 us at most, where old values are read element by element).
ASB_HD long long tile_work(int steps) {
    return (long long)steps + 32;
}
ASB_HD unsigned long long wait_limit_ns(long long work) {
    return 2000000000ull + (unsigned long long)work * 10000ull;
}

}  // namespace asb
