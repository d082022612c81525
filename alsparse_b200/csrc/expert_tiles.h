// How the experts' products cut the rows of an expert into tiles.  Row counts go to 2^31 - 4097.
// Plain C++ as well, so that the arithmetic is tested on the host at the limits.
#pragma once

#include "index_bounds.h"

namespace asb {

// Rows of each but the last of `tiles` tiles that n > 0 rows are cut into: equal shares, rounded up to a multiple of `unit`.
// (n + tiles - 1 may pass an int where n does not.)
ASB_HD int equal_share(int n, int tiles, int unit) {
    return ((n - 1) / tiles / unit + 1) * unit;
}

}  // namespace asb
