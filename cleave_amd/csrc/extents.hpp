// extents.hpp -- tiles of an extent of up to 2^31 - 1 rows, by sums that do not
// pass it.  Plain C++ with no HIP dependency (constexpr serves host
// and device), so a CPU test can check them at the largest extents.
#pragma once

namespace ch {

// Tiles of `tile` that cover n > 0.
constexpr int tiles_of(int n, int tile) { return (n - 1) / tile + 1; }

// Whether the tile of `size` that starts at `at` < n lies in n whole.
constexpr bool whole_tile(int at, int size, int n) { return n - at >= size; }

}  // namespace ch
