// tile_units.h -- which bytes of a [tokens][columns] tensor the threads of a workgroup load into an LDS tile.  Plain C++, so
// that the rule is checked on the host over all sizes (tests/test_tile_units.py).
#pragma once

#include <cstdint>

namespace triune {

constexpr int TILE_SKIP = 0x40000000;  // an offset past every resource: reads 0, writes nothing

// A tile of ROWS x D values in units of E columns, taken by NTH threads in turn, PER units a thread.
template <int ROWS, int D, int E, int NTH>
struct TileUnits {
    static constexpr int UNITS = D / E, N = ROWS * UNITS, PER = (N + NTH - 1) / NTH;
    static constexpr int row(int thread, int i) { return (thread + i * NTH) / UNITS; }
    static constexpr int col(int thread, int i) { return (thread + i * NTH) % UNITS * E; }
    // Whether unit i of a thread is in the tensor, which has `rows` rows and `cols` columns from the tile's first on: either
    // may be fewer than the tile's.
    static constexpr bool in(int thread, int i, int rows, int cols) {
        return row(thread, i) < (rows < ROWS ? rows : ROWS) && col(thread, i) < cols;
    }
    // Its bytes behind the tile's first value, in a tensor with rows `st` values of `size` bytes apart.
    static constexpr int offset(int thread, int i, int64_t st, int size) {
        return (int)((row(thread, i) * st + col(thread, i)) * size);
    }
    // What is loaded from, `offset` given: past the end of a resource where the unit is not in the tensor.
    static constexpr int load_from(int offset, int thread, int i, int rows, int cols) {
        return in(thread, i, rows, cols) ? offset : TILE_SKIP;
    }
};

}  // namespace triune
