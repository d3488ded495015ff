"""CPU: the bytes that the decay attention kernels load into LDS tiles lie in the tensor, and each of its units is loaded once,
for every number of value dims, over all slices, types and tile forms (triune_amd/csrc/tile_units.h, compiled for the host)."""

import shutil
import subprocess
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "triune_amd" / "csrc"

PROGRAM = r"""
#include "tile_units.h"
#include <cstdio>
#include <vector>

using namespace triune;

// ROWS x D tiles of NTH threads over the columns of a [rows][cols] tensor whose rows are st values apart, as kernels walk
// them: from the tile's first value at column col0.
template <int ROWS, int D, int E, int SIZE, int NTH>
int check(int rows, int Dv, int64_t st) {
    using U = TileUnits<ROWS, D, E, NTH>;
    const int64_t end = ((rows - 1) * st + Dv) * SIZE;  // bytes of the tensor
    std::vector<int> seen(rows * (Dv / E), 0);
    for (int col0 = 0; col0 < Dv; col0 += D)
        for (int t = 0; t < NTH; ++t)
            for (int i = 0; i < U::PER; ++i) {
                const int64_t off = U::load_from(U::offset(t, i, st, SIZE), t, i, rows, Dv - col0);
                if (off == TILE_SKIP) continue;
                const int64_t at = off + (int64_t)col0 * SIZE, row = at / (st * SIZE), byte = at % (st * SIZE);
                if (off < 0 || at + E * SIZE > end || byte + E * SIZE > Dv * SIZE || row >= rows || row >= ROWS) {
                    std::printf("E %d size %d D %d threads %d: %d rows of %d: %lld bytes past the end, row %lld\n", E, SIZE, D,
                                NTH, rows, Dv, (long long)(at + E * SIZE - end), (long long)row);
                    return 1;
                }
                ++seen[row * (Dv / E) + byte / (E * SIZE)];
            }
    for (int n : seen)
        if (n != 1) {
            std::printf("E %d size %d D %d threads %d: %d rows of %d: a unit loaded %d times\n", E, SIZE, D, NTH, rows, Dv, n);
            return 1;
        }
    return 0;
}
template <int ROWS, int D, int E, int SIZE, int NTH>
int sizes() {
    const int least[] = {1, 2, ROWS - 1, ROWS};
    int bad = 0;
    for (int Dv = E; Dv <= 256; Dv += E)
        for (int rows : least)
            for (int64_t st : {(int64_t)Dv, (int64_t)Dv + E, (int64_t)((1 << 22) - E)})
                bad += check<ROWS, D, E, SIZE, NTH>(rows, Dv, st);
    return bad;
}
// The gradients' chunk of 64 or 32 tokens by 32 value dims; 32 tokens by the widths of the walks and their key dims.
template <int E, int SIZE>
int forms() {
    return sizes<E == 8 ? 64 : 32, 32, E, SIZE, 256>() + sizes<E == 8 ? 64 : 32, 64, E, SIZE, 256>() +
           sizes<E == 8 ? 64 : 32, 128, E, SIZE, 256>() + sizes<32, 32, E, SIZE, 128>() + sizes<32, 32, E, SIZE, 256>() +
           sizes<32, 64, E, SIZE, 128>() + sizes<32, 64, E, SIZE, 256>() + sizes<32, 128, E, SIZE, 128>() +
           sizes<32, 128, E, SIZE, 256>();
}
int main() {
    const int bf16 = forms<8, 2>(), fp16 = forms<4, 2>(), fp32 = forms<4, 4>();
    return bf16 + fp16 + fp32 != 0;
}
"""


def test_loads_stay_in_the_tensor(tmp_path):
    src, exe = tmp_path / "units.cpp", tmp_path / "units"
    src.write_text(PROGRAM)
    cxx = shutil.which("g++") or shutil.which("c++")
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", f"-I{CSRC}", "-o", str(exe), str(src)], check=True)
    got = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert got.returncode == 0, got.stdout[-2000:]
