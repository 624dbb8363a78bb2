"""Tiles of a product's rows (cleave_amd/csrc/extents.hpp, used by the 8-bit products) up to the largest extent an int
holds: they have to cover every row, and only a tile inside the matrix is a whole one.  A sum past 2^31 - 1 on the way
would give negative tile counts and part tiles taken for whole ones.  Checked on the CPU by
compiling the header into a small C++ program; no GPU needed."""
from __future__ import annotations

import subprocess

from conftest import ROOT

CHECK = r"""
#include <cstdint>
#include <cstdio>
#include <initializer_list>
#include "extents.hpp"

int main() {
    const int64_t top = 2147483647;
    long long checked = 0;
    for (int64_t near : {int64_t(1), int64_t(700), int64_t(1) << 24, int64_t(1) << 30, top - 300})
        for (int64_t n = near; n < near + 600 && n <= top; ++n)
            for (int64_t tile : {32, 64, 128, 256}) {
                const int64_t tiles = ch::tiles_of((int)n, (int)tile);
                if (tiles < 1 || tiles * tile < n || (tiles - 1) * tile >= n) { printf("tiles %lld %lld\n", (long long)n, (long long)tile); return 1; }
                for (int64_t t : {int64_t(0), tiles / 2, tiles - 2, tiles - 1}) {
                    if (t < 0) continue;
                    if (ch::whole_tile((int)(t * tile), (int)tile, (int)n) != ((t + 1) * tile <= n)) {
                        printf("whole %lld %lld %lld\n", (long long)n, (long long)tile, (long long)t);
                        return 1;
                    }
                }
                ++checked;
            }
    printf("ok %lld\n", checked);
    return 0;
}
"""


def test_weight_gradient_refuses_rows_past_its_sums():
    # null pointers: refused before any device work, the rows before the pointers
    from cleave_amd import _lib

    lib = _lib.load()
    for rows in (2**31 - 1, 2**31 - 4095):
        held = lib.cleave_hip_fp8_codes_len(rows, 1), lib.cleave_hip_fp8_scales_len(rows, 1)
        assert lib.cleave_hip_weight_grad_fp8(None, held[0], None, held[1], None, rows * 4, None, 4, rows, 1, 4) == _lib.ERR_ARG
        assert "rows" in _lib.last_error()[1]
    rows = 2**31 - 4096
    held = lib.cleave_hip_fp8_codes_len(rows, 1), lib.cleave_hip_fp8_scales_len(rows, 1)
    assert lib.cleave_hip_weight_grad_fp8(None, held[0], None, held[1], None, rows * 4, None, 4, rows, 1, 4) == _lib.ERR_ARG
    assert "null" in _lib.last_error()[1]


def test_extents_up_to_the_largest(tmp_path):
    src = tmp_path / "check.cpp"
    src.write_text(CHECK)
    exe = tmp_path / "check"
    subprocess.run(["g++", "-std=c++17", "-O2", "-I", str(ROOT / "cleave_amd" / "csrc"), "-o", str(exe), str(src)],
                   check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.startswith("ok "), r.stdout
