"""Where a product of 8 bits keeps the rows that it converts (rllama_amd/csrc/f8_layout.h), on the CPU over all sizes: sixteen bytes at a time are read from aligned places, and
nothing overlaps."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rllama_amd", "csrc")

PROGRAM = r"""
#include "f8_layout.h"
#include <cstdio>
using namespace rlh;

int main() {
    long places = 0;
    for (int m = 1; m <= 16; m++)
        for (int k = 16; k <= 200000; k += 16) {
            const int across = f8_blocks(k), share = rows_f8_share(k);
            const size_t region = rows_f8_region(m, k), items = (size_t)share * m;
            if (share * kRfWaves < across) return printf("k %d: %d blocks, %d a wavefront\n", k, across, share), 1;
            for (int wave = 0; wave < kRfWaves; wave++) {
                const size_t codes = wave * region, scales = codes + items * kRfRow;
                if (codes % 16 != 0 || (codes + kRfRow) % 16 != 0 || scales % 4 != 0) return printf("m %d k %d: wavefront %d at %zu, scales at %zu\n", m, k, wave, codes, scales), 1;
                if (scales + items * 4 > codes + region || codes + region > rows_f8_lds(m, k)) return printf("m %d k %d: wavefront %d of %zu bytes ends past its region\n", m, k, wave, region), 1;
                places++;
            }
        }
    printf("%ld regions\n", places);
    return 0;
}
"""


def test_every_region_is_aligned(tmp_path):
    src, exe = tmp_path / "layout.cpp", tmp_path / "layout"
    src.write_text(PROGRAM)
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-I", CSRC, str(src), "-o", str(exe)])
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout
