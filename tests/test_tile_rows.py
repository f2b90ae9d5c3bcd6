"""The row tiles of the CTA-pair product, computed by the kernel's own function
compiled for the host, up to the largest extent that a view may have."""
import subprocess

from momiru_b200 import build

SOURCE = r"""
#include <cstdio>
#include <cstdlib>
#include "linear_pair.cuh"
int main(int argc, char** argv) {
  for (int i = 1; i < argc; ++i) {
    const int rows = atoi(argv[i]), tiles = int((rows + 255ll) / 256);
    printf("%d\n", mmr::lp_tile_rows(rows, tiles));
  }
}
"""


def test_tile_rows(tmp_path):
    src, exe = tmp_path / "rows.cu", tmp_path / "rows"
    src.write_text(SOURCE)
    subprocess.run([build._nvcc(), "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-I", build.CSRC, "-o", str(exe),
                    str(src)], check=True, capture_output=True)
    most = 2 ** 31 - 1024  # the largest extent admitted
    rows = [1, 2, 31, 32, 33, 255, 256, 257, 288, 300, 511, 512, 513, 4097, 65537, 10 ** 6 + 7, 2 ** 30, 2 ** 30 + 1,
            2139127680, 2139127681, 2139127681 + 256, 2 ** 31 - 2 ** 18, most - 255, most - 1, most]
    got = [int(v) for v in subprocess.run([str(exe), *map(str, rows)], check=True, capture_output=True, text=True).stdout.split()]
    for m, per in zip(rows, got):
        tiles = -(-m // 256)
        assert per % 32 == 0 and 32 <= per <= 256, (m, per)
        assert per * tiles >= m and per * (tiles - 1) < m, (m, per)  # all rows, and no tile without one
