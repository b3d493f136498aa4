"""Dense layer: places and choices made on the host or by code that a host compiler takes (no GPU)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run_cpp(tmp_path, body):
    src, exe = tmp_path / "check.cpp", tmp_path / "check"
    src.write_text(body)
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", os.path.join(ROOT, "disn_amd", "csrc"), "-o", str(exe), str(src)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout


def test_pieces_of_a_tile_stay_in_their_line(tmp_path):
    """every piece of every tile of a line of n >= V values: read inside the line, and holding the line's values at its own
    place, where there are any, and zeros behind the line's end"""
    run_cpp(tmp_path, r"""
#include <cstdio>
#include "tile_edge.h"
int main() {
  const int V = 4;
  for (int rows = 128; rows <= 256; rows *= 2)
    for (int n = V; n < 1300; ++n)
      for (int i0 = 0; i0 < n; i0 += rows)
        for (int c = 0; c < rows; c += V) {
          const int left = n - i0;
          const EdgePiece e = edge_piece(c, left, V);
          const int first = i0 + e.at - e.back;
          if (first < 0 || first + V > n || e.back < 0 || e.back >= V) {
            std::printf("tile of %d, line of %d: the piece at column %d is read at %d (back %d)\n", rows, n, i0 + c, first, e.back);
            return 1;
          }
          for (int i = 0; i < V; ++i)
            if (c < left && (i + e.back < V ? first + e.back + i != i0 + c + i : c + i < left)) {
              std::printf("tile of %d, line of %d: column %d is not what it should be\n", rows, n, i0 + c + i);
              return 1;
            }
        }
}
""")
