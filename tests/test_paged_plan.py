"""The cut of a paged batch's tiles into pieces, at the limits of what a call may
be: the same header as the kernel's, compiled for the CPU."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <algorithm>
#include <vector>
#include "paged_pieces.h"

// Tiles of nb blocks each, on per_head workgroups
static void check(const std::vector<int>& nb, int per_head) {
  long long sum = 0;
  int most = 1;
  for (int n : nb) sum += n, most = std::max(most, n);
  if (sum > 1 << 30) std::abort();
  const int size = bmx::piece_size(static_cast<int>(sum), per_head, most);
  long long slots = 0, items = 0, covered = 0;
  bool bad = size < 1 || size > most;
  for (int n : nb) {
    int len = -1;
    const long long parts = bmx::piece_count(n, size, &len);
    items += parts;
    if (parts > 1) slots += parts;
    bad = bad || parts < 1 || len < 0 || len > size || len * (parts - 1) > n || (n > 0 && len * (parts - 1) == n) || len * parts < n;
    covered += n;
  }
  // what the workspace has room for
  if (bad || slots > 2LL * per_head || items > static_cast<long long>(nb.size()) + 2LL * per_head) {
    std::printf("%zu tiles, %lld blocks, %d workgroups: size %d, %lld pieces, %lld in slots\n", nb.size(), sum, per_head, size,
                items, slots);
    std::exit(1);
  }
}

int main() {
  const int blocks = 1 << 18;  // 2^24 rows
  unsigned seed = 1;
  auto rnd = [&](int n) { return static_cast<int>((seed = seed * 1664525u + 1013904223u) / 4294967296.0 * n); };
  for (int per_head : {1, 2, 3, 4, 8, 17, 64, 170, 256, 512}) {
    for (int n : {1, 2, 3, 5, 63, 64, 65, 511, 1000, 2730, 2731, 2732, 4095, 4096}) {
      check(std::vector<int>(n, blocks), per_head);
      check(std::vector<int>(n, blocks - 1), per_head);
      for (int nb : {0, 1, 2, 3, 4, 5, 6, 7, 100}) {
        std::vector<int> v(n, nb);
        check(v, per_head);
        v[n / 2] = blocks;
        check(v, per_head);
      }
      std::vector<int> v(n);
      for (int top : {10, 300, blocks})
        for (int i = 0; i < 20; i++) {
          for (int& x : v) x = rnd(top + 1) >> rnd(10);
          check(v, per_head);
        }
    }
    // many short tiles, to the most blocks of a call
    for (int nb : {1, 3, 4, 5, 64, 700})
      check(std::vector<int>(std::min(1 << 21, (1 << 30) / nb), nb), per_head);
  }
  return 0;
}
"""


@pytest.mark.parametrize("flags", [["-O2"], ["-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all"]])
def test_pieces_fit_the_workspace(tmp_path, flags):
    src, exe = tmp_path / "pieces.cpp", tmp_path / "pieces"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", *flags, "-I", os.path.join(ROOT, "base-mlx_amd", "csrc"),
                    str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout + r.stderr
