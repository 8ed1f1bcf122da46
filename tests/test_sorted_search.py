"""pv2::lower_bound (csrc/sorted_search.h), which finds where the groups begin among sorted ids: compiled for the host with
checks of signed arithmetic, over keys that a formula gives, up to the largest number of rows."""
import os
import shutil
import subprocess

import pytest

from ponderv2_amd import row_groups

CSRC = os.path.join(os.path.dirname(os.path.abspath(row_groups.__file__)), "csrc")

PROGRAM = """
#include <cstdio>
#include <cstdlib>
#include <initializer_list>
#define __host__
#define __device__
#include "sorted_search.h"
struct Keys {   // `each` keys of every number
  int n, each;
  int operator[](int i) const {
    if (i < 0 || i >= n) { std::printf("key %d of %d\\n", i, n); std::exit(1); }
    return i / each;
  }
};
int main() {
  const int sizes[] = {1, 2, 3, 1000, 1 << 20, (1 << 30) - 1, 1 << 30, (1 << 30) + 1, (1 << 30) + (1 << 29), MAX_ROWS};
  for (int n : sizes)
    for (int each : {1, 3, 1000, 1 << 21, 1 << 30}) {
      const Keys keys = {n, each};
      const int last = (n - 1) / each;
      for (int v : {0, 1, 2, last / 2, last - 1, last, last + 1}) {
        if (v < 0) continue;
        const long long begins = (long long)v * each, want = begins < n ? begins : n;
        const int got = pv2::lower_bound(keys, n, v);
        if (got != want) { std::printf("n %d each %d v %d: %d, not %lld\\n", n, each, v, got, want); return 1; }
      }
    }
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a host compiler")
def test_lower_bound_up_to_the_most_rows(tmp_path):
    source, program = tmp_path / "search.cpp", tmp_path / "search"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    f"-DMAX_ROWS={row_groups.MAX_ROWS}", "-I", CSRC, str(source), "-o", str(program)], check=True)
    run = subprocess.run([str(program)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout + run.stderr
