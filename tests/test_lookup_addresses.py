"""Every address that the lookup forms for rows that are no whole number of 16 bytes, walked on the host: no load may leave
the ids or the table, and each output element takes its own table element."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xnn_b200", "csrc")

PROGRAM = r"""
#include <cstdio>
#include <vector>
#include "embedding_impl.h"

template <int W> int check(int64_t N, int64_t V, uint32_t C, const std::vector<long long>& ids) {
  const uint32_t items = (uint32_t)(N * C);
  for (uint32_t e0 = 0; e0 < items; e0 += W) {
    int64_t at[W];
    for (int e = 0; e < W; ++e) at[e] = -1;
    const auto take = [&](int e, int64_t v, uint32_t c) { at[e] = v < 0 ? -1 : v * C + c; };
    if (e0 + W <= items) walk_elements<W, true>(e0, items, C, V, ids.data(), take);
    else walk_elements<W, false>(e0, items, C, V, ids.data(), take);
    for (int e = 0; e < W; ++e) {
      const int64_t n = (e0 + e) / C, v = e0 + e < items ? ids[n] : -1;
      const int64_t want = e0 + e < items && v >= 0 && v < V ? v * C + (e0 + e) % C : -1;
      if (at[e] != want) { std::printf("W %d N %lld V %lld C %u element %u: %lld, not %lld\n", W, (long long)N, (long long)V, C, e0 + e, (long long)at[e], (long long)want); return 1; }
    }
  }
  return 0;
}

int main() {
  int bad = 0;
  for (int64_t N : {1, 2, 3, 4, 5, 7, 8, 33})
    for (int64_t V : {1, 2, 4, 9})
      for (uint32_t C = 1; C <= 131; C = C < 20 ? C + 1 : C + 37) {
        for (int kind = 0; kind < 3; ++kind) {
          std::vector<long long> ids(N);
          for (int64_t i = 0; i < N; ++i) ids[i] = kind == 0 ? V - 1 : kind == 1 ? (i * 7 + 3) % V : (i * 5) % (V + 2) - 1;
          bad += check<4>(N, V, C, ids) + check<2>(N, V, C, ids);
        }
      }
  return bad != 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a C++ compiler")
def test_every_element_is_in_its_row(tmp_path):
    source = tmp_path / "walk.cpp"
    source.write_text(PROGRAM)
    program = str(tmp_path / "walk")
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=address,undefined", "-I", CSRC, str(source), "-o", program], check=True)
    # the sanitizer's runtime wants to be the first library, and leaks are not what is looked for
    env = {**{k: v for k, v in os.environ.items() if k != "LD_PRELOAD"}, "ASAN_OPTIONS": "detect_leaks=0"}
    out = subprocess.run([program], capture_output=True, text=True, env=env)
    assert out.returncode == 0, out.stdout[-2000:] + out.stderr[-2000:]
