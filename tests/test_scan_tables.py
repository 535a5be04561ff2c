"""The index arithmetic of the packed-sequence kernels, compiled for the host
and run for offsets of every kind, decreasing ones among them."""

from __future__ import annotations

import subprocess

import pytest

from ervf_b200 import _lib, build

CODE = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "ssm_dev.cuh"

using namespace ervf;

#define CHECK(c) \
  if (!(c)) { \
    printf("%s: line %d, offsets %d, tokens %d, seqs %d\n", #c, __LINE__, which, p.tokens, p.seqs); \
    return 1; \
  }

// which 0: rising, with empty ones; 1: 0, T, 0, T, ...; 2: falling; 3: anything, outside the tokens too
std::vector<int> offsets(int which, int tokens, int seqs) {
  std::vector<int> cu(seqs + 1);
  for (int i = 0; i <= seqs; ++i)
    cu[i] = which == 0 ? (i % 3 == 2 && i < seqs ? 0 : (int)((long long)tokens * i / seqs))
            : which == 1 ? (i & 1) * tokens
            : which == 2 ? tokens - (int)((long long)tokens * i / seqs)
                         : rand() % (3 * tokens + 1) - tokens;
  if (which == 0)
    for (int i = 1; i <= seqs; ++i) cu[i] = cu[i] < cu[i - 1] ? cu[i - 1] : cu[i];
  return cu;
}

int main() {
  constexpr int kQ = 128;
  for (int which = 0; which < 4; ++which)
    for (int tokens : {33, 127, 128, 200, 1000, 4099})
      for (int seqs : {1, 2, 3, 4, 9, 40, 300}) {
        const std::vector<int> cu = offsets(which, tokens, seqs);
        const Packing p{cu.data(), nullptr, nullptr, seqs, tokens, 0};
        int tiles = 0;
        for (int i = 0; i < seqs; ++i) {
          int b, len;
          seq_range(p, i, b, len);
          CHECK(b >= 0 && len >= 0 && b + len <= tokens);
          tiles += (len + kQ - 1) / kQ;
        }
        // places: one for each tile, found by the largest first place not behind it
        for (int shift : {5, 6, 7}) {
          const int size = 1 << shift;
          std::vector<int> taken(tokens / size + seqs);
          for (int i = 0; which == 0 && i < seqs; ++i) {
            int b, len;
            seq_range(p, i, b, len);
            for (int k = 0; k < (len ? (len + size - 1) / size : 1); ++k) {
              const int place = first_place(b, i, shift) + k;
              CHECK(place >= 0 && place < (int)taken.size() && taken[place]++ == 0);
              CHECK(i + 1 == seqs || place < first_place(cu[i + 1], i + 1, shift));
            }
          }
        }
        const int most = most_chunks(p, kQ), total = tiles < most ? tiles : most, pairs = 5;
        CHECK(which != 0 || tiles <= most);
        // a launch has as many blocks as chunks or as pieces to plan, whichever is more
        const int blocks = most > 19 ? most : 19;
        std::vector<int> seen(2 * (size_t)most * pairs);
        for (int chunk = 0; chunk < blocks && chunk < tiles; ++chunk)
          for (int k = 0; k < 2 * pairs; ++k) {
            const long long e = step_entry(k, chunk, total);
            CHECK(e < (long long)seen.size() && (e >= 0) == (chunk < total));
            if (e >= 0) CHECK(seen[e]++ == 0);  // nobody else's
          }
      }
  printf("tables ok\n");
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    at = tmp_path_factory.mktemp("tables")
    (at / "t.cu").write_text(CODE)
    cmd = [build.nvcc(), *build.ARCH, "-std=c++17", f"-I{build.CSRC}", f"-I{build.INCLUDE}",
           str(at / "t.cu"), "-o", str(at / "t")]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
    return at / "t"


def test_entries_stay_in_the_table(program):
    r = subprocess.run([str(program)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "tables ok" in r.stdout, r.stdout


def test_packs_of_more_sequences_than_the_tables_are_walked_for():
    """They go token by token, which takes no scratch."""
    need = _lib.load().ervf_ssm_prompt_scratch_bytes
    assert need(_lib.BF16, 1 << 20, 16384, 64, 64, 8, 128) > 0
    assert need(_lib.BF16, 1 << 20, 16385, 64, 64, 8, 128) == 0
    assert need(_lib.BF16, 1 << 26, 1 << 26, 64, 64, 8, 128) == 0
