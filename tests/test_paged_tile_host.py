"""Which bytes of a page's rows the attention kernel asks for, for every head size: the header that says so, compiled for the host."""
import os
import subprocess

import pytest

import shainet_amd as sa

CSRC = os.path.join(os.path.dirname(sa.__file__), "csrc")

PROGRAM = r"""
#include <cstdio>
#include <vector>
#include "paged_tile.hpp"
using namespace shainet;

// A lane is a row m of an operand, 0 .. 15, in quarter j; widths as the kernel takes them.
template <int DTYPE, int HD>
void look(int above) {
  typedef PageTile<DTYPE, HD> T;
  for (int hd = above + 8; hd <= HD; hd += 8) {
    const int bytes = hd * T::E;
    int behind = 0, missed = 0, odd = 0, twice = 0;
    std::vector<int> key(bytes, 0), value(hd, 0);
    for (int u = 0; u < T::CHUNKS; ++u)
      for (int j = 0; j < 4; ++j) {
        const int at = T::key_byte(u, j, bytes);
        if (at < 0 || at + 16 > bytes) ++behind;
        if (at & 15) ++odd;
        if ((u * 4 + j) * 16 < bytes) {  // (a query number stands against it)
          if (at != (u * 4 + j) * 16) ++missed;
          for (int b = 0; b < 16 && at + b < bytes; ++b) ++key[at + b];
        }
      }
    for (int u = 0; u < T::PIECES; ++u)
      for (int m = 0; m < 16; ++m) {
        const int d = T::value_column(u, m, hd), begin = T::VEC * (m + 16 * u);
        if (d < 0 || (d * T::E) + T::WORDS * 4 > bytes) ++behind;
        if (d * T::E % 4) ++odd;
        if (begin >= hd) continue;  // (not written to the outputs)
        if (begin + T::VEC <= hd && d != begin) ++missed;
        for (int e = 0; e < T::VEC && d + e < hd; ++e) ++value[d + e];
      }
    for (int b = 0; b < bytes; ++b)
      if (key[b] != 1) ++missed;
    for (int d = 0; d < hd; ++d) {
      if (value[d] < 1) ++missed;
      if (value[d] > 1) ++twice;
    }
    std::printf("%d %d %d %d %d %d %d\n", DTYPE, HD, hd, behind, missed, odd, twice);
  }
}
template <int DTYPE>
void all() {
  look<DTYPE, 64>(0);
  look<DTYPE, 96>(64);
  look<DTYPE, 128>(96);
  look<DTYPE, 256>(128);
}
int main() {
  all<kPageF32>();
  all<kPageBf16>();
  all<kPageF16>();
}
"""


@pytest.fixture(scope="module")
def looked_at(tmp_path_factory):
    at = tmp_path_factory.mktemp("tile")
    (at / "look.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", CSRC, "-o", str(at / "look"), str(at / "look.cpp")], check=True)
    lines = subprocess.run([str(at / "look")], check=True, capture_output=True, text=True).stdout.splitlines()
    return [tuple(map(int, line.split())) for line in lines]


def test_every_type_and_head_size_is_looked_at(looked_at):
    assert sorted((t, hd) for t, _, hd, *_ in looked_at) == [(t, hd) for t in range(3) for hd in range(8, 257, 8)]


def test_no_piece_ends_behind_its_row(looked_at):
    assert [line for line in looked_at if line[3]] == []


def test_every_number_of_a_row_is_asked_for(looked_at):
    """And keys once; of values that two pieces have, which are written twice, there are few."""
    assert [line for line in looked_at if line[4] or line[5]] == []
    assert {(line[2], line[6]) for line in looked_at if line[6]} == {(80, 1), (80, 4), (88, 2)}
