"""How long a context's table of cosines and sines becomes: the header that says so, compiled for the host."""
import os
import subprocess

import pytest

import shainet_amd as sa

CSRC = os.path.join(os.path.dirname(sa.__file__), "csrc")
MOST = 8 << 30

PROGRAM = r"""
#include <cstdio>
#include "rope_table.hpp"
int main() {
  int have, positions, bytes;
  while (std::scanf("%d %d %d", &have, &positions, &bytes) == 3)
    std::printf("%d %lld\n", shainet::table_positions(have, positions, bytes), shainet::most_table_positions(bytes));
}
"""


@pytest.fixture(scope="module")
def lengths(tmp_path_factory):
    at = tmp_path_factory.mktemp("table")
    (at / "look.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-ftrapv", "-I", CSRC, "-o", str(at / "look"), str(at / "look.cpp")], check=True)

    def ask(cases):
        out = subprocess.run([str(at / "look")], input="\n".join("%d %d %d" % c for c in cases), check=True, capture_output=True, text=True).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]

    return ask


def test_tables_double_below_the_bound(lengths):
    cases = [(0, 1, 512), (0, 1024, 512), (0, 1025, 512), (3000, 3001, 512), (1024, 131072, 512), (1024, 131073, 256), (1000, 5000, 32)]
    assert [n for n, _ in lengths(cases)] == [1024, 1024, 2048, 6000, 131072, 262144, 8000]


@pytest.mark.parametrize("hd", list(range(8, 257, 8)))
def test_no_table_is_longer_than_the_bound_or_what_was_asked_for(lengths, hd):
    bytes_each = 4 * hd
    most = MOST // bytes_each
    limit = min(most, 2 ** 31 - 1)
    cases = [(have, positions, bytes_each) for have in (0, 1024, 3000, limit // 2 + 1, limit - 1)
             for positions in (limit // 4 + 1, limit // 2 + 3, limit - 5, limit) if positions > have]
    cases += [(1024, min(limit + 1, 2 ** 31 - 1), bytes_each), (limit // 3, min(limit + 7, 2 ** 31 - 1), bytes_each)]
    for (have, positions, _), (got, bound) in zip(cases, lengths(cases)):
        assert bound == most and got >= positions
        assert got * bytes_each <= MOST or got == positions
        assert got >= 2 * have or got == limit or got == positions  # (few tables on the way to a long one)


def test_tables_without_angles(lengths):
    assert [n for n, _ in lengths([(0, 5000, 0), (1024, 2 ** 31 - 1, 0)])] == [8192, 2 ** 31 - 1]


@pytest.mark.parametrize("hd", [8, 80, 96, 128, 200, 256])
def test_the_tables_before_are_less_than_twice_the_last(lengths, hd):
    have, made = 0, []
    while have < MOST // (4 * hd) and have < 2 ** 31 - 1:
        have = lengths([(have, have + 1, 4 * hd)])[0][0]
        made.append(have)
    assert sum(made[:-1]) < 2 * made[-1] and made[-1] * 4 * hd <= MOST
