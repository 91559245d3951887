"""What one call reports of several device error words (``csrc/device_status.cuh``), built with the host compiler."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "nnunet-mlx_b200" / "csrc"

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "device_status.cuh"
// argv: reset, then a status and a site for each word; prints two calls' statuses and sites, and the words that are left
int main(int argc, char** argv) {
  int status[4] = {}, site[4] = {};
  const int words = (argc - 2) / 2;
  for (int i = 0; i < words; ++i) status[i] = atoi(argv[2 + 2 * i]), site[i] = atoi(argv[3 + 2 * i]);
  auto read = [&](int i, int* where) { return *where = site[i], status[i]; };
  auto clear = [&](int i) { status[i] = site[i] = 0; };
  for (int call = 0; call < 2; ++call) {
    int where = 0;
    const int found = nnb::first_error(words, atoi(argv[1]) != 0, &where, read, clear);
    printf("%d %d ", found, where);
  }
  for (int i = 0; i < words; ++i) printf("%d ", status[i]);
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    folder = tmp_path_factory.mktemp("device_status")
    (folder / "main.cc").write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-I", str(CSRC), str(folder / "main.cc"), "-o", str(folder / "main")], check=True)
    return folder / "main"


@pytest.mark.parametrize("reset,words,want", [
    (1, (0, 0, 0, 0), (0, 0, 0, 0, 0, 0)),
    (1, (-4, 21, 0, 0), (-4, 21, 0, 0, 0, 0)),
    (1, (0, 0, -4, 64), (-4, 64, 0, 0, 0, 0)),
    (1, (-4, 21, -4, 64), (-4, 21, -4, 64, 0, 0)),     # the second one outlives the first one's reset
    (0, (-4, 21, -4, 64), (-4, 21, -4, 21, -4, -4)),   # nothing is cleared without a reset
    (0, (0, 0, -4, 64), (-4, 64, -4, 64, 0, -4)),
])
def test_one_error_at_a_time(program, reset, words, want):
    out = subprocess.run([str(program), str(reset), *map(str, words)], check=True, capture_output=True, text=True)
    assert tuple(map(int, out.stdout.split())) == want
