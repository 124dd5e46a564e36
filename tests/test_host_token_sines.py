"""The rotation's sine and cosine, compiled for the host with checks of undefined behaviour."""

from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest

SOURCE = Path(__file__).resolve().parents[1] / "nnunet-mlx_amd" / "csrc" / "nnx_tokens.hip"

MAIN = r"""
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#define __device__
#define __forceinline__ inline
%s
int main() {
  double worst = 0;
  auto check = [&](int32_t turns) {
    float s, c;
    sincos_turns(turns, s, c);
    const double angle = turns * (2 * M_PI / 4294967296.0);
    worst = std::max(worst, std::max(std::fabs(s - std::sin(angle)), std::fabs(c - std::cos(angle))));
  };
  for (int64_t t = INT32_MIN; t <= INT32_MAX; t += 10007) check((int32_t)t);
  for (int eighth = -4; eighth <= 4; ++eighth)
    for (int near = -3; near <= 3; ++near)
      check((int32_t)std::min<int64_t>(INT32_MAX, std::max<int64_t>(INT32_MIN, eighth * 536870912ll + near)));
  std::printf("%%g\n", worst);
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_sine_and_cosine_of_every_eighth_of_a_turn(tmp_path):
    """Both within 3e-7 (a rounded quarter-turn polynomial: z and its square to 2^-24 each, the sum to
    2^-24), and no signed overflow near half a turn."""
    function = re.search(r"__device__ __forceinline__ void sincos_turns\(.*?\n}\n", SOURCE.read_text(), re.S).group()
    (tmp_path / "sines.cpp").write_text(MAIN % function)
    subprocess.run(["g++", "-O1", "-std=c++17", "-ffp-contract=off", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    "sines.cpp", "-o", "sines"], cwd=tmp_path, check=True)
    done = subprocess.run(["./sines"], cwd=tmp_path, capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    assert float(done.stdout) <= 3e-7
