"""The masses that filtered sampling adds up, from the kernel's own header compiled for the host."""
import os
import shutil
import subprocess
from decimal import Decimal, getcontext

import numpy as np
import pytest

from subspec_amd import build as build_mod

PROGRAM = r"""
#include "mass_series.h"
#include <cstdio>
int main() {
  constexpr subspec::SeriesTable table = subspec::series_table();
  double f;
  while (fread(&f, 8, 1, stdin) == 1) {
    const double m = subspec::series_value(table.c, f);
    fwrite(&m, 8, 1, stdout);
  }
}
"""


def test_a_mass_is_within_a_twentieth_of_its_unit_before_it_is_rounded(tmp_path):
    """2^f in units of 2^-42.  What the series leaves out is the twelfth power, (ln 2 / 2)^12 / 12! = 6.3e-15, and 1e-15 of the powers beyond
    and of the economized eleventh, 0.033 units together; each of ten steps rounds a value below 2^42.5, half a step of it (2^-11), and
    scales the errors of those before by at most 1/2: 0.002."""
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc is not installed")
    src, exe = tmp_path / "series.cpp", str(tmp_path / "series")
    src.write_text(PROGRAM)
    subprocess.run([hipcc, "-x", "hip", "--cuda-host-only", "-std=c++17", "-O1", "-ffp-contract=off", "-w", "-I", build_mod.CSRC, str(src), "-o", exe],
                   check=True, timeout=300)
    rng = np.random.default_rng(0)
    f = np.concatenate([[-0.5, 0.5, 0.0, -2.0 ** -30, 2.0 ** -1000], np.linspace(-0.5, 0.5, 1001), rng.uniform(-0.5, 0.5, 1000)])
    got = np.frombuffer(subprocess.run([exe], input=f.tobytes(), stdout=subprocess.PIPE, check=True, timeout=60).stdout)
    assert got.shape == f.shape
    getcontext().prec = 40
    ln2 = Decimal(2).ln()
    off = [abs(Decimal(float(m)) - (Decimal(float(x)) * ln2).exp() * 2 ** 42) for x, m in zip(f, got)]
    assert max(off) <= Decimal("0.035")
