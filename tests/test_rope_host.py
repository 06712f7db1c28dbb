"""Rotary positions, the parts that need no device, compiled by the host's compiler."""
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run(tmp_path, body):
    src = tmp_path / "a.cpp"
    src.write_text('#include <cstdint>\n#include <cstdio>\n#include "rope.hpp"\nusing namespace trhip;\nint main() {\n' + body + "\nreturn 0; }\n")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "tcb_amd", "csrc"), str(src), "-o", str(tmp_path / "a")], check=True)
    return subprocess.run([str(tmp_path / "a")], check=True, capture_output=True, text=True).stdout


@pytest.mark.parametrize("name", ["sin", "cos"])
def test_what_the_series_leave_out(tmp_path, name):
    """In 64 bits, on an eighth of a turn both ways: below 2^-28, and the constants' nine digits add less than 2^-30."""
    call = "rope_sin(x, x * x)" if name == "sin" else "rope_cos(x * x)"
    out = run(tmp_path, 'for (int i = -4000; i <= 4000; i++) { double x = i * (0.78539816339744831 / 4000); printf("%%.17g\\n", %s); }' % call)
    x = np.arange(-4000, 4001) * (0.78539816339744831 / 4000)
    off = np.abs(np.array([float(v) for v in out.split()]) - getattr(np, name)(x))
    assert len(off) == 8001 and off.max() <= 2.0 ** -28 + 2.0 ** -30, np.log2(off.max())
