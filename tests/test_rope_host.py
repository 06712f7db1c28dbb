"""Rotary positions, the parts that need no device, compiled by the host's compiler."""
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run(tmp_path, body):
    src = tmp_path / "a.cpp"
    src.write_text('#include <cstdint>\n#include <cstdio>\n#include <initializer_list>\n#include "rope.hpp"\nusing namespace trhip;\nint main() {\n' + body + "\nreturn 0; }\n")
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


def test_launches(tmp_path):
    """Calls of up to 2^31 - 1 tokens in launches of less than 2^32 threads, with one and with four tokens a workgroup; every token once, and only a
    call's last launch may have a rest of four."""
    out = run(tmp_path, """
    static_assert(kRopeTokens % 4 == 0, "");
    const int64_t some[] = {1, 2, 3, 4, 5, 4095, 8192, 1 << 22, (1 << 23) - 1, 1 << 23, (1 << 23) + 1, 1 << 24, (1 << 24) + 1, (1 << 26) + 5, (1LL << 31) - 1};
    for (int64_t tokens : some)
        for (int each : {1, 4}) {
            int64_t done = 0, most = 0;
            bool whole = true;
            for (int64_t t = 0; t < tokens; t += kRopeTokens) {
                const RopeLaunch l = rope_launch(tokens - t, each);
                whole = whole && t == done && (int64_t)l.groups * each >= l.tokens && ((int64_t)l.groups - 1) * each < l.tokens;
                done += l.tokens;
                if ((int64_t)l.groups * kRopeThreads > most) most = (int64_t)l.groups * kRopeThreads;
            }
            printf("%lld %d %lld %lld %d\\n", (long long)tokens, each, (long long)done, (long long)most, whole);
        }""")
    lines = [[int(v) for v in line.split()] for line in out.splitlines()]
    assert len(lines) == 30
    for tokens, each, done, most, whole in lines:
        assert done == tokens and whole and 0 < most < 1 << 32, (tokens, each)
