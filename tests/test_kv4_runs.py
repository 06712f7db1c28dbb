"""Which tokens the 4-bit cache's row kernels take together, compiled by the host's compiler: no array is read past its ends, at any number of
tokens that a call may have."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROGRAM = r"""
#include <cstdint>
#include <cstdio>
#include <initializer_list>
#include "kv4_runs.hpp"
using namespace trhip;

struct Slots {  // slot t is t + shift; reads out of range are counted
    int64_t tokens, shift;
    mutable long outside = 0;
    int64_t operator[](int64_t t) const {
        if (t < 0 || t >= tokens) outside++;
        return t + shift;
    }
};

int main() {
    for (int64_t tokens : {1LL, 2LL, 3LL, 4LL, 5LL, 9LL, 1000LL, (1LL << 31) - 4, (1LL << 31) - 3, (1LL << 31) - 2, (1LL << 31) - 1})
        for (int64_t shift : {0, 1, 2, 3}) {
            const Slots s = {tokens, shift};
            long taken = 0;
            const int64_t from = tokens > 1000 ? tokens - 1000 : 0;
            for (int64_t t = from; t < tokens; t++) {
                int64_t slot;
                const int n = kv4_together(s, (uint32_t)tokens, (int64_t)1 << 40, (uint32_t)t, slot);
                taken += n;
            }
            // (a run that starts before `from` takes its tokens from there)
            long before = 0;
            for (int64_t t = from < 3 ? 0 : from - 3; t < from; t++) {
                int64_t slot;
                const int n = kv4_together(s, (uint32_t)tokens, (int64_t)1 << 40, (uint32_t)t, slot);
                if (n == 4) before += t + 4 - from > 0 ? t + 4 - from : 0;
            }
            printf("%ld %ld\n", s.outside, taken + before - (long)(tokens - from));
        }
    // the steps of a workgroup pass the last token, and do not come round
    for (uint32_t run : {1u, 4u})
        for (uint32_t t : {0x7FFFFFFEu, 0x7FFFFFFFu - kKv4Groups * run}) printf("0 %d\n", kv4_next(t, kKv4Groups, run) <= t);
    return 0;
}
"""


def test_runs(tmp_path):
    (tmp_path / "a.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fwrapv", "-Wall", "-Wno-unknown-pragmas", "-Werror", "-I", os.path.join(ROOT, "tcb_amd", "csrc"),
                    str(tmp_path / "a.cpp"), "-o", str(tmp_path / "a")], check=True)
    lines = [[int(v) for v in x.split()] for x in subprocess.run([str(tmp_path / "a")], check=True, capture_output=True, text=True).stdout.splitlines()]
    assert len(lines) == 48
    for i, (outside, wrong) in enumerate(lines):
        assert outside == 0 and wrong == 0, (i, outside, wrong)
