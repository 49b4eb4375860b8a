"""What the operators' outputs share, from the function that refuses them: against every row of small layouts, on the CPU."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r'''
#include <stdio.h>

#include <algorithm>
#include <vector>

#include "token_layout.h"

// Whether any element belongs to two rows.
static bool shares(const fc_axis (&a)[3], long row) {
    std::vector<long> all;
    for (long i = 0; i < a[0].n; i++)
        for (long j = 0; j < a[1].n; j++)
            for (long k = 0; k < a[2].n; k++)
                for (long e = 0; e < row; e++) all.push_back(i * a[0].stride + j * a[1].stride + k * a[2].stride + e);
    std::sort(all.begin(), all.end());
    return std::adjacent_find(all.begin(), all.end()) != all.end();
}

int main() {
    long bad = 0, refused = 0, taken = 0;
    for (long row = 1; row <= 3; row++)
        for (long n0 = 1; n0 <= 3; n0++)
            for (long n1 = 1; n1 <= 3; n1++)
                for (long n2 = 1; n2 <= 2; n2++)
                    for (long s0 = 0; s0 <= 13; s0++)
                        for (long s1 = 0; s1 <= 13; s1++)
                            for (long s2 = 0; s2 <= 7; s2++) {
                                const fc_axis a[3] = {{n0, s0}, {n1, s1}, {n2, s2}};
                                const bool apart = fc_apart(a, row), truth = !shares(a, row);
                                if (apart != truth) bad++;
                                (apart ? taken : refused)++;
                                // one axis alone: as exact as that of one axis
                                if (n1 == 1 && n2 == 1 && apart != fc_apart(n0, s0, row)) bad++;
                            }
    // long axes: nested ones of any length, woven ones that share nothing, and share one row, and ones that are too many to look at
    const fc_axis two[2] = {{1l << 20, 300}, {2, 150}}, far_two[2] = {{1l << 20, 300}, {2, 450}}, one[2] = {{1l << 20, 300}, {2, 299 * 300l}};
    if (!fc_apart(two, 150) || !fc_apart(far_two, 150) || fc_apart(far_two, 151) || fc_apart(one, 1)) bad++;
    const fc_axis woven[2] = {{1l << 22, 4}, {1l << 21, 6}};
    if (fc_apart(woven, 1)) bad++;
    // strides whose products pass 64 bits
    const fc_axis far[3] = {{1l << 24, 1l << 60}, {1l << 30, 1l << 40}, {2, 100}};
    if (fc_apart(far, 10)) bad++;
    const fc_axis wide[2] = {{1l << 24, 1l << 62}, {1l << 20, 1l << 40}};
    if (!fc_apart(wide, 1l << 20)) bad++;
    printf("%ld wrong, %ld taken, %ld refused\n", bad, taken, refused);
    return bad ? 1 : 0;
}
'''


def test_rows_that_share_elements_are_told(tmp_path):
    src, exe = tmp_path / "layout.cpp", tmp_path / "layout"
    src.write_text(PROGRAM)
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I",
                           os.path.join(ROOT, "fastconv_amd", "csrc"), str(src), "-o", str(exe)])
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout + r.stderr
