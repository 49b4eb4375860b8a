"""Where the selective scan's threads read in a tile, from the numbers that its kernels are built with: every value of a tile by one thread, and nothing
past it.  The windows of the tensors are 2^31 - 1 bytes, so that what a thread must not read has to lie behind that, whatever the tokens' distance; a tile
that is the tensors' last ends where they do.  Built with g++ and run here, no GPU."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r'''
#include <stdio.h>
#include <stdlib.h>

#include <set>
#include <utility>

#include "selective_scan_forms.h"

static int failures = 0;
static void fail(const char *what, int N, int thread, long at) {
    if (failures++ < 20) printf("%s: %d states, thread %d, token or byte %ld\n", what, N, thread, at);
}

// What a window of 2^31 - 1 bytes returns for an access at `offset` and, beside it, the scalar `further`: its place, or -1 for zeros.
static long place(uint32_t offset, uint64_t further) {
    const uint64_t at = offset + further;
    return at < 0x7fffffffu ? (long)at : -1;
}

// One axis of a thread's: its first value's offset, tokens from `first` on, every `step`th, `count` of them.
template <class Seen>
static void walk(const char *what, int N, int thread, uint32_t offset, int first, int step, int count, uint32_t token, bool there, long begin, Seen seen) {
    for (int k = 0; k < count; k++) {
        const long at = place(offset, (uint64_t)k * step * token);      // of whole tiles: distances of tokens are scalars
        const int t = first + k * step;
        if (there && t < kScanTile) {
            if (at != begin + (long)t * token) fail(what, N, thread, at);
            seen(t);
        } else if (at != -1) {
            fail(what, N, thread, t);
        }
        // of parts of tiles the offset is one number, and is nowhere past the tokens that are there: it must not pass 32 bits
        if (t < kScanTile && (uint64_t)offset + (uint64_t)k * step * token > 0xffffffffu) fail("a sum passes 32 bits", N, thread, t);
    }
}

int main() {
    for (int N = 1; N <= 64; N++)
        for (uint32_t size : {2u, 4u})
            for (long token : {0l, 1l, (long)N, 64l, 2048l, (1l << 24) - 1})      // values from one token to the next
                with_lanes(N, [&](auto lanes, auto states) {
                    typedef scan_form<decltype(lanes)::value, decltype(states)::value> F;
                    static_assert(F::CH * F::ROWS == F::THREADS && F::EACH * F::ROWS == kScanTile, "");
                    if (F::NP < N || fc_scan_channels(N) != F::CH) fail("lanes", N, 0, F::NP);
                    const uint32_t bytes = (uint32_t)token * size;
                    std::set<std::pair<int, int>> shared, channels;
                    for (int thread = 0; thread < F::THREADS; thread++) {
                        const int n = F::shared_state(thread);
                        walk("B and C", N, thread, F::shared_offset(thread, N, size, bytes), F::shared_token(thread), F::BC, F::SHARED, bytes, n < N, (long)n * size,
                             [&](int t) { if (!shared.insert({t, n}).second) fail("read twice", N, thread, t); });
                        for (int there = 0; there < 2; there++)
                            walk("channels", N, thread, F::channel_offset(thread, there, size, bytes), F::row(thread), F::ROWS, F::EACH, bytes, there,
                                 (long)F::channel(thread) * size, [&](int t) { if (!channels.insert({t, F::channel(thread)}).second) fail("read twice", N, thread, t); });
                    }
                    if ((int)shared.size() != kScanTile * N) fail("B and C of a tile", N, -1, (long)shared.size());
                    if ((int)channels.size() != kScanTile * F::CH) fail("channels of a tile", N, -1, (long)channels.size());
                });
    printf("%d failures\n", failures);
    return failures ? 1 : 0;
}
'''


@pytest.mark.parametrize("sanitize", [[], ["-fsanitize=undefined", "-fno-sanitize-recover=all"]], ids=["plain", "undefined"])
def test_threads_read_their_tile_and_nothing_else(tmp_path, sanitize):
    src, exe = tmp_path / "forms.cpp", tmp_path / "forms"
    src.write_text(PROGRAM)
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "fastconv_amd", "csrc"), str(src), "-o", str(exe)] + sanitize)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout + r.stderr
