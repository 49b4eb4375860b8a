"""The state-space block over a video's patches, from the convolution that embeds them to the gradients of what goes into norm, scan and convolution:
scan_test checks itself against the same chain in double on the host."""
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fastconv_amd")


def program():
    exe = os.path.join(PKG, "bin", "scan_test")
    if not os.path.exists(exe):
        subprocess.check_call(["make", "-C", PKG, "-s", "host"])
    return exe


@pytest.mark.parametrize("args", [
    [],
    ["-f", "2", "-g", "1", "1", "-c", "48", "-e", "50", "-s", "1", "-k", "2"],          # a token a frame
    ["-f", "4", "-g", "7", "9", "-p", "7", "-c", "64", "-e", "130", "-s", "11", "-k", "3"],
    ["-f", "6", "-g", "14", "14", "-p", "2", "-c", "100", "-e", "192", "-s", "16"],      # a prompt that is cut
    ["-f", "3", "-g", "3", "5", "-c", "72", "-e", "66", "-s", "64", "-k", "8"],
], ids=lambda a: " ".join(a) or "default")
def test_block_passes_its_own_check(args):
    print("scan_test", args, flush=True)
    r = subprocess.run([program(), "-i", "2"] + args, capture_output=True, text=True, timeout=110)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.count("PASS") == 8 and "FAIL" not in r.stdout


def test_bad_sizes_are_refused_before_the_gpu():
    for args in (["-f", "1"], ["-s", "65"], ["-k", "1"], ["-k", "9"], ["-x"]):
        r = subprocess.run([program()] + args, capture_output=True, text=True, timeout=60)
        assert r.returncode == 1 and "Error" in r.stderr
