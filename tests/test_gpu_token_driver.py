"""The block over a video's patches, from the convolution that embeds them to the gradient of its projections: token_test checks
itself against the same chain in double on the host."""
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fastconv_amd")


@pytest.mark.parametrize("args", [
    [],
    ["-f", "2", "-g", "1", "1", "-c", "8", "-n", "1", "-k", "1", "-d", "8"],          # a token a frame
    ["-f", "4", "-g", "7", "9", "-p", "7", "-c", "64", "-n", "6", "-k", "3", "-d", "64"],
    ["-f", "5", "-g", "14", "14", "-p", "2", "-c", "96", "-n", "2", "-k", "1", "-d", "128"],
], ids=lambda a: " ".join(a) or "default")
def test_block_passes_its_own_check(args):
    exe = os.path.join(PKG, "bin", "token_test")
    if not os.path.exists(exe):
        subprocess.check_call(["make", "-C", PKG, "-s", "host"])
    print("token_test", args, flush=True)
    r = subprocess.run([exe, "-i", "2"] + args, capture_output=True, text=True, timeout=110)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.count("PASS") == 2 and "FAIL" not in r.stdout


def test_bad_sizes_are_refused_before_the_gpu():
    exe = os.path.join(PKG, "bin", "token_test")
    for args in (["-f", "1"], ["-d", "12"], ["-n", "3", "-k", "2"], ["-x"]):
        r = subprocess.run([exe] + args, capture_output=True, text=True, timeout=60)
        assert r.returncode == 1 and "Error" in r.stderr
