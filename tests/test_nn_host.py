"""CPU tests of what the operators on ciphertexts decide on the host: launches and addresses, recorded without a GPU."""
import os
import shutil
import subprocess

import pytest

from conftest import ROOT

HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


@pytest.fixture(scope="module")
def linear_parts(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    exe = str(tmp_path_factory.mktemp("nn") / "linear_parts")
    # the host pass alone (the device code takes half a minute and is never launched): its reference to the device code stays unresolved
    subprocess.check_call([HIPCC, "-x", "hip", "--cuda-host-only", "--offload-arch=gfx950", "-O1", "-std=c++17", "-Wno-unused-function",
                           "-Wl,--unresolved-symbols=ignore-all", "-I", os.path.join(ROOT, "ace-compiler_amd", "csrc"), "-I", os.path.join(ROOT, "include"),
                           os.path.join(ROOT, "tests", "c", "linear_parts.cpp"), "-o", exe])

    def run(*numbers):
        r = subprocess.run([exe, *map(str, numbers)], capture_output=True, text=True, timeout=60)
        words = r.stdout.split()
        return r.returncode, dict(zip(words[::2], map(int, words[1::2])))

    return run


@pytest.mark.parametrize("n_in,ld", [(1, 1), (3, 3), (3, 20), (5, 5), (7, 7), (15, 15), (16, 16), (70, 71), (130, 130)])
@pytest.mark.parametrize("rest", [0, 1, 2, 3, 5, 6, 16, 17, 32, 33, 100])
def test_packed_weights_are_read_inside_their_array(linear_parts, n_in, ld, rest):
    """layers cut at what a workspace of 32 tiles of 16 outputs holds, with every kind of last part: a few bytes, up to 32 outputs, more"""
    part, workspace = 512, 32 * 1024 * ((n_in + 63) // 64)
    rc, got = linear_parts(64, 30, n_in, 2 * part + rest, ld, workspace)
    assert rc == 0 and got["bad"] == 0, got
    assert got["packs"] == 2 + (rest > 32) and got["products"] == 2 + (rest > 0), got


@pytest.mark.parametrize("kind", ["asan", "tsan"])
def test_argument_checks_under_sanitizer(kind):
    """tests/c/san_nn.cpp: random calls of every entry point, from one thread and from four"""
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    subprocess.check_call(["make", "-s", "-C", os.path.join(ROOT, "oracle"), kind + "_nn"])
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=0", UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1", TSAN_OPTIONS="halt_on_error=1")
    r = subprocess.run([os.path.join(ROOT, "oracle", "_san", "san_nn_" + kind)], capture_output=True, text=True, timeout=600, env=env)
    assert r.returncode == 0 and "san_nn: OK" in r.stdout, (r.stdout[-2000:], r.stderr[-4000:])
    assert "ERROR: " not in r.stderr and "WARNING: ThreadSanitizer" not in r.stderr, r.stderr[-4000:]
