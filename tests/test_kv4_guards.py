"""What keeps the attention over the 4-bit cache inside its memory when a bounded wait
gives up: compiled from the kernels' own headers, the host side run here."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from lunelette_b200 import build

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def guards(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("guards") / "guards.so")
    flags = [f for f in build.NVFLAGS if f not in ("-Xptxas", "-v")]
    run = subprocess.run([build.NVCC] + flags + build.INCLUDES + [
        "-shared", os.path.join(REPO, "tests", "c_drivers", "kv4_guards.cu"), "-o", out], capture_output=True, text=True)
    assert run.returncode == 0, run.stderr
    return ctypes.CDLL(out)


def test_records_that_are_followed_stay_among_the_parts(guards):
    """The join reads part `first`, then part 2 w of each warp w after its own up to `last`: all of 2 warps
    parts, whatever a workspace without content holds, and every record that the list's warps write."""
    rng = np.random.default_rng(0)
    edge = [-2 ** 31, -7, -2, -1, 0, 1, 2, 3, 6, 7, 8, 9, 15, 16, 2 ** 30, 2 ** 31 - 2, 2 ** 31 - 1]
    words = edge + rng.integers(-2 ** 31, 2 ** 31, 60).tolist() + rng.integers(0, 20, 20).tolist()
    for warps in (1, 4, 8, 2368):
        for first in words:
            for last in words:
                ok = guards.valid_record(first, last, warps)
                if ok:
                    parts = [first, 2 * (first >> 1), 2 * last]
                    assert all(0 <= p < 2 * warps for p in parts) and 1 <= last - (first >> 1) + 1 <= warps
                if 0 <= first < 2 * warps and (first >> 1) <= last < warps:
                    assert ok
