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


@pytest.mark.gpu
@pytest.mark.parametrize("aborted", [0, 1])
def test_waits_end_and_copies_in_flight_are_seen_to_land(guards, aborted):
    """A barrier that nothing completes: a wait ends after a second, or soon once another warp gave up. What is
    in flight is waited for all the same, and that wait ends too."""
    import torch

    class Waits(ctypes.Structure):
        _fields_ = [(n, ctypes.c_int) for n in ("waited", "landed", "copied", "abort_word")] + [
            ("wait_ns", ctypes.c_ulonglong), ("land_ns", ctypes.c_ulonglong), ("words_right", ctypes.c_int)]

    src = torch.arange(1024, dtype=torch.int32, device="cuda")
    out = torch.zeros(ctypes.sizeof(Waits), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    assert guards.run_waits(ctypes.c_void_p(out.data_ptr()), ctypes.c_void_p(src.data_ptr()), aborted) == 0
    got = Waits.from_buffer_copy(out.cpu().numpy().tobytes())
    assert got.copied and got.words_right == 1024
    assert not got.waited and got.abort_word == 1
    if aborted:
        assert got.wait_ns < 5e8
    else:
        assert 0.99e9 < got.wait_ns < 2e9
    assert not got.landed and got.land_ns < 1e8
