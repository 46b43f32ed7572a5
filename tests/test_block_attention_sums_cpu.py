"""The sums of key tiles that the device cuts into runs, in 32 bits: the host's rule (csrc/block_plan.hpp, compiled for the CPU from the
library's own header) against the largest sums that a call's table allows, in whole numbers, whatever max_len says."""
import ctypes
import random
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "comfyui-powershard_amd" / "powershard_amd" / "csrc"
SHIM = """
#include "block_plan.hpp"
extern "C" int fits(long long units, long long table, long long n, long long window, long long sinks)
{
    return psq::block::sums_fit(units, table, n, window, sinks, 64);
}
"""


@pytest.fixture(scope="module")
def fits(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    d = tmp_path_factory.mktemp("sums")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run([gxx, "-O2", "-std=c++20", "-shared", "-fPIC", f"-I{CSRC}", "-o", str(d / "sums.so"), str(d / "shim.cpp")], check=True)
    fn = ctypes.CDLL(str(d / "sums.so")).fits
    fn.argtypes = [ctypes.c_longlong] * 5
    return lambda *a: bool(fn(*a))


def tiles(table, n, length, window, sinks):
    """Key tiles of a sequence's list, as the kernel counts them: those that its last n tokens see, sinks in front."""
    length = min(length, table + n + 64)
    hi = (length + 63) // 64
    lo = min(max(length - n - window + 1, 0) // 64, hi) if window else 0
    return max(min(-(-sinks // 64), lo) + hi - lo, 1)


def test_no_sum_passes_32_bits(fits):
    rng, tight = random.Random(3), 0
    for _ in range(20000):
        table = 16 * int(2 ** rng.uniform(0, 26))
        rows, heads, group = int(2 ** rng.uniform(0, 20)), rng.randint(1, 64), rng.randint(1, 16)
        batch = min(int(2 ** rng.uniform(0, 16)), rows)
        window = rng.choice([0, int(2 ** rng.uniform(0, 30))])
        sinks = rng.choice([0, int(2 ** rng.uniform(0, 30))]) if window else 0
        each = rows // batch
        units = heads * (rows * group // 128 + batch + 1)
        far = tiles(table, each, 2 ** 31 - 1, window, sinks)
        total = batch * heads * -(-each * group // 128) * max(far, tiles(table, each, table, window, sinks))
        if fits(units, table, rows, window, sinks):
            assert total < 2 ** 32
            tight += total > 2 ** 30
    assert tight > 20


@pytest.mark.parametrize("units,table,n,window,sinks,want", [
    (8 * (8191 * 5 // 128 + 2), 131072, 8191, 0, 0, True), (8 * 64, 131072, 64, 0, 0, True), (65535 * 8, 8192, 64, 0, 0, True),
    (60000, 2 ** 23, 8, 0, 0, False), (60000, 2 ** 23, 8, 4096, 64, True), (60000, 2 ** 30 - 16, 8, 2 ** 29, 0, False)])
def test_limits(fits, units, table, n, window, sinks, want):
    """Long texts on many units fit; tables of millions of tokens under tens of thousands of units do not, without a window."""
    assert fits(units, table, n, window, sinks) == want
