"""CPU: the pair kernel's division by multiplication, compiled from its source and run with reciprocals as far off as
the hardware's division may be (2 units in the last place), at the largest tile numbers that a call can have: 2^23 columns
of tiles (2^31 columns of a few groups' rows) and tile numbers up to 2^31."""
import ctypes
import os
import random
import re
import struct
import subprocess

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tilelang_b200", "csrc", "fp8_pair_gemm.cuh")


@pytest.fixture(scope="module")
def div_small(tmp_path_factory):
    with open(SOURCE) as f:
        text = re.search(r"__device__ __forceinline__ (int div_small\(.*?\n\})", f.read(), re.S).group(1)
    folder = tmp_path_factory.mktemp("div")
    (folder / "div.cc").write_text('extern "C" ' + text)
    subprocess.run(["g++", "-O1", "-ffp-contract=off", "-shared", "-fPIC", "-o", str(folder / "div.so"), str(folder / "div.cc")], check=True)
    f = ctypes.CDLL(str(folder / "div.so")).div_small
    f.argtypes, f.restype = [ctypes.c_int, ctypes.c_int, ctypes.c_float], ctypes.c_int
    return f


def reciprocal(d, ulps):
    """1 / d in float32, some units in the last place off."""
    bits = struct.unpack("<I", struct.pack("<f", 1.0 / d))[0]
    return struct.unpack("<f", struct.pack("<I", bits + ulps))[0]


@pytest.mark.parametrize("d,top", [(1, 1 << 23), (2, 1 << 24), (3, 3 << 23), (5, 5 << 23), (7, 7 << 23), (15, 15 << 23), (16, 1 << 27),
                                   (16 * 3, 1 << 28), (16 * 65537, (1 << 31) - 1), (16 * (1 << 23), (1 << 31) - 1)])
def test_quotients(div_small, d, top):
    rng = random.Random(d)
    numbers = {top - 1 - i for i in range(40)} | {rng.randrange(top) for _ in range(400)}
    numbers |= {min(top - 1, max(0, rng.randrange(top) // d * d + i)) for _ in range(200) for i in (-1, 0, 1)}
    for ulps in (-2, -1, 0, 1, 2):
        inv = reciprocal(d, ulps)
        for n in numbers:
            assert div_small(n, d, inv) == n // d, (n, d, ulps)
