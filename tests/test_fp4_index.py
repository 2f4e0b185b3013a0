"""Index arithmetic of the 4-bit float products, compiled for the host."""
import ctypes
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "relax_b200", "csrc")


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("index")
    src, so = str(d / "index.cc"), str(d / "index.so")
    with open(src, "w") as f:
        f.write('#include "fp4_index.h"\n'
                'extern "C" int tile_width(int m, int m0, int most) { return rb200::f4::tile_width(m, m0, most); }\n')
    subprocess.check_call(["g++", "-O1", "-fwrapv", "-shared", "-fPIC", "-I" + CSRC, src, "-o", so])
    return ctypes.CDLL(so)


@pytest.mark.parametrize("m", [1, 31, 32, 65, 255, 256, 257, 300, 512, 1000, 2 ** 31 - 257, 2 ** 31 - 33, 2 ** 31 - 32, 2 ** 31 - 1])
def test_width_of_every_kind_of_tile(lib, m):
    tiles = -(-m // 256)
    for t in {0, tiles // 2, max(tiles - 2, 0), tiles - 1}:
        w = lib.tile_width(m, t * 256, 256)
        left = min(256, m - t * 256)
        assert w % 32 == 0 and left <= w < left + 32
