"""CPU: the whole-number part of the attention kernels (maidenx_amd/csrc/attention_walk.hpp), compiled for the host."""
import ctypes as C
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
SRC = os.path.join(HERE, "native", "attention_walk_host.cpp")
LIB = os.path.join(HERE, "native", "libattention_walk_host.so")


@pytest.fixture(scope="module")
def walk():
    hdr = os.path.join(HERE, "..", "maidenx_amd", "csrc", "attention_walk.hpp")
    if not os.path.exists(LIB) or os.path.getmtime(LIB) < max(os.path.getmtime(SRC), os.path.getmtime(hdr)):
        subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Wextra", "-shared", "-fPIC", SRC, "-o", LIB], check=True)
    return C.CDLL(LIB)


def test_a_tile_comes_whole_and_every_wave_issues_what_it_counts(walk):
    assert walk.walk_shares() == 0


@pytest.mark.parametrize("own", [0, 1])
@pytest.mark.parametrize("direct", [(1, 1), (1, 0), (0, 1), (0, 0)])
def test_no_wave_goes_on_before_its_tile_has_come(walk, direct, own):
    """For every size of tile and number of waves, places 2 to 4, walks of one to nine tiles; `own`: a load of a wave's own besides
    the tiles (the row statistics in the kernel of the keys)."""
    for stages in (2, 3, 4):
        for total in range(1, 10):
            assert walk.walk_waits(stages, total, *direct, own) == 0, (stages, total)
