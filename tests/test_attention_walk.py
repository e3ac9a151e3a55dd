"""CPU: the whole-number part of the attention kernels (maidenx_amd/csrc/attention_walk.hpp), compiled for the host."""
import ctypes as C
import os
import subprocess

import numpy as np
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


def offsets_of(kind, r, tokens, sequences):
    if kind == "ascending":
        return np.sort(r.integers(0, tokens + 1, sequences + 1))
    if kind == "any":
        return r.integers(-tokens, 2 * tokens, sequences + 1)
    if kind == "extreme":
        return r.choice([-2 ** 31, -1, 0, 1, tokens - 1, tokens, tokens + 1, 2 ** 31 - 1], sequences + 1)
    o = np.sort(r.integers(0, tokens + 1, sequences + 1))            # a few out of place
    o[r.integers(0, sequences + 1, 1 + sequences // 20)] = r.integers(0, tokens + 1, 1 + sequences // 20)
    return o


@pytest.mark.parametrize("kind", ["ascending", "any", "extreme", "disturbed"])
@pytest.mark.parametrize("sequences", [1, 5, 63, 64, 70, 300])
def test_walks_stay_within_the_tokens(walk, kind, sequences):
    """Whatever the offsets hold, every tile of a walk begins in front of the token up to which it is fetched."""
    r = np.random.default_rng(sequences)
    for tokens in (1, 33, 300, 1500):
        for _ in range(20):
            o = np.ascontiguousarray(offsets_of(kind, r, tokens, sequences), dtype=np.int32)
            assert walk.walk_offsets(o.ctypes.data_as(C.c_void_p), sequences, tokens, kind == "ascending") == 0, (tokens, o.tolist())


def test_a_first_row_that_sees_further_than_the_last(walk):
    o = np.array([0] + [5000] * 31 + [20] + [30] * 32, dtype=np.int32)
    assert walk.walk_offsets(o.ctypes.data_as(C.c_void_p), 64, 5000, 0) == 0
