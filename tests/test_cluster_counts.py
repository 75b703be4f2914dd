"""What is kept of the driver's answers about resident clusters (cluster_counts.h, compiled for the host)."""
import ctypes as C
import os
import random
import subprocess

import pytest

from tests.conftest import ROOT

SOURCE = """
#include "cluster_counts.h"
static adk::ClusterCounts counts;
extern "C" void forget() { counts = {}; }
extern "C" uint32_t find(int device, uint32_t parts, unsigned long long smem) { return counts.find(adk::ClusterCounts::key(device, parts, smem)); }
extern "C" void keep(int device, uint32_t parts, unsigned long long smem, uint32_t n) { counts.keep(adk::ClusterCounts::key(device, parts, smem), n); }
"""


@pytest.fixture(scope="module")
def counts(tmp_path_factory):
    d = tmp_path_factory.mktemp("counts")
    (d / "counts.cc").write_text(SOURCE)
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-I", os.path.join(ROOT, "arraydiff_cuda_b200", "csrc"), str(d / "counts.cc"), "-o", str(d / "counts.so")])
    L = C.CDLL(str(d / "counts.so"))
    L.find.argtypes = [C.c_int, C.c_uint32, C.c_uint64]
    L.keep.argtypes = [C.c_int, C.c_uint32, C.c_uint64, C.c_uint32]
    L.find.restype = C.c_uint32
    return L


def test_devices_and_sizes_have_their_own_answers(counts):
    """A second device, another cluster size and another amount of shared memory are asked for themselves, and calls that
    alternate between shapes find all of them again"""
    counts.forget()
    assert counts.find(0, 1, 49152) == 0
    answers = {(0, 1, 49152): 444, (1, 1, 49152): 222, (0, 2, 49152): 216, (0, 1, 65536): 443, (7, 8, 223232): 9, (0, 8, 223232): 16}
    for shape, n in answers.items():
        assert counts.find(*shape) == 0
        counts.keep(*shape, n)
    for _ in range(3):
        for shape, n in answers.items():
            assert counts.find(*shape) == n


def test_many_shapes_lose_answers_but_never_mix_them(counts):
    counts.forget()
    rng = random.Random(3)
    shapes = [(rng.randrange(0, 64), rng.choice([1, 2, 4, 8]), rng.randrange(1, 223233)) for _ in range(60)]
    for _ in range(2000):
        s = rng.choice(shapes)
        n = counts.find(*s)
        assert n in (0, 1 + shapes.index(s))
        if n == 0:
            counts.keep(*s, 1 + shapes.index(s))
            assert counts.find(*s) == 1 + shapes.index(s)
