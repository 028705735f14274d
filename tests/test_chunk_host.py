"""Which positions and tiles a chunk walks, checked on the host against the
definition (tests/native/chunk_host.cu)."""

from __future__ import annotations

import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from insitu_b200 import _lib

HERE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "native")
NONE = 1 << 30


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("chunk_host")
    so, fake = str(d / "chunk_host.so"), str(d / "fake_cuda.o")
    cuda = os.path.join(os.path.dirname(os.path.dirname(_lib.nvcc())), "include")
    subprocess.run(["g++", "-O1", "-fPIC", f"-I{cuda}", "-c", "-o", fake, os.path.join(HERE, "fake_cuda.cpp")], check=True)
    subprocess.run([_lib.nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-O1", "-std=c++17", "-Xcompiler", "-fPIC",
                    "-shared", "-cudart", "none", "-Xlinker", "-Bsymbolic", "-o", so,
                    os.path.join(HERE, "chunk_host.cu"), fake], check=True)
    return C.CDLL(so)


@pytest.mark.parametrize("groups", [1, 2, 4, 8])
def test_walks_and_row_tiles(host, groups):
    rng = np.random.default_rng(groups)
    edges = [1, 2, 63, 64, 65, 127, 128, 129, 255, 256, 257, 383, 384, 385, 700]
    for case in range(400):
        window = NONE if rng.random() < 0.2 else int(rng.choice(edges + [1500]))
        sinks = 0 if window == NONE else int(rng.choice([0, 1, 4] + edges))
        n = int(rng.choice(edges[:13]))
        length = n + int(rng.choice([0] + edges + [1200]))
        assert host.chunk_check(window, sinks, length, n, groups) == 0, (window, sinks, length, n, groups)
