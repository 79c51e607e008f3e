"""Copies that do not arrive in time: the launch reports it, waits for what is in flight and returns.

The kernels are built once more with a bound of 0 polls, so that every wait for a copy runs out.
"""

import ctypes as C
import os
import subprocess

import pytest
import torch

import orthocache_gpu_b200 as oc
from orthocache_gpu_b200 import _build, _lib

pytestmark = pytest.mark.gpu
TIMEOUT = 1


@pytest.fixture(scope="module")
def impatient(tmp_path_factory):
    """A library of one translation unit in which no wait succeeds."""
    def load(unit):
        out = str(tmp_path_factory.mktemp("late") / f"{unit}.so")
        subprocess.run([_build.nvcc(), *_build.ARCH, "-O3", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
                        "-DOC_WAIT_POLLS=0", "-shared", os.path.join(_build.CSRC, f"{unit}.cu"), "-o", out, "-lcudart"], check=True)
        lib = C.CDLL(out)
        for name, (res, args) in _lib.SIGNATURES.items():
            if hasattr(lib, name):
                getattr(lib, name).restype, getattr(lib, name).argtypes = res, args
        return lib
    return load


def _stream():
    return _lib.stream_ptr(torch.device("cuda", torch.cuda.current_device()))


def test_page_copies(impatient):
    lib, status = impatient("oc_pages"), torch.zeros(1, dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    for pairs, page_bytes in ((1, 16), (3, 8192 + 64), (40, 65536)):  # one piece a warp, and many
        caches = [torch.randint(0, 255, (2 * pairs, page_bytes), generator=g, device="cuda", dtype=torch.uint8) for _ in range(9)]
        before = [c.clone() for c in caches]
        src = torch.arange(pairs, dtype=torch.int32, device="cuda")
        dst = src + pairs
        at, stride = (C.c_void_p * 9)(*[c.data_ptr() for c in caches]), (C.c_int64 * 9)(*[page_bytes] * 9)
        assert lib.oc_copy_pages(at, stride, 9, page_bytes, 2 * pairs, src.data_ptr(), dst.data_ptr(), pairs,
                                 status.data_ptr(), 148, _stream()) == 0
        assert status.item() == TIMEOUT
        status.zero_()
        assert all(torch.equal(a, b) for a, b in zip(caches, before))
        oc.copy_pages(caches, src, dst)  # and the GPU goes on
        oc.check_status()
        for c, b in zip(caches, before):
            assert torch.equal(c[pairs:], b[:pairs])
