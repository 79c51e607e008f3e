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
    done = {}

    def load(unit):
        if unit in done:
            return done[unit]
        out = str(tmp_path_factory.mktemp("late") / f"{unit}.so")
        subprocess.run([_build.nvcc(), *_build.ARCH, "-O3", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
                        "-DOC_WAIT_POLLS=0", "-shared", os.path.join(_build.CSRC, f"{unit}.cu"), "-o", out, "-lcudart"], check=True)
        lib = C.CDLL(out)
        for name, (res, args) in _lib.SIGNATURES.items():
            if hasattr(lib, name):
                getattr(lib, name).restype, getattr(lib, name).argtypes = res, args
        done[unit] = lib
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


@pytest.mark.parametrize("lens", [[40, 300, 0], [1, 20000]])
def test_paged_decode(impatient, lens):
    """Units of a CTA each, and units that are split: the launch ends, and the next one of the same GPU is right."""
    from test_paged_decode_plan import Args
    from serving_helpers import pages_for
    lib = impatient("oc_paged_attn")
    table, pages = pages_for(lens, 16, "cuda")
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn(len(lens), 8, 64, device="cuda", dtype=torch.bfloat16)
    k, v = (torch.randn(pages, 2, 16, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    want = oc.paged_decode_attention(q, k, v, table, n)
    out, status = torch.empty_like(q), torch.zeros(1, dtype=torch.int32, device="cuda")
    a = Args(q=q.data_ptr(), k_cache=k.data_ptr(), v_cache=v.data_ptr(), out=out.data_ptr(), block_tables=table.data_ptr(),
             seq_lens=n.data_ptr(), q_seq_stride=q.stride(0), q_head_stride=q.stride(1), out_seq_stride=out.stride(0),
             out_head_stride=out.stride(1), kc_block_stride=k.stride(0), kc_head_stride=k.stride(1), kc_tok_stride=k.stride(2),
             vc_block_stride=v.stride(0), vc_head_stride=v.stride(1), vc_tok_stride=v.stride(2),
             block_table_stride=table.stride(0), num_blocks=pages, status=status.data_ptr(), scale=0.125, k_scale=1.0,
             v_scale=1.0, num_seqs=len(lens), kv_heads=2, group=4, head_dim=64, dtype=_lib.OC_BF16, cache_dtype=_lib.OC_BF16,
             block_size=16, max_blocks=table.shape[1], num_sms=148)
    a.workspace_bytes = lib.oc_paged_decode_workspace_bytes(C.byref(a))
    space = torch.empty(max(1, a.workspace_bytes), dtype=torch.uint8, device="cuda")
    a.workspace = space.data_ptr()
    assert lib.oc_paged_decode_attention(C.byref(a), _stream()) == 0
    assert status.item() == TIMEOUT
    assert torch.equal(oc.paged_decode_attention(q, k, v, table, n), want)
    oc.check_status()
