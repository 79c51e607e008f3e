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


class RotaryArgs(C.Structure):
    """oc_rotary_args of include/orthocache_b200.h."""

    _fields_ = [(n, C.c_void_p) for n in ("q", "k", "v", "q_out", "k_out")] + \
        [(n, C.c_int64) for n in ("q_tok_stride", "q_head_stride", "k_tok_stride", "k_head_stride", "v_tok_stride",
                                  "v_head_stride", "qo_tok_stride", "qo_head_stride", "ko_tok_stride", "ko_head_stride", "tokens")] + \
        [(n, C.c_void_p) for n in ("positions", "seq_ids", "cos_tab", "sin_tab")] + [("table_rows", C.c_int64)] + \
        [(n, C.c_void_p) for n in ("k_cache", "v_cache")] + \
        [(n, C.c_int64) for n in ("kc_block_stride", "kc_head_stride", "kc_tok_stride", "vc_block_stride", "vc_head_stride",
                                  "vc_tok_stride")] + [("block_tables", C.c_void_p)] + \
        [(n, C.c_int64) for n in ("block_table_stride", "num_blocks")] + [("status", C.c_void_p)] + \
        [(n, C.c_float) for n in ("k_scale", "v_scale")] + \
        [(n, C.c_int) for n in ("q_heads", "kv_heads", "head_dim", "rotary_dim", "dtype", "cache_dtype", "positions_64", "flags",
                                "block_size", "max_blocks", "num_seqs", "num_sms")]


@pytest.mark.parametrize("T, H", [(2400, 1), (2400, 40), (9000, 3)])
def test_rotary_of_prompts(impatient, T, H):
    """One piece a warp, and more than its ring holds."""
    lib, status = impatient("oc_rotary"), torch.zeros(1, dtype=torch.int32, device="cuda")
    x = torch.randn(T, H, 128, device="cuda", dtype=torch.float16)
    pos = torch.arange(T, device="cuda", dtype=torch.int32)
    cos, sin = oc.rotary_tables(128, T, device="cuda")
    want = oc.rotary_embedding(x, pos, cos, sin)
    out = torch.full_like(x, 7.0)
    a = RotaryArgs(q=x.data_ptr(), q_out=out.data_ptr(), q_tok_stride=x.stride(0), q_head_stride=x.stride(1),
                   qo_tok_stride=x.stride(0), qo_head_stride=x.stride(1), tokens=T, positions=pos.data_ptr(),
                   cos_tab=cos.data_ptr(), sin_tab=sin.data_ptr(), table_rows=T, status=status.data_ptr(), k_scale=1.0, v_scale=1.0,
                   q_heads=H, head_dim=128, rotary_dim=128, dtype=_lib.OC_F16, num_sms=148)
    assert lib.oc_rotary_append_paged(C.byref(a), _stream()) == 0
    assert status.item() == TIMEOUT and bool((out == 7.0).all())
    assert torch.equal(oc.rotary_embedding(x, pos, cos, sin), want)
    oc.check_status()


class PromptArgs(C.Structure):
    """oc_prompt_args of include/orthocache_b200.h."""

    _fields_ = [(n, C.c_void_p) for n in ("q", "k", "v", "out", "lse", "slopes", "cu_q", "cu_k", "prefix_lens")] + \
        [(n, C.c_int64) for n in ("q_tok_stride", "q_head_stride", "k_tok_stride", "k_head_stride", "v_tok_stride",
                                  "v_head_stride", "out_tok_stride", "out_head_stride", "lse_tok_stride", "tokens", "key_tokens")] + \
        [("status", C.c_void_p)] + [(n, C.c_float) for n in ("scale", "softcap")] + \
        [(n, C.c_int) for n in ("docs", "kv_heads", "group", "head_dim", "dtype", "causal", "window", "num_sms")]


@pytest.mark.parametrize("T, D", [(100, 64), (900, 64), (900, 128), (5000, 64)])
def test_prompt_attention(impatient, T, D):
    """Tensor memory and the SM are given back: the next launches are right."""
    lib, status = impatient("oc_prompt_attn"), torch.zeros(1, dtype=torch.int32, device="cuda")
    q, k, v = (torch.randn(T, h, D, device="cuda", dtype=torch.bfloat16) for h in (4, 2, 2))
    want, out = oc.prompt_attention(q, k, v), torch.empty_like(q)
    a = PromptArgs(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(), q_tok_stride=q.stride(0),
                   q_head_stride=D, k_tok_stride=k.stride(0), k_head_stride=D, v_tok_stride=v.stride(0), v_head_stride=D,
                   out_tok_stride=out.stride(0), out_head_stride=D, tokens=T, key_tokens=T, status=status.data_ptr(),
                   scale=D ** -0.5, docs=1, kv_heads=2, group=2, head_dim=D, dtype=_lib.OC_BF16, causal=1, num_sms=148)
    for _ in range(3):
        assert lib.oc_prompt_attention(C.byref(a), _stream()) == 0
    assert status.item() == TIMEOUT
    assert torch.equal(oc.prompt_attention(q, k, v), want)
    oc.check_status()
