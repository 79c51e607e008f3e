"""How the paged decode is planned, as its workspace shows it: host arithmetic, without a GPU."""

import ctypes as C
import os

import pytest

from orthocache_gpu_b200 import _lib

pytestmark = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")


class Args(C.Structure):
    """oc_paged_decode_args of include/orthocache_b200.h."""

    _fields_ = [(n, C.c_void_p) for n in ("q", "k_cache", "v_cache", "out", "lse", "slopes", "block_tables", "seq_lens")] + \
        [(n, C.c_int64) for n in ("q_seq_stride", "q_head_stride", "out_seq_stride", "out_head_stride", "kc_block_stride",
                                  "kc_head_stride", "kc_tok_stride", "vc_block_stride", "vc_head_stride", "vc_tok_stride",
                                  "block_table_stride", "num_blocks")] + \
        [("status", C.c_void_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)] + \
        [(n, C.c_float) for n in ("scale", "softcap", "k_scale", "v_scale")] + \
        [(n, C.c_int) for n in ("num_seqs", "kv_heads", "group", "head_dim", "dtype", "cache_dtype", "block_size",
                                "max_blocks", "window", "num_sms")]


def args(**kw):
    a = Args(scale=1.0, k_scale=1.0, v_scale=1.0, num_seqs=4, kv_heads=8, group=4, head_dim=128, dtype=_lib.OC_BF16,
             cache_dtype=_lib.OC_BF16, block_size=16, max_blocks=2048, num_sms=148, num_blocks=8192)
    for name in ("k", "v"):
        setattr(a, f"{name}c_tok_stride", 128)
        setattr(a, f"{name}c_head_stride", 128 * 16)
        setattr(a, f"{name}c_block_stride", 128 * 16 * 8)
    for name, x in kw.items():
        setattr(a, name, x)
    return a


def test_a_window_that_hides_nothing_does_not_change_the_plan():
    lib = _lib.load()
    whole = lib.oc_paged_decode_workspace_bytes(C.byref(args()))
    assert whole > 0  # units are split over the cache's length
    for window in (2048 * 16, 2 ** 31 - 33, 2 ** 31 - 1):
        assert lib.oc_paged_decode_workspace_bytes(C.byref(args(window=window))) == whole, window
    assert lib.oc_paged_decode_workspace_bytes(C.byref(args(window=64))) == 0  # a few tiles: no split


def test_more_tiles_than_32_bits_count_are_refused_before_any_cuda_call():
    """A table of 65535 sequences of up to 2^20 tokens and 64 kv heads: 2^22 units of more than 2^12 tiles."""
    lib, at = _lib.load(), 1 << 20  # an aligned address that nothing reads
    big = dict(num_seqs=65535, kv_heads=64, group=1, block_size=16, max_blocks=1 << 16, q=at, k_cache=at, v_cache=at, out=at,
               block_tables=at, seq_lens=at, workspace=at, workspace_bytes=1 << 40)
    assert lib.oc_paged_decode_attention(C.byref(args(**big)), None) == 5
    assert lib.oc_paged_decode_attention(C.byref(args(**dict(big, dtype=_lib.OC_F16, cache_dtype=_lib.OC_F8E4M3, head_dim=64,
                                                             max_blocks=1 << 20))), None) == 5
