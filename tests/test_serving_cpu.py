"""CPU tests of the paged-serving operators: rotary tables, refusals of the C ABI and of the binding."""

import ctypes
import math
import os

import pytest
import torch

import orthocache_gpu_b200 as oc
from orthocache_gpu_b200 import _lib

needs_library = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")
needs_binding = pytest.mark.skipif(not os.path.exists(os.path.join(os.path.dirname(_lib.LIB_PATH), "oc_torch.so")),
                                   reason="binding not built")


def _angle(cos, sin, pos, i):
    return math.atan2(float(sin[pos, i]), float(cos[pos, i]))


def test_rotary_tables_are_the_cosines_and_sines_of_the_angles():
    cos, sin = oc.rotary_tables(8, 100000, 10000.0)
    assert cos.shape == sin.shape == (100000, 4) and cos.dtype == torch.float32
    for pos in (0, 1, 77, 99999):
        for i in range(4):
            a = pos * 10000.0 ** (-2 * i / 8)
            # one rounding to float32 of a value of at most 1
            assert abs(float(cos[pos, i]) - math.cos(a)) <= 2.0 ** -24
            assert abs(float(sin[pos, i]) - math.sin(a)) <= 2.0 ** -24


def test_rotary_scaling():
    plain = oc.rotary_tables(64, 64)
    cos, sin = oc.rotary_tables(64, 256, scaling={"type": "linear", "factor": 4.0})
    assert torch.allclose(cos[::4][:64], plain[0], atol=2e-7) and torch.allclose(sin[::4][:64], plain[1], atol=2e-7)
    # ntk: the fastest pair is kept, the slowest divided by the factor
    cos, sin = oc.rotary_tables(64, 64, scaling={"type": "ntk", "factor": 4.0})
    assert abs(_angle(cos, sin, 1, 0) - 1.0) < 1e-6
    assert abs(_angle(cos, sin, 60, 31) / _angle(*plain, 60, 31) - 0.25) < 1e-4
    # yarn: fast pairs kept, slow ones divided, and the magnitude
    cos, sin = oc.rotary_tables(64, 64, scaling={"type": "yarn", "factor": 4.0, "original": 2048})
    size = (cos.double() ** 2 + sin.double() ** 2).sqrt()
    assert torch.allclose(size, torch.full_like(size, 0.1 * math.log(4.0) + 1.0), atol=1e-6)
    assert abs(_angle(cos, sin, 1, 0) - 1.0) < 1e-6
    assert abs(_angle(cos, sin, 60, 31) / _angle(*plain, 60, 31) - 0.25) < 1e-4
    # bands: by wavelength
    cos, sin = oc.rotary_tables(64, 64, scaling={"type": "bands", "factor": 8.0, "original": 4096, "low": 1, "high": 4})
    assert abs(_angle(cos, sin, 1, 0) - 1.0) < 1e-6
    assert abs(_angle(cos, sin, 60, 31) / _angle(*plain, 60, 31) - 0.125) < 1e-4


@pytest.mark.parametrize("args, kw", [((7, 10), {}), ((8, 0), {}), ((8, 10, -1.0), {}),
                                      ((8, 10), dict(scaling={"type": "linear", "factor": 0.0})),
                                      ((8, 10), dict(scaling={"type": "nothing"})),
                                      ((8, 10), dict(scaling={"type": "linear", "factor": 2.0, "orignal": 1}))])
def test_rotary_tables_refuse(args, kw):
    with pytest.raises(ValueError):
        oc.rotary_tables(*args, **kw)


@needs_library
def test_c_abi_refuses_before_any_cuda_call():
    lib = _lib.load()
    zero = ctypes.create_string_buffer(1024)  # a struct of zeros: no pointers, no sizes
    for name in ("oc_rotary_append_paged", "oc_paged_decode_attention", "oc_prompt_attention"):
        fn = getattr(lib, name)
        assert fn(None, None) == 1, name
        assert fn(zero, None) == 1, name
    assert lib.oc_copy_pages(None, None, 1, 16, 4, None, None, 1, None, 148, None) == 1
    assert lib.oc_copy_pages(None, None, 0, 16, 4, None, None, 0, None, 148, None) == 0  # nothing to do
    assert lib.oc_fork_sequences(None, 0, None, 0, None, None, None, None, None, 1, 1, 4, 16, None, None) == 1
    assert lib.oc_fork_sequences(None, 0, None, 0, None, None, None, None, None, 0, 0, 0, 0, None, None) == 1
    assert lib.oc_reserve_pages(None, None, 0, 16, None, 0, None, None, None, 1, 1, 4, 16, None, 0, None, 148,
                                None) == 1
    buf = ctypes.create_string_buffer(64)
    at = ctypes.addressof(buf)
    # too many rows; a workspace that is missing
    assert lib.oc_reserve_pages(None, None, 0, 16, at, 1, at, at, at, 5000, 1, 4, 16, None, 0, None, 148, None) == 5
    assert lib.oc_reserve_pages(None, None, 0, 16, at, 1, at, at, at, 1, 1, 4, 16, None, 0, None, 148, None) == 3
    assert lib.oc_compact_pages(None, None, 0, 16, None, 0, None, 0, at, at, 0, 0, 4, None, 0, None, 148, None) == 1
    assert lib.oc_reserve_workspace_bytes(8, 100) >= 4 * (2 * 8 + 100)
    assert lib.oc_compact_workspace_bytes(100) >= 3 * 4 * 100
    assert lib.oc_paged_decode_workspace_bytes(None) == 0


def _t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


@needs_binding
def test_no_cpu_fallback():
    pos, table = torch.zeros(2, dtype=torch.long), torch.zeros(2, 1, dtype=torch.int32)
    cos = _t(4, 8)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        oc.rotary_embedding(_t(2, 2, 16), pos, cos, cos)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        oc.rotary_append_paged(_t(2, 2, 16), _t(2, 1, 16), _t(2, 1, 16), pos, cos, cos, _t(4, 1, 16, 16),
                               _t(4, 1, 16, 16), table)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        oc.paged_decode_attention(_t(2, 2, 16), _t(4, 1, 16, 16), _t(4, 1, 16, 16), table, table[:, 0])
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        oc.prompt_attention(_t(2, 2, 16), _t(2, 1, 16), _t(2, 1, 16))
    refs = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        oc.fork_sequences(table, table[:, 0], refs, table[:, 0], 16)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        oc.reserve_pages([], table, table[:, 0], refs, table[:, 0], 16)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        oc.compact_pages([], table, refs)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        oc.copy_pages([], table[:, 0], table[:, 0])


@needs_binding
def test_messages_of_the_binding_carry_numbers_and_shapes():
    b, x = _lib.binding(), _t(2, 2, 32)
    with pytest.raises(RuntimeError, match=r"fused_orthocache_attention_v2: invalid argument .*\(code 1\)"):
        b.v2(x[0], x, x, 1.0, 1, 148, torch.float32, None, 0, 0, 0, 0, 0)
    with pytest.raises(ValueError, match="give q, k or both"):
        b.rotary(None, None, None, x, None, None, None, None, None, None, False, False, 1.0, 1.0, False)
    with pytest.raises(TypeError, match="q must be a tensor"):
        b.decode(3, *[x] * 4, None, 0.0, None, 0, 1.0, 1.0, False)


def test_paged_cache_refuses_a_block_size_that_is_no_power_of_two():
    with pytest.raises(ValueError, match="power of 2"):
        oc.PagedKVCache(1, 4, 1, 16, max_seqs=1, max_tokens=16, block_size=24, device="cpu")
