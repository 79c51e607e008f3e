"""Windows and prefixes at the ends of their range: what they leave visible, exactly as a mask says."""

import pytest
import torch

import orthocache_gpu_b200 as oc

pytestmark = pytest.mark.gpu


def _data(T, TK, D, dtype):
    g = torch.Generator(device="cuda").manual_seed(T + D)
    return [torch.randn(n, h, D, device="cuda", generator=g).to(dtype) for n, h in ((T, 4), (TK, 2), (TK, 2))]


def _ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype, D", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 40)])
@pytest.mark.parametrize("cu, cu_k", [((0, 300), (0, 90)), ((0, 200, 500), (0, 200, 230)), ((0, 20), (0, 7)), ((0, 300), (0, 300))])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [500, 2 ** 31 - 101, 2 ** 31 - 1])
def test_a_window_that_hides_nothing(dtype, D, cu, cu_k, causal, window):
    """Queries before the first key too: with fewer keys than queries their positions are negative."""
    q, k, v = _data(cu[-1], cu_k[-1], D, dtype)
    kw = dict(cu_seqlens_k=_ints(*cu_k), causal=causal, return_lse=True)
    want = oc.prompt_attention(q, k, v, _ints(*cu), **kw)
    got = oc.prompt_attention(q, k, v, _ints(*cu), window=window, **kw)
    oc.check_status()
    if not causal:
        assert want[1].isfinite().all()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype, D", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 40)])
@pytest.mark.parametrize("prefix", [-1, -500, -2 ** 31])
@pytest.mark.parametrize("window", [0, 40])
def test_a_negative_prefix_is_none(dtype, D, prefix, window):
    q, k, v = _data(500, 500, D, dtype)
    want = oc.prompt_attention(q, k, v, _ints(0, 200, 500), window=window, prefix_lens=_ints(0, 0), return_lse=True)
    got = oc.prompt_attention(q, k, v, _ints(0, 200, 500), window=window, prefix_lens=_ints(prefix, prefix), return_lse=True)
    oc.check_status()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
