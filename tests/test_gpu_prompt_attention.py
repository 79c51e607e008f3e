"""Attention of packed prompts against a plain 64-bit implementation."""

import pytest
import torch

import orthocache_gpu_b200 as oc
from serving_helpers import assert_attention, assert_lse, attend

pytestmark = pytest.mark.gpu


def data(cu, cu_k, HK, G, D, dtype, seed=0, spare=0):
    g = torch.Generator(device="cuda").manual_seed(seed + D + cu[-1])
    T, TK = cu[-1] + spare, (cu_k or cu)[-1] + spare
    q = torch.randn(T, HK * G, D, device="cuda", generator=g).to(dtype) * 2
    k, v = (torch.randn(TK, HK, D, device="cuda", generator=g).to(dtype) for _ in range(2))
    return q, k, v


def masks(n, m, causal, prefix, window):
    p, j = torch.arange(n, device="cuda")[:, None] + m - n, torch.arange(m, device="cuda")[None]
    seen = (j <= p) if causal else torch.ones(n, m, dtype=torch.bool, device="cuda")
    if window:
        seen = seen & (j > p - window)
    return seen | (j < prefix), (p - j).abs().double()


def run(cu, HK, G, D, dtype, cu_k=None, causal=True, prefix=None, window=0, softcap=0.0, alibi=False, scale=None, spare=0,
        q=None, k=None, v=None):
    if q is None:
        q, k, v = data(cu, cu_k, HK, G, D, dtype, spare=spare)
    slopes = 2.0 ** -torch.arange(1, HK * G + 1, device="cuda", dtype=torch.float32) if alibi else None
    ints = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    out, lse = oc.prompt_attention(q, k, v, ints(cu), cu_seqlens_k=ints(cu_k), causal=causal, prefix_lens=ints(prefix),
                                   window=window, scale=scale, softcap=softcap, alibi_slopes=slopes, return_lse=True)
    oc.check_status()
    assert out.dtype == dtype and out.shape == q.shape and lse.shape == q.shape[:2]
    ck = cu_k or cu
    for d in range(len(cu) - 1):
        rows, keys = slice(cu[d], cu[d + 1]), slice(ck[d], ck[d + 1])
        n, m = cu[d + 1] - cu[d], ck[d + 1] - ck[d]
        seen, away = masks(n, m, causal, prefix[d] if prefix else 0, window)
        for h in range(HK * G):
            bias = -slopes[h].double() * away if alibi else torch.zeros_like(away)
            o, size, l, noise = attend(q[rows, h].double(), k[keys, h // G].double(), v[keys, h // G].double(), seen, bias,
                                D ** -0.5 if scale is None else scale, softcap)
            assert_attention(out[rows, h], o, size, noise, dtype, f"document {d}, head {h}")
            assert_lse(lse[rows, h], l, noise, f"document {d}, head {h}")
    outside = torch.ones(q.shape[0], dtype=torch.bool, device="cuda")
    outside[cu[0]:cu[-1]] = False
    assert not out[outside].any() and bool(lse[outside].isneginf().all())
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [8, 64, 72, 80, 96, 128])
@pytest.mark.parametrize("cu", [[0, 1], [0, 128], [0, 129], [0, 300], [0, 1, 1, 78, 206, 700], [3, 260, 517]])
def test_dims_and_documents(dtype, D, cu):
    run(cu, 2, 2, D, dtype, spare=2)


@pytest.mark.parametrize("dtype, D", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 40)])
@pytest.mark.parametrize("kw", [dict(causal=False), dict(window=1), dict(window=100), dict(causal=False, window=130),
                                dict(prefix=[0, 50, 300]), dict(prefix=[1, 20, 400], window=64), dict(softcap=20.0),
                                dict(softcap=2.0), dict(alibi=True), dict(alibi=True, causal=False),
                                dict(alibi=True, softcap=30.0, window=90, prefix=[0, 130, 10]), dict(scale=-0.2),
                                dict(scale=0.0), dict(scale=1.5)])
def test_masks_and_scores(dtype, D, kw):
    run([0, 70, 330, 700], 1, 3, D, dtype, **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cu, cu_k", [([0, 10, 200], [0, 300, 500]), ([0, 130, 131], [0, 40, 41]), ([0, 5, 150], [0, 0, 600]),
                                      ([0, 0, 260], [0, 100, 100])])
@pytest.mark.parametrize("causal", [True, False])
def test_keys_of_another_length(dtype, cu, cu_k, causal):
    """More keys than queries (a cached prefix), fewer (rows that see nothing), none."""
    run(cu, 1, 2, 64, dtype, cu_k=cu_k, causal=causal)


@pytest.mark.parametrize("G, HK", [(1, 3), (7, 1), (5, 2)])
def test_groups(G, HK):
    run([0, 200, 391], HK, G, 64, torch.float16)


def test_one_document_by_default_and_long_sums():
    q, k, v = data([0, 3001], None, 1, 2, 128, torch.bfloat16)
    out = run([0, 3001], 1, 2, 128, torch.bfloat16, q=q, k=k, v=v)
    assert torch.equal(out, oc.prompt_attention(q, k, v))
    run([0, 4500], 1, 1, 64, torch.float16, window=1000)


@pytest.mark.parametrize("dtype, D", [(torch.bfloat16, 64), (torch.float16, 56)])
@pytest.mark.parametrize("cu, kw", [([0, 4353], {}), ([2, 4300], dict(softcap=30.0, alibi=True)), ([0, 8200, 8230], {}),
                                    ([0, 4133], dict(prefix=[200], window=4100)), ([0, 4224], dict(causal=False))])
def test_long_documents_of_narrow_heads(dtype, D, cu, kw):
    """Documents of more than 4096 tokens on average take two query tiles a CTA where shorter ones take one."""
    run(cu, 1, 2, D, dtype, spare=1, **kw)


@pytest.mark.parametrize("dtype, D", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 24)])
def test_hidden_nan_and_infinities_have_no_effect(dtype, D):
    cu = [0, 150, 400]
    q, k, v = data(cu, None, 2, 2, D, dtype)
    clean = oc.prompt_attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"))
    k2, v2 = k.clone(), v.clone()
    k2[149], v2[149] = float("nan"), float("inf")   # the last token of the first document
    v2[390, 0, 3] = float("-inf")                   # seen by the last ten rows of two heads
    got = run(cu, 2, 2, D, dtype, q=q, k=k2, v=v2)
    assert got[:149].isfinite().all() and got[150:390].isfinite().all()
    assert got[149].isnan().all() and bool(got[390:, :2, 3].isinf().all()) and got[390:, 2:].isfinite().all()
    assert float((got[:149] - clean[:149]).abs().max()) <= 2.0 ** -6 * float(clean[:149].abs().max())


def test_scores_far_apart_and_of_the_lowest_value():
    """Maxima that grow from tile to tile by more than the lazy rescaling allows, and all but one key far below."""
    T, D = 700, 64
    q = torch.full((T, 1, D), 4.0, device="cuda", dtype=torch.float16)
    k = torch.zeros(T, 1, D, device="cuda", dtype=torch.float16)
    k[:, 0, 0] = torch.linspace(-60000, 60000, T, device="cuda").half()
    v = torch.randn(T, 1, D, device="cuda", dtype=torch.float16)
    run([0, T], 1, 1, D, torch.float16, q=q, k=k, v=v, scale=1e-3)
    run([0, T], 1, 1, D, torch.float16, q=q, k=k.flip(0), v=v, scale=1e-3)


def test_views_and_orders():
    cu = torch.tensor([0, 100, 260], dtype=torch.int32, device="cuda")
    qkv = torch.randn(260, 8, 64, device="cuda", dtype=torch.bfloat16)
    want = oc.prompt_attention(qkv[:, :4].contiguous(), qkv[:, 4:6].contiguous(), qkv[:, 6:].contiguous(), cu)
    assert torch.equal(oc.prompt_attention(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], cu), want)
    head_major = qkv.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(oc.prompt_attention(head_major[:, :4], head_major[:, 4:6], head_major[:, 6:], cu), want)
    assert torch.equal(oc.prompt_attention(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], cu.long()), want)
    odd = torch.randn(260 * 8 * 64 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(260, 8, 64)  # not 16-byte aligned
    odd.copy_(qkv)
    got = oc.prompt_attention(odd[:, :4], odd[:, 4:6], odd[:, 6:], cu)
    assert float((got - want).abs().max()) <= 2.0 ** -6 * float(want.abs().max())
    columns = qkv.transpose(1, 2).contiguous().transpose(1, 2)  # the last dimension is not contiguous
    assert torch.equal(oc.prompt_attention(columns[:, :4], columns[:, 4:6], columns[:, 6:], cu), want)


def test_documents_outside_are_reported():
    q, k, v = data([0, 64], None, 1, 1, 64, torch.float16)
    for cu in ([0, 40, 20], [0, 70], [-1, 10]):
        oc.prompt_attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"))
        with pytest.raises(RuntimeError, match="outside its tables"):
            oc.check_status()


def test_refusals():
    q, k, v = data([0, 64], None, 2, 2, 64, torch.float16)
    cu = torch.tensor([0, 64], dtype=torch.int32, device="cuda")
    for err, args, kw in [(ValueError, (q[0], k, v), {}), (ValueError, (q, k, v[:5]), {}), (ValueError, (q[:, :3], k, v), {}),
                          (TypeError, (q, k.float(), v), {}), (TypeError, (q.double(), k.double(), v.double()), {}),
                          (ValueError, (q, k[:5], v[:5], cu), {}), (ValueError, (q, k, v), dict(cu_seqlens_k=cu)),
                          (ValueError, (q, k, v, cu), dict(cu_seqlens_k=cu[:1])), (ValueError, (q, k, v, cu[:0]), {}),
                          (TypeError, (q, k, v, cu.float()), {}), (ValueError, (q, k, v, cu), dict(prefix_lens=cu)),
                          (ValueError, (q, k, v), dict(window=-1)), (ValueError, (q, k, v), dict(softcap=-1.0)),
                          (ValueError, (q, k, v), dict(alibi_slopes=torch.ones(3, device="cuda"))),
                          (ValueError, (q[..., :20], k[..., :20], v[..., :20]), {}), (RuntimeError, (q, k.cpu(), v), {}),
                          (RuntimeError, (q, k, v.clone().requires_grad_()), {})]:
        with pytest.raises(err):
            oc.prompt_attention(*args, **kw)
    wide = torch.zeros(4, 2, 136, device="cuda", dtype=torch.float16)
    with pytest.raises(ValueError, match="multiple of 8 up to 128"):
        oc.prompt_attention(wide, wide, wide)
    assert oc.prompt_attention(q[:0], k, v).shape == (0, 4, 64)
    assert not oc.prompt_attention(q, k[:0], v[:0]).any()
