"""The forms of the serving kernels that small inputs do not reach, against 64-bit formulas.

Decode: a batch of 24 places (tiles, and 3 for each unit) or more for every resident CTA, 4 an SM of 148 at 64 columns
in 16 bits, 14208, has a finer tail; more than 32 sequences are found by the whole CTA, more than 128 in several
rounds; units of up to 8 tiles at the table's width go to a CTA each, so tables are wider than the sequences here.
Rotary: a token for each of 16 warps of 148 SMs, 2368, and the heads of a projection longer than 4096 bytes a token,
or apart.
"""

import random

import pytest
import torch

import orthocache_gpu_b200 as oc
from serving_helpers import pages_for
from test_gpu_paged_decode import run
from test_gpu_rotary import check, turned

pytestmark = pytest.mark.gpu


def _places(lens, units, keys=128):
    return sum(units * (max(1, -(-n // keys)) + 3) for n in lens)


@pytest.mark.parametrize("kw", [{}, dict(softcap=30.0, alibi=True), dict(window=1000)])
def test_decode_of_many_sequences_with_a_finer_tail(kw):
    """Three rounds of the search, half of the sequences of a tile or none."""
    rng = random.Random(1)
    lens = [rng.choice([0, rng.randint(1, 128), rng.randint(1, 700)]) for _ in range(297)] + [1280, 1, 1100]
    assert _places(lens, 16) >= 14208
    run(lens, 16, 2, 64, 16, torch.float16, table_cols=80, **kw)


def test_decode_of_few_long_sequences_with_a_finer_tail():
    lens = [4200 - 97 * i for i in range(16)]
    lens[5] = 0
    assert _places(lens, 32) >= 14208
    run(lens, 32, 1, 64, 32, torch.bfloat16)


@pytest.mark.parametrize("S", [33, 128, 129, 260])
@pytest.mark.parametrize("HK, G, D, dtype, f8", [(2, 3, 128, torch.bfloat16, True), (1, 4, 256, torch.bfloat16, False),
                                                 (1, 12, 64, torch.float16, False), (2, 1, 80, torch.float16, True)])
def test_decode_of_many_sequences_that_are_split(S, HK, G, D, dtype, f8):
    rng = random.Random(S)
    run([rng.choice([0, 1, rng.randint(1, 1500)]) for _ in range(S)], HK, G, D, 16, dtype, f8, table_cols=200, softcap=20.0)


@pytest.mark.parametrize("HQ, HK, D, R, apart", [(32, 8, 128, 128, False), (20, 4, 80, 32, False), (24, 2, 96, 96, False),
                                                 (3, 2, 64, 64, True), (2, 1, 256, 128, True), (1, 1, 40, 16, True)])
@pytest.mark.parametrize("dtype, f8", [(torch.bfloat16, False), (torch.float16, True), (torch.float32, False), (torch.float32, True)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T, return_keys", [(2371, True), (5000, False)])
def test_rotary_of_prompts_whose_tokens_are_several_pieces(HQ, HK, D, R, apart, dtype, f8, interleaved, T, return_keys):
    g = torch.Generator(device="cuda").manual_seed(T + D)
    qkv = torch.randn(T, HQ + 2 * HK, D, device="cuda", generator=g).to(dtype)
    q, k, v = qkv[:, :HQ], qkv[:, HQ:HQ + HK], qkv[:, HQ + HK:]
    if apart:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    block, half = 32, T // 2
    table, pages = pages_for([half, T - half], block, "cuda")
    seq = (torch.arange(T, device="cuda") >= half).int()
    pos = torch.arange(T, device="cuda") - seq * half
    place = seq.clone()
    place[::7] = -1  # not kept
    kept = (place >= 0).nonzero()[:, 0]
    kind = torch.float8_e4m3fn if f8 else dtype
    kc, vc = (torch.zeros(pages, HK, block, D, device="cuda", dtype=kind) for _ in range(2))
    cos, sin = oc.rotary_tables(R, T, device="cuda")
    ks, vs = (0.25, 0.3) if f8 else (1.0, 1.0)
    got = oc.rotary_append_paged(q, k, v, pos, cos, sin, kc, vc, table, seq_ids=place, interleaved=interleaved, k_scale=ks,
                                 v_scale=vs, return_keys=return_keys)
    oc.check_status()
    ky, ksize = turned(k, cos, sin, pos, R, interleaved)
    if return_keys:
        check(got[1], ky, ksize, what="k")
        got = got[0]
    check(got, *turned(q, cos, sin, pos, R, interleaved), what="q")
    bits = (lambda c: c.view(torch.uint8)) if f8 else (lambda c: c)
    page, slot = table[seq[kept].long(), pos[kept] // block].long(), pos[kept] % block
    check(bits(kc)[page, :, slot].view(kind), ky[kept], ksize[kept], ks * (1 + 2.0 ** -23) if f8 else 1.0, "k cache")
    vv = v[kept].double()
    check(bits(vc)[page, :, slot].view(kind), vv, vv.abs(), vs, "v cache")
    untouched = torch.ones(pages, block, dtype=torch.bool, device="cuda")
    untouched[page, slot] = False
    assert not bits(kc)[untouched[:, None].expand(pages, HK, block)].any() and not bits(vc)[untouched[:, None].expand(pages, HK, block)].any()


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("H, D, R", [(40, 128, 64), (7, 96, 96)])
def test_rotary_embedding_of_prompts(H, D, R, inverse):
    x = torch.randn(2500, H, D, device="cuda", dtype=torch.bfloat16)
    cos, sin = oc.rotary_tables(R, 2500, device="cuda")
    pos = torch.randperm(2500, device="cuda")
    check(oc.rotary_embedding(x, pos, cos, sin, inverse=inverse), *turned(x, cos, sin, pos, R, False, inverse), what="x")
