"""Attention of one new token over a paged cache against a plain 64-bit implementation."""

import pytest
import torch

import orthocache_gpu_b200 as oc
from serving_helpers import assert_attention, assert_lse, attend, pages_for

pytestmark = pytest.mark.gpu


def run(lens, HK, G, D, block, dtype, f8=False, softcap=0.0, window=0, alibi=False, seed=0, poison=None, table_cols=0):
    """Calls the operator on random data and compares every output."""
    g = torch.Generator(device="cuda").manual_seed(seed + D + block)
    S = len(lens)
    table, pages = pages_for(lens, block, "cuda", seed=seed)
    if table_cols > table.shape[1]:
        table = torch.cat([table, torch.full((S, table_cols - table.shape[1]), -1, dtype=torch.int32, device="cuda")], 1)
    q = torch.randn(S, HK * G, D, device="cuda", generator=g).to(dtype) * 2
    kc, vc = (torch.randn(pages, HK, block, D, device="cuda", generator=g).to(dtype) for _ in range(2))
    ks, vs = 1.0, 1.0
    if f8:
        kc, vc, ks, vs = (kc * 16).to(torch.float8_e4m3fn), (vc * 16).to(torch.float8_e4m3fn), 1 / 16, 1 / 8
    if poison is not None:  # every slot that no sequence may see
        seen = torch.zeros(pages, block, dtype=torch.bool, device="cuda")
        for i, n in enumerate(lens):
            for j in range(max(0, n - window) if window else 0, n):
                seen[table[i, j // block], j % block] = True
        hidden = ~seen[:, None, :].expand(pages, HK, block)
        for c in (kc, vc):
            if f8:
                c.view(torch.uint8)[hidden] = 0x7F  # NaN
            else:
                c[hidden] = poison
    slopes = 2.0 ** -torch.arange(1, HK * G + 1, device="cuda", dtype=torch.float32) if alibi else None
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, lse = oc.paged_decode_attention(q, kc, vc, table, n, softcap=softcap, alibi_slopes=slopes, window=window,
                                         k_scale=ks, v_scale=vs, return_lse=True)
    oc.check_status()
    assert out.dtype == dtype and out.shape == q.shape and lse.dtype == torch.float32
    product = torch.float16 if f8 and dtype == torch.bfloat16 else dtype
    for i, m in enumerate(lens):
        first = max(0, m - window) if window else 0
        ids = table[i, : -(-m // block)].long()
        flat = [c.double()[ids].transpose(0, 1).reshape(HK, -1, D)[:, first:m] * s for c, s in ((kc, ks), (vc, vs))]
        away = torch.arange(first - m + 1, 1, device="cuda", dtype=torch.float64)[None]
        for h in range(HK):
            rows = slice(h * G, h * G + G)
            bias = slopes[rows, None].double() * away if alibi else torch.zeros(G, m - first, device="cuda", dtype=torch.float64)
            seen = torch.ones(G, m - first, dtype=torch.bool, device="cuda")
            o, size, l, noise = attend(q[i, rows].double(), flat[0][h], flat[1][h], seen, bias, D ** -0.5, softcap)
            what = f"sequence {i} of {m} tokens, kv head {h}"
            assert_attention(out[i, rows], o, size, noise, product, what)
            assert_lse(lse[i, rows], l, noise, what)


LENS = [0, 1, 15, 16, 17, 63, 64, 65, 333, 700]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("HK, G, D, block", [(2, 1, 64, 16), (1, 8, 128, 16), (2, 7, 64, 8), (1, 9, 128, 32),
                                             (1, 20, 64, 64), (2, 4, 256, 16), (1, 12, 256, 8), (1, 2, 80, 128),
                                             (1, 3, 96, 4), (3, 4, 48, 2), (1, 4, 16, 16), (1, 2, 144, 16)])
def test_lengths_groups_and_dims(dtype, f8, HK, G, D, block):
    run(LENS, HK, G, D, block, dtype, f8)


@pytest.mark.parametrize("dtype, f8", [(torch.bfloat16, False), (torch.float16, True), (torch.float32, False)])
@pytest.mark.parametrize("softcap, window, alibi", [(30.0, 0, False), (0.0, 50, False), (0.0, 0, True), (20.0, 100, True),
                                                    (0.0, 1, False)])
def test_score_modifiers(dtype, f8, softcap, window, alibi):
    run([0, 1, 49, 50, 51, 400], 2, 4, 64, 16, dtype, f8, softcap, window, alibi)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("D, block", [(64, 16), (20, 1), (33, 4)])
def test_any_type_and_alignment(dtype, D, block):
    run([0, 1, 30, 333], 2, 3, D, block, dtype, softcap=15.0)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype, f8, D, window", [(torch.bfloat16, False, 128, 0), (torch.float16, False, 64, 37),
                                                  (torch.float16, True, 128, 37), (torch.float32, False, 32, 5)])
def test_slots_that_are_not_seen_have_no_effect(value, dtype, f8, D, window):
    run([1, 17, 100, 257, 600], 2, 2, D, 16, dtype, f8, window=window, poison=value)


def test_split_over_a_long_cache_and_ragged_batches():
    run([20000], 1, 4, 64, 16, torch.bfloat16)
    run([9000, 0, 3, 5000, 0, 1], 2, 2, 128, 32, torch.float16)
    run([40 * (i % 7) for i in range(150)], 1, 2, 64, 16, torch.bfloat16, table_cols=64)   # more sequences than a CTA's threads
    run([2000 + 13 * i for i in range(40)], 2, 4, 64, 16, torch.float16)                  # runs with a finer tail


def test_a_table_wider_than_the_sequences():
    run([5, 300], 2, 4, 64, 16, torch.float16, table_cols=2048)


def test_views_and_other_cache_orders():
    """Queries with strides, caches whose heads are the inner dimension, expanded (broadcast) heads."""
    D, HK, G, block, n = 64, 2, 4, 16, 200
    table, pages = pages_for([n], block, "cuda")
    lens = torch.tensor([n], device="cuda")
    q = torch.randn(1, D, HK * G, device="cuda", dtype=torch.bfloat16).transpose(1, 2)
    kc, vc = (torch.randn(pages, block, HK, D, device="cuda", dtype=torch.bfloat16).transpose(1, 2) for _ in range(2))
    got = oc.paged_decode_attention(q, kc, vc, table, lens)
    want = oc.paged_decode_attention(q.contiguous(), kc.contiguous(), vc.contiguous(), table, lens)
    assert torch.equal(got, want)
    one, two = (c[:, :1].expand(pages, HK, block, D) for c in (kc, vc))
    got = oc.paged_decode_attention(q, one, two, table, lens)
    want = oc.paged_decode_attention(q, one.contiguous(), two.contiguous(), table, lens)
    assert float((got - want).abs().max()) <= 2.0 ** -7 * float(want.abs().max())  # another kernel: one step of the type
    oc.check_status()


def test_visible_nan_and_infinities_stay():
    D, block = 64, 16
    table, pages = pages_for([40, 40, 40], block, "cuda")
    q = torch.ones(3, 2, D, device="cuda", dtype=torch.float16)
    kc, vc = (torch.randn(pages, 1, block, D, device="cuda", dtype=torch.float16) for _ in range(2))
    kc[table[0, 1], 0, 3, 0] = float("nan")
    vc[table[1, 2], 0, 7, 5] = float("inf")
    out = oc.paged_decode_attention(q, kc, vc, table, torch.tensor([40, 40, 40], device="cuda"))
    assert out[0].isnan().all() and out[1, :, 5].isinf().all() and out[1, :, :5].isfinite().all() and out[2].isfinite().all()


def test_the_result_does_not_change_from_call_to_call_and_graphs_replay():
    lens = [3000, 1, 700]
    table, pages = pages_for(lens, 16, "cuda")
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn(3, 8, 128, device="cuda", dtype=torch.bfloat16)
    kc, vc = (torch.randn(pages, 2, 16, 128, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    want = oc.paged_decode_attention(q, kc, vc, table, n)
    for _ in range(5):
        assert torch.equal(oc.paged_decode_attention(q, kc, vc, table, n), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        oc.paged_decode_attention(q, kc, vc, table, n)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            got = oc.paged_decode_attention(q, kc, vc, table, n)
    n.copy_(torch.tensor([100, 0, 699], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, oc.paged_decode_attention(q, kc, vc, table, n))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_lengths_and_pages_outside_are_reported(dtype):
    table, pages = pages_for([40, 40], 16, "cuda")
    q = torch.randn(2, 2, 64, device="cuda", dtype=dtype)
    kc = torch.randn(pages, 1, 16, 64, device="cuda", dtype=dtype)
    for lens in ([40, -1], [40, 1000]):
        oc.paged_decode_attention(q, kc, kc, table, torch.tensor(lens, device="cuda"))
        with pytest.raises(RuntimeError, match="outside its tables"):
            oc.check_status()
    bad = table.clone()
    bad[1, 1] = -1
    out = oc.paged_decode_attention(q, kc, kc, bad, torch.tensor([40, 40], device="cuda"))
    with pytest.raises(RuntimeError, match="block-table entry"):
        oc.check_status()
    want = oc.paged_decode_attention(q, kc, kc, table, torch.tensor([40, 40], device="cuda"))
    assert torch.equal(out[0], want[0])  # the other sequence is right


def test_refusals():
    q = torch.zeros(2, 4, 64, device="cuda", dtype=torch.float16)
    c = torch.zeros(4, 2, 16, 64, device="cuda", dtype=torch.float16)
    table, lens = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    for err, args, kw in [(ValueError, (q[0], c, c, table, lens), {}), (ValueError, (q[:, :3], c, c, table, lens), {}),
                          (ValueError, (q, c, c[:2], table, lens), {}), (TypeError, (q, c, c.float(), table, lens), {}),
                          (TypeError, (q, c.bfloat16(), c.bfloat16(), table, lens), {}),
                          (TypeError, (q.double(), c, c, table, lens), {}), (ValueError, (q, c, c, table[:1], lens), {}),
                          (ValueError, (q, c, c, table, lens[:1]), {}), (TypeError, (q, c, c, table, lens.float()), {}),
                          (ValueError, (q, c, c, table, lens), dict(softcap=-1.0)),
                          (ValueError, (q, c, c, table, lens), dict(window=-1)),
                          (ValueError, (q, c, c, table, lens), dict(k_scale=2.0)),
                          (ValueError, (q, c, c, table, lens), dict(alibi_slopes=torch.ones(3, device="cuda"))),
                          (TypeError, (q, c, c, table, lens), dict(alibi_slopes=torch.ones(4, device="cuda").half())),
                          (RuntimeError, (q, c.cpu(), c.cpu(), table, lens), {}),
                          (RuntimeError, (q.clone().requires_grad_(), c, c, table, lens), {})]:
        with pytest.raises(err):
            oc.paged_decode_attention(*args, **kw)
    wide = torch.zeros(2, 4, 264, device="cuda", dtype=torch.float16)
    with pytest.raises(ValueError, match="between 1 and 256"):
        oc.paged_decode_attention(wide, torch.zeros(4, 2, 16, 264, device="cuda", dtype=torch.float16),
                                  torch.zeros(4, 2, 16, 264, device="cuda", dtype=torch.float16), table, lens)
    assert oc.paged_decode_attention(q[:0], c, c, table[:0], lens[:0]).shape == (0, 4, 64)
