"""Visible scores of -inf: a row of nothing else is NaN (0 / 0), and 0 times an infinite value is NaN."""

import pytest
import torch

import orthocache_gpu_b200 as oc
from serving_helpers import assert_attention, assert_lse, attend, pages_for

pytestmark = pytest.mark.gpu
INF = float("inf")


def _mark(k, v, keys, heads, special):
    """Keys of -inf in column 0 (queries have a positive one): scores of -inf; `special`: their values' column 3."""
    k[keys, heads, 0] = -INF
    if special is not None:
        v[keys, heads, 3] = special


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("special", [None, INF, float("nan")])
@pytest.mark.parametrize("lens, D, cols, window", [([40, 1, 0, 300], 64, 0, 0), ([300, 40], 128, 0, 33), ([40, 300], 256, 0, 0),
                                                   ([1500, 12000, 5], 64, 0, 0), ([700, 30], 128, 4096, 100), ([333, 0], 20, 0, 0)])
def test_decode(dtype, special, lens, D, cols, window):
    """Sequences whose every key, whose first half, and whose last key has a score of -inf; two kv heads, one marked."""
    block, HK, G = 16, 2, 2
    table, pages = pages_for(lens, block, "cuda")
    if cols > table.shape[1]:
        table = torch.cat([table, torch.full((len(lens), cols - table.shape[1]), -1, dtype=torch.int32, device="cuda")], 1)
    n = torch.tensor(lens, device="cuda")
    for part in (slice(None), slice(0.5), slice(-1, None)):
        g = torch.Generator(device="cuda").manual_seed(D)
        q = torch.rand(len(lens), HK * G, D, device="cuda", generator=g).to(dtype) + 0.25
        flat = [[torch.randn(m, HK, D, device="cuda", generator=g).to(dtype) for m in lens] for _ in range(2)]
        kc, vc = (torch.zeros(pages, HK, block, D, device="cuda", dtype=dtype) for _ in range(2))
        for i, m in enumerate(lens):
            keys = slice(0, m // 2) if part.stop == 0.5 else part
            _mark(flat[0][i], flat[1][i], keys, slice(0, 1), special)
            j = torch.arange(m, device="cuda")
            for c, x in zip((kc, vc), flat):
                c[table[i, j // block].long(), :, j % block] = x[i]
        out, lse = oc.paged_decode_attention(q, kc, vc, table, n, window=window, return_lse=True)
        oc.check_status()
        for i, m in enumerate(lens):
            first = max(0, m - window) if window else 0
            for h in range(HK):
                rows = slice(h * G, h * G + G)
                seen = torch.ones(G, m - first, dtype=torch.bool, device="cuda")
                o, size, l, noise = attend(q[i, rows].double(), flat[0][i][first:, h].double(), flat[1][i][first:, h].double(),
                                           seen, torch.zeros_like(seen, dtype=torch.float64), D ** -0.5, 0.0)
                what = f"sequence {i} of {m} tokens, kv head {h}, marked {part}"
                assert_attention(out[i, rows], o, size, noise, dtype, what)
                assert_lse(lse[i, rows], l, noise, what)


@pytest.mark.parametrize("dtype, D", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float16, 40), (torch.float32, 48)])
@pytest.mark.parametrize("special", [None, INF])
@pytest.mark.parametrize("cu", [[0, 20], [0, 140, 430], [0, 4400]])
@pytest.mark.parametrize("kw", [{}, dict(window=7), dict(prefix=3), dict(causal=False), dict(window=7, prefix=3)])
def test_prompt(dtype, D, special, cu, kw):
    """The first keys of every document, and a stretch longer than the window, have scores of -inf for one kv head."""
    HK, G, T = 2, 2, cu[-1]
    g = torch.Generator(device="cuda").manual_seed(D + T)
    q = torch.rand(T, HK * G, D, device="cuda", generator=g).to(dtype) + 0.25
    k, v = (torch.randn(T, HK, D, device="cuda", generator=g).to(dtype) for _ in range(2))
    for d in range(len(cu) - 1):
        n = cu[d + 1] - cu[d]
        for keys in (slice(cu[d], cu[d] + 5), slice(cu[d] + n // 2, cu[d] + n // 2 + 9)):
            _mark(k, v, keys, slice(0, 1), special)
    window, prefix, causal = kw.get("window", 0), kw.get("prefix", 0), kw.get("causal", True)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    out, lse = oc.prompt_attention(q, k, v, ints(cu), causal=causal, window=window, return_lse=True,
                                   prefix_lens=ints([prefix] * (len(cu) - 1)) if prefix else None)
    oc.check_status()
    for d in range(len(cu) - 1):
        rows, n = slice(cu[d], cu[d + 1]), cu[d + 1] - cu[d]
        p, j = torch.arange(n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
        seen = (j <= p) if causal else torch.ones(n, n, dtype=torch.bool, device="cuda")
        if window:
            seen = seen & (j > p - window)
        seen = seen | (j < prefix)
        for h in range(HK * G):
            qd, kd, vd = q[rows, h].double(), k[rows, h // G].double(), v[rows, h // G].double()
            what = f"document {d}, head {h}"
            picked = torch.arange(n, device="cuda") if n < 500 else torch.cat(
                [torch.arange(0, 20), torch.arange(n // 2 - 3, n // 2 + 20), torch.arange(n - 130, n, 7)]).cuda()
            o, size, l, noise = attend(qd[picked], kd, vd, seen[picked], torch.zeros(picked.numel(), n, device="cuda", dtype=torch.float64),
                                       D ** -0.5, 0.0)
            assert_attention(out[rows, h][picked], o, size, noise, dtype, what)
            assert_lse(lse[rows, h][picked], l, noise, what)
    if not window and causal and not prefix:
        assert out[cu[0], :G].isnan().all() and out[cu[0], G:].isfinite().all()
