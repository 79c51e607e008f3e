"""Rotary embedding and the append to the paged cache against 64-bit formulas.

y = x_a c - x_b s in float32: two products and a sum, each rounded to 2^-24 relative, then one rounding to the
output's type: |error| <= 3 2^-24 (|x_a c| + |x_b s|) + u |y|; the spacing of float16's smallest numbers and,
for 8 bits, u = 2^-4 and 2^-10 (half the smallest spacing), saturated at 448.
"""

import pytest
import torch

import orthocache_gpu_b200 as oc
from serving_helpers import pages_for

pytestmark = pytest.mark.gpu
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float8_e4m3fn: 2.0 ** -4}
SMALL = {torch.float32: 1e-38, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-38, torch.float8_e4m3fn: 2.0 ** -10}


def turned(x, cos, sin, positions, rotary_dim, interleaved, inverse=False):
    """(y, |x_a c| + |x_b s|) in 64 bits."""
    x = x.double()
    y, size = x.clone(), x.abs()
    half = rotary_dim // 2
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    c, s = cos.double()[positions][:, None], sin.double()[positions][:, None] * (-1 if inverse else 1)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    size[..., a] = (x[..., a] * c).abs() + (x[..., b] * s).abs()
    size[..., b] = (x[..., b] * c).abs() + (x[..., a] * s).abs()
    return y, size


def check(got, y, size, scale=1.0, what=""):
    y, size = y / scale, size / scale
    if got.dtype == torch.float8_e4m3fn:
        y = y.clamp(-448, 448)
    tol = 4 * 2.0 ** -24 * size + U[got.dtype] * y.abs() + SMALL[got.dtype]
    over = ((got.double() - y).abs() - tol).max()
    assert float(over) <= 0, f"{what}: {float(over):.3g}"


CASES = [  # tokens, q heads, kv heads, head_dim, rotary_dim
    (1, 8, 2, 64, 64), (5, 3, 1, 64, 32), (33, 8, 8, 128, 128), (7, 4, 2, 80, 32), (9, 2, 2, 96, 96),
    (4, 6, 2, 48, 10), (3, 2, 1, 17, 6), (2500, 8, 2, 64, 64), (2500, 5, 1, 128, 64), (6, 2, 1, 256, 128), (0, 4, 2, 64, 64)]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("f8", [False, True])
def test_rotates_and_appends(case, dtype, interleaved, f8):
    T, HQ, HK, D, R = case
    g = torch.Generator(device="cuda").manual_seed(T + D)
    qkv = torch.randn(T, HQ + 2 * HK, D, device="cuda", generator=g).to(dtype)
    q, k, v = qkv[:, :HQ], qkv[:, HQ:HQ + HK], qkv[:, HQ + HK:]  # views with strides
    block, seqs = 16, 3
    lens = [T // 2 + 1, T - T // 2 + 4, 0]
    table, pages = pages_for(lens, block, "cuda")
    seq = torch.arange(T, device="cuda", dtype=torch.int32) % 2
    pos = torch.arange(T, device="cuda") // 2
    if T > 2:
        seq[1] = -1  # this token is not kept
    cache_dtype = torch.float8_e4m3fn if f8 else dtype
    kc = torch.randn(pages, HK, block, D, device="cuda", generator=g).to(cache_dtype)
    vc = torch.randn(pages, HK, block, D, device="cuda", generator=g).to(cache_dtype)
    k0, v0 = kc.double(), vc.double()
    ks, vs = (0.25, 0.3) if f8 else (1.0, 1.0)
    cos, sin = oc.rotary_tables(R, 2000, device="cuda")
    out, keys = oc.rotary_append_paged(q, k, v, pos, cos, sin, kc, vc, table, seq_ids=seq, interleaved=interleaved,
                                       k_scale=ks, v_scale=vs, return_keys=True)
    oc.check_status()
    assert out.dtype == dtype and out.shape == q.shape and keys.shape == k.shape
    if T == 0:
        return
    check(out, *turned(q, cos, sin, pos, R, interleaved), what="q")
    ky, ksize = turned(k, cos, sin, pos, R, interleaved)
    check(keys, ky, ksize, what="k")
    kept = (seq >= 0).nonzero()[:, 0]
    page, slot = table[seq[kept].long(), pos[kept] // block].long(), pos[kept] % block
    as_bytes = (lambda c: c.view(torch.uint8)) if f8 else (lambda c: c)
    check(as_bytes(kc)[page, :, slot].view(cache_dtype), ky[kept], ksize[kept], ks * (1 + 2.0 ** -23) if f8 else 1.0, "k cache")
    vv = v[kept].double()
    check(as_bytes(vc)[page, :, slot].view(cache_dtype), vv, vv.abs(), vs, "v cache")
    if not f8:
        assert torch.equal(as_bytes(vc)[page, :, slot], v[kept])  # copied
    # nothing else changed
    touched = torch.zeros(pages, block, dtype=torch.bool, device="cuda")
    touched[page, slot] = True
    other = ~touched[:, None, :].expand(pages, HK, block)
    assert torch.equal(kc.double()[other], k0[other]) and torch.equal(vc.double()[other], v0[other])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("pos_dtype", [torch.int32, torch.int64])
def test_inverse_is_the_gradient(interleaved, pos_dtype):
    """The inverse turn is the transposed map: the formula's gradient, and what differences give."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(6, 2, 32, device="cuda", generator=g)
    w = torch.randn(6, 2, 32, device="cuda", generator=g)  # d loss / d y
    cos, sin = oc.rotary_tables(24, 50, device="cuda")
    pos = torch.tensor([0, 3, 49, 7, 7, 1], device="cuda", dtype=pos_dtype)
    grad = oc.rotary_embedding(w, pos, cos, sin, interleaved=interleaved, inverse=True)
    check(grad, *turned(w, cos, sin, pos.long(), 24, interleaved, inverse=True), what="formula")
    xd = x.double().requires_grad_()
    turned(xd, cos, sin, pos.long(), 24, interleaved)[0].backward(w.double())
    assert float((grad.double() - xd.grad).abs().max()) <= 6 * 2.0 ** -24 * 8  # |w| below 8
    # the map is linear: a difference along one column is exact up to rounding
    step = torch.zeros_like(x)
    step[2, 1, 5] = 1.0
    up, down = (oc.rotary_embedding(x + s * step, pos, cos, sin, interleaved=interleaved) for s in (1, -1))
    slope = float(((up - down).double() / 2 * w.double()).sum())
    assert abs(slope - float(grad[2, 1, 5])) <= 64 * 2.0 ** -24 * 16


def test_appends_without_rotating():
    table, pages = pages_for([5, 9], 8, "cuda")
    k, v = (torch.randn(2, 3, 40, device="cuda", dtype=torch.float16) for _ in range(2))
    kc, vc = (torch.zeros(pages, 3, 8, 40, device="cuda", dtype=torch.float16) for _ in range(2))
    pos = torch.tensor([4, 8], device="cuda")
    assert oc.rotary_append_paged(None, k, v, pos, None, None, kc, vc, table) is None
    oc.check_status()
    for i in range(2):
        page, slot = int(table[i, int(pos[i]) // 8]), int(pos[i]) % 8
        assert torch.equal(kc[page, :, slot], k[i]) and torch.equal(vc[page, :, slot], v[i])


def test_token_major_caches_and_unaligned_views():
    """Caches whose heads are the inner dimension, and inputs that start at an odd element."""
    T, H, D = 20, 2, 64
    flat = torch.randn(T * 3 * H * D + 1, device="cuda", dtype=torch.bfloat16)[1:]
    qkv = flat.view(T, 3 * H, D)
    table, pages = pages_for([T], 4, "cuda")
    kc = torch.zeros(pages, 4, H, D, device="cuda", dtype=torch.bfloat16).transpose(1, 2)
    vc = torch.zeros_like(kc)
    cos, sin = oc.rotary_tables(D, T, device="cuda")
    pos = torch.arange(T, device="cuda")
    q = oc.rotary_append_paged(qkv[:, :H], qkv[:, H:2 * H], qkv[:, 2 * H:], pos, cos, sin, kc, vc, table,
                               seq_ids=torch.zeros(T, device="cuda", dtype=torch.int32))
    oc.check_status()
    check(q, *turned(qkv[:, :H], cos, sin, pos, D, False), what="q")
    ids = table[0].long()
    check(kc[ids].transpose(1, 2).reshape(-1, H, D)[:T], *turned(qkv[:, H:2 * H], cos, sin, pos, D, False), what="k")
    assert torch.equal(vc[ids].transpose(1, 2).reshape(-1, H, D)[:T], qkv[:, 2 * H:])


@pytest.mark.parametrize("T", [4, 4000])
@pytest.mark.parametrize("bad", ["negative", "table", "column", "page", "sequence"])
def test_places_outside_are_reported_and_skipped(T, bad):
    """T: the kernel for steps, and the one for prompts."""
    D, block = 64, 16
    table, pages = pages_for([T], block, "cuda")
    kc = torch.zeros(pages, 1, block, D, device="cuda", dtype=torch.float16)
    vc = torch.zeros_like(kc)
    x = torch.ones(T, 1, D, device="cuda", dtype=torch.float16)
    pos, seq = torch.arange(T, device="cuda"), torch.zeros(T, device="cuda", dtype=torch.int32)
    cos, sin = oc.rotary_tables(D, T + block * 4 if bad == "column" else T, device="cuda")
    slot = (int(table[0, (T - 1) // block]), (T - 1) % block)
    if bad == "page":
        table[0, (T - 1) // block] = pages
    elif bad == "sequence":
        seq[T - 1] = 1
    else:
        pos[T - 1] = {"negative": -1, "table": T, "column": table.shape[1] * block}[bad]
    oc.rotary_append_paged(x, x, x, pos, cos, sin, kc, vc, table, seq_ids=seq)
    with pytest.raises(RuntimeError, match="block-table entry" if bad == "page" else "outside its tables"):
        oc.check_status()
    oc.check_status()  # cleared
    assert not kc[slot[0], :, slot[1]].any() and not vc[slot[0], :, slot[1]].any()


def test_refusals():
    x = torch.zeros(2, 2, 32, device="cuda", dtype=torch.float16)
    kv = torch.zeros(2, 1, 32, device="cuda", dtype=torch.float16)
    pos = torch.zeros(2, device="cuda", dtype=torch.long)
    cos, sin = oc.rotary_tables(32, 8, device="cuda")
    cache = torch.zeros(4, 1, 16, 32, device="cuda", dtype=torch.float16)
    table = torch.zeros(2, 1, device="cuda", dtype=torch.int32)

    def call(**kw):
        a = dict(q=x, k=kv, v=kv, positions=pos, cos=cos, sin=sin, k_cache=cache, v_cache=cache.clone(), block_tables=table)
        a.update(kw)
        return oc.rotary_append_paged(**a)

    call()
    wide = oc.rotary_tables(64, 8, device="cuda")
    for err, kw in [(ValueError, dict(positions=pos[:1])), (TypeError, dict(positions=pos.float())),
                    (ValueError, dict(cos=wide[0], sin=wide[1])), (ValueError, dict(sin=None)),
                    (TypeError, dict(cos=cos.half(), sin=sin.half())), (TypeError, dict(k=kv.float())),
                    (ValueError, dict(v=kv[:1])), (ValueError, dict(v_cache=cache[:2])),
                    (TypeError, dict(k_cache=cache.float(), v_cache=cache.float())),
                    (ValueError, dict(k_cache=torch.zeros(4, 1, 12, 32, device="cuda", dtype=torch.float16),
                                      v_cache=torch.zeros(4, 1, 12, 32, device="cuda", dtype=torch.float16))),
                    (ValueError, dict(k_scale=0.5)), (ValueError, dict(block_tables=table[:1])),
                    (ValueError, dict(seq_ids=table[:1, 0])), (RuntimeError, dict(q=x.cpu())),
                    (TypeError, dict(q=x.double()))]:
        with pytest.raises(err):
            call(**kw)
    with pytest.raises(RuntimeError, match="no backward pass"):
        call(q=x.clone().requires_grad_())
