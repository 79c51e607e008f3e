"""Plain 64-bit implementations of the paged-serving operators, and the tolerances they are held to.

Attention weighs values with P rounded to the products' 16-bit type and its sum kept in float32, and rounds
the result once: |out - exact| <= u_p A + u_out |exact| + e A with A = sum_j p_j |v_j|, u the unit roundoff
of either type (2^-8 bfloat16, 2^-11 float16: a significand of 8 and 11 bits; 0 float32) and e for the
float32 arithmetic: 5e-5 for the exponentials, caps, biases and sums, and, since an error of a score is a
relative error of its weight, 2^-19 |scale| sum_k |q_k k_k|, the products' sums with up to 16 roundings (or
truncations, of 2^-23) one after the other.  The queries of 8-bit caches go through float16 times a power of
two, which is exact down to 2^-24 of the largest.
"""

import torch

ROUNDOFF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 0.0}
ARITHMETIC = 5e-5


def attend(q, k, v, visible, bias, scale, softcap):
    """q (n, d), k / v (m, d), visible / bias (n, m), in 64 bits: (out, A, lse, noise of the scores (n,)).

    Rows that see nothing: 0, -inf.
    Keys that a row does not see do not take part at all.
    """
    out = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    lse = torch.full((q.shape[0],), -float("inf"), dtype=torch.float64, device=q.device)
    noise = torch.zeros(q.shape[0], dtype=torch.float64, device=q.device)
    finite = bool(torch.isfinite(k).all() and torch.isfinite(v).all() and torch.isfinite(q).all())
    if finite:  # all rows at once
        s = q @ k.T * scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        s = (s + bias).masked_fill(~visible, -float("inf"))
        some = visible.any(1)
        if k.shape[0]:
            noise = 2.0 ** -19 * abs(scale) * (q.abs() @ k.abs().T).masked_fill(~visible, 0).amax(1)
        p = torch.softmax(s[some], -1)
        out[some], size[some], lse[some] = p @ v, p @ v.abs(), torch.logsumexp(s[some], -1)
        return out, size, lse, noise
    for i in range(q.shape[0]):
        at = visible[i].nonzero()[:, 0]
        if at.numel():
            s = (k[at] @ q[i]) * scale
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            s = s + bias[i, at]
            p = torch.softmax(s, -1)
            noise[i] = 2.0 ** -19 * abs(scale) * (k[at].abs() @ q[i].abs()).nan_to_num(0, 0, 0).amax()
            out[i], size[i], lse[i] = p @ v[at], p @ v[at].abs(), torch.logsumexp(s, -1)
    return out, size, lse, noise


def assert_attention(got, exact, size, noise, product_dtype, what=""):
    if got.numel() == 0:
        return
    tol = (ROUNDOFF[product_dtype] + ARITHMETIC + noise[:, None]) * size + ROUNDOFF[got.dtype] * exact.abs() + 1e-9
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25  # the spacing of its smallest numbers
    same = torch.isnan(got.double()) == torch.isnan(exact)
    assert bool(same.all()), f"{what}: NaN in other places"
    over = ((got.double() - exact).abs() - tol).nan_to_num(0.0)
    assert float(over.max()) <= 0, f"{what}: off by {float(over.max()):.3g} more than the bound"


def assert_lse(got, exact, noise, what=""):
    assert torch.equal(torch.isinf(got), torch.isinf(exact.float())), what
    ok = torch.isfinite(exact)
    err = (got.double()[ok] - exact[ok]).abs()
    assert err.numel() == 0 or float((err - 2e-5 - 1e-6 * exact[ok].abs() - noise[ok]).max()) <= 0, f"{what}: {float(err.max()):.3g}"


def pages_for(lens, block, device, spare=3, seed=0):
    """A shuffled block table for sequences of these lengths (-1 where there is no page) and the number of pages."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // block) for n in lens]
    total = sum(counts) + spare
    order = torch.randperm(total, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(1, max(counts))), -1, dtype=torch.int32)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c]
        at += c
    return table.to(device), total
