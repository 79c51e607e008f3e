"""The serving operators have no backward pass: whatever carries a derivative is refused, and what they write to is marked."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

import orthocache_gpu_b200 as oc

pytestmark = pytest.mark.gpu


def _inputs():
    f = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    return dict(q=f(2, 4, 32), k=f(2, 2, 32), v=f(2, 2, 32), cos=f(8, 16), sin=f(8, 16), k_cache=f(4, 2, 16, 32),
                v_cache=f(4, 2, 16, 32), slopes=f(4))


def _calls():
    pos = torch.zeros(2, dtype=torch.long, device="cuda")
    table = torch.tensor([[0], [1]], dtype=torch.int32, device="cuda")
    lens, refs = torch.ones(2, dtype=torch.int32, device="cuda"), torch.tensor([1, 1, 0, 0], dtype=torch.int32, device="cuda")
    pair = torch.tensor([0], device="cuda"), torch.tensor([3], device="cuda")
    return {
        "embedding": (("q", "cos", "sin"), lambda x: oc.rotary_embedding(x["q"], pos, x["cos"], x["sin"])),
        "append": (("q", "k", "v", "cos", "sin", "k_cache", "v_cache"),
                   lambda x: oc.rotary_append_paged(x["q"], x["k"], x["v"], pos, x["cos"], x["sin"], x["k_cache"], x["v_cache"], table)),
        "decode": (("q", "k_cache", "v_cache", "slopes"),
                   lambda x: oc.paged_decode_attention(x["q"], x["k_cache"], x["v_cache"], table, lens, alibi_slopes=x["slopes"])),
        "prompt": (("q", "k", "v", "slopes"), lambda x: oc.prompt_attention(x["q"], x["k"], x["v"], alibi_slopes=x["slopes"])),
        "reserve": (("k_cache", "v_cache"), lambda x: oc.reserve_pages([x["k_cache"], x["v_cache"]], table, lens, refs, lens, 16)),
        "compact": (("k_cache", "v_cache"), lambda x: oc.compact_pages([x["k_cache"], x["v_cache"]], table, refs)),
        "copy": (("k_cache", "v_cache"), lambda x: oc.copy_pages([x["k_cache"], x["v_cache"]], *pair)),
    }


@pytest.mark.parametrize("name", ["embedding", "append", "decode", "prompt", "reserve", "compact", "copy"])
def test_inputs_that_carry_a_derivative_are_refused(name):
    used, call = _calls()[name]
    for key in used:
        x = _inputs()
        x[key].requires_grad_()
        with pytest.raises(RuntimeError, match="no backward pass"):
            call(x)
        with torch.no_grad():
            call(x)
        with torch.inference_mode():
            call(x)
        with fwd.dual_level():
            x = _inputs()
            x[key] = fwd.make_dual(x[key], torch.ones_like(x[key]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(x)
    with fwd.dual_level():
        call(_inputs())
    oc.check_status()


def test_tensors_that_are_written_to_get_a_new_version():
    """As torch's in-place operations do it, so that a backward pass that saved the old contents fails."""
    x = _inputs()
    calls = _calls()
    saved = (x["k_cache"] * torch.ones((), device="cuda", requires_grad=True)).sum()  # saves k_cache
    for name in ("append", "reserve", "compact", "copy"):
        before = [x[c]._version for c in ("k_cache", "v_cache")]
        calls[name][1](x)
        assert [x[c]._version for c in ("k_cache", "v_cache")] == [v + 1 for v in before], name
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.backward()
    table, refs = torch.full((2, 2), -1, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    lens, before = torch.zeros(2, dtype=torch.int32, device="cuda"), (table._version, refs._version)
    oc.reserve_pages([], table, lens, refs, lens + 1, 16)
    assert (table._version, refs._version) == (before[0] + 1, before[1] + 1)
    with torch.inference_mode():  # such tensors have no version
        y = _inputs()
    calls["append"][1](y)
    calls["copy"][1](y)
    oc.check_status()
