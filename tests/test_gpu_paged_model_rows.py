"""Rows of the paged decoder: full, idle, in use, out of pages."""

import pytest
import torch

pytestmark = pytest.mark.gpu

VOCAB = 300


def _paged(num_pages=24, max_seqs=3, max_tokens=48, **kw):
    from orthocache_gpu_b200.model import GatedLlama, LlamaShape
    from orthocache_gpu_b200.paged_model import PagedLlama
    m = GatedLlama(LlamaShape(layers=2, hidden=128, heads=4, kv_heads=2, head_dim=32, mlp=128, vocab=VOCAB), max_len=64, seed=1)
    return PagedLlama(m, num_pages=num_pages, max_seqs=max_seqs, max_tokens=max_tokens, **kw)


def _prompts(*lens):
    g = torch.Generator(device="cuda").manual_seed(5)
    return [torch.randint(0, VOCAB, (n,), generator=g, device="cuda") for n in lens]


def _ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("kw", [{}, dict(alibi=True)])
def test_a_full_idle_row_does_not_stop_the_others(kw):
    p = _paged(**kw)
    p.prefill(_prompts(48, 5), [0, 2])
    tokens = torch.zeros(3, dtype=torch.long, device="cuda")
    for _ in range(3):
        logits = p.step(tokens, _ints(0, 0, 1))
        assert logits[2].isfinite().all()
    assert p.cache.seq_lens.tolist() == [48, 0, 8]
    with pytest.raises(RuntimeError, match="too few free pages"):
        p.step(tokens, _ints(1, 0, 1))  # the full row cannot go on
    assert p.cache.seq_lens.tolist() == [48, 0, 8]
    import orthocache_gpu_b200 as oc
    oc.check_status()
