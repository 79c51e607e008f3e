"""The paged decoder against the dense one, and samples that share their prompt."""

import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPE = dict(layers=2, hidden=256, heads=8, kv_heads=2, head_dim=64, mlp=512, vocab=1000)


def _models(**kw):
    from orthocache_gpu_b200.model import GatedLlama, LlamaShape
    from orthocache_gpu_b200.paged_model import PagedLlama
    m = GatedLlama(LlamaShape(**SHAPE), max_len=512, seed=1)
    return m, PagedLlama(m, num_pages=96, max_seqs=6, max_tokens=512, **kw)


def _prompts(*lens):
    g = torch.Generator(device="cuda").manual_seed(5)
    return [torch.randint(0, SHAPE["vocab"], (n,), generator=g, device="cuda") for n in lens]


def test_prompts_and_steps_match_the_dense_decoder():
    """Two decoders of the same 16-bit weights; logits agree to a few steps of bfloat16."""
    m, p = _models()
    prompts = _prompts(40, 300, 1)
    logits = p.prefill(prompts, [4, 0, 2])
    live = torch.tensor([1, 0, 1, 0, 1, 0], dtype=torch.int32, device="cuda")
    tokens = torch.zeros(6, dtype=torch.long, device="cuda")
    tokens[[4, 0, 2]] = logits.argmax(-1)
    paged = [logits] + [p.step(tokens, live)[[4, 0, 2]] for _ in range(3)]
    for i, prompt in enumerate(prompts):
        m.length = 0
        dense = [m.prefill(prompt)] + [m.step(tokens[[4, 0, 2][i]].reshape(1), None) for _ in range(3)]
        for a, b in zip(paged, dense):
            assert float((a[i].float() - b[0].float()).abs().max()) <= 2e-2 * float(b.abs().max()) + 1e-3
    assert p.cache.seq_lens.tolist() == [303, 0, 4, 0, 43, 0]


@pytest.mark.parametrize("kw", [dict(), dict(softcap=30.0), dict(alibi=True), dict(window=40), dict(block_size=32)])
def test_samples_share_their_prompt_and_greedy_ones_agree(kw):
    m, p = _models(**kw)
    prompts = _prompts(37, 90)
    alone = [p.sample([x], 1, 6, temperature=0)[0][0] for x in prompts]
    together = p.sample(prompts, 3, 6, temperature=0)
    assert p.cache.free_pages() == 96
    for want, got in zip(alone, together):
        assert all(len(t) == 6 for t in got) and got[0] == got[1] == got[2]
        assert got[0][0] == want[0]  # batches round differently; the first token is the prompt's


def test_a_prompts_pages_are_held_once():
    m, p = _models()
    (prompt,) = _prompts(130)
    p.prefill([prompt], [0])
    used = 96 - p.cache.free_pages()
    assert used == -(-130 // 16)
    p.cache.fork(torch.zeros(6, dtype=torch.int32, device="cuda"))
    assert 96 - p.cache.free_pages() == used
    p.step(torch.arange(6, device="cuda"), torch.ones(6, dtype=torch.int32, device="cuda"))
    assert 96 - p.cache.free_pages() == used + 5  # five copies of the unfilled page


def test_too_many_tokens_are_refused_before_anything_is_written():
    m, p = _models()
    with pytest.raises(ValueError, match="rows"):
        p.sample(_prompts(5), 7, 2)
    with pytest.raises(ValueError, match="empty"):
        p.prefill(_prompts(5, 0), [0, 1])
    with pytest.raises(RuntimeError, match="too few free pages"):
        p.prefill(_prompts(600), [0])
    assert p.cache.free_pages() == 96
