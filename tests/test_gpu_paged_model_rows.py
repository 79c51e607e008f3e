"""Rows of the paged decoder: full, idle, in use, out of pages."""

import pytest
import torch

import orthocache_gpu_b200 as oc

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
    oc.check_status()


def test_a_step_without_pages_changes_no_sequence_when_the_host_does_not_wait():
    """Two samples share the unfilled page of their prompt, and no page is free."""
    p = _paged(num_pages=1, max_seqs=2)
    c = p.cache
    p.prefill(_prompts(5), [0])
    c.fork(_ints(0, 0))
    before = [x.clone() for x in (c.block_tables, c.refcounts, c.seq_lens, *c.caches)]
    p.step(torch.tensor([3, 4], device="cuda"), _ints(1, 1), check=False)
    for x, y in zip((c.block_tables, c.refcounts, c.seq_lens, *c.caches), before):
        assert torch.equal(x, y)
    with pytest.raises(RuntimeError, match="too few free pages"):
        oc.check_status()
    c.fork(_ints(0, -1))  # one holder: it goes on
    logits = p.step(torch.tensor([3, 4], device="cuda"), _ints(1, 0), check=False)
    oc.check_status()
    assert c.seq_lens.tolist() == [6, 0] and logits[0].isfinite().all()


def test_steps_of_a_captured_graph_go_on_until_the_pages_are_full():
    p = _paged(num_pages=4, max_seqs=2)
    eager = _paged(num_pages=4, max_seqs=2)
    for x in (p, eager):
        x.prefill(_prompts(30, 14), [0, 1])  # three pages; the second row needs the fourth at 16 tokens, the first at 32
    tokens, live = torch.tensor([3, 4], device="cuda"), _ints(1, 1)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        got = p.step(tokens, live, check=False)
    for _ in range(2):
        graph.replay()
        assert torch.equal(got, eager.step(tokens, live))
    oc.check_status()
    graph.replay()  # both rows need a page, one is left
    with pytest.raises(RuntimeError, match="too few free pages"):
        oc.check_status()
    assert p.cache.seq_lens.tolist() == [32, 16] and p.cache.free_pages() == 1


def test_reserve_tells_on_the_device_whether_it_was_done():
    c = oc.PagedKVCache(1, 4, 1, 8, max_seqs=2, max_tokens=64, block_size=4)
    assert c.reserve(_ints(4, 4)) is None
    done = c.reserve(_ints(8, 8), check=False)
    assert done.is_cuda and done.dtype == torch.int32 and done.shape == () and int(done) == 1
    oc.check_status()
    assert int(c.reserve(_ints(9, 8), check=False)) == 0
    with pytest.raises(RuntimeError, match="too few free pages"):
        oc.check_status()
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert int(oc.reserve_pages([], none[:, None], none, c.refcounts, none, 4, return_done=True)) == 1


def test_prompts_are_refused_on_rows_that_are_in_use():
    p = _paged()
    c = p.cache
    p.prefill(_prompts(20), [0])
    c.fork(_ints(0, -1, 0))
    before = [x.clone() for x in (c.block_tables, c.refcounts, c.seq_lens, *c.caches)]
    for rows in ([0], [2], [1, 2], [1, 1]):
        with pytest.raises(ValueError, match="distinct" if rows == [1, 1] else "idle"):
            p.prefill(_prompts(*[9] * len(rows)), rows)
    for x, y in zip((c.block_tables, c.refcounts, c.seq_lens, *c.caches), before):
        assert torch.equal(x, y)
    c.free([2])
    p.prefill(_prompts(9, 7), [2, 1])
    assert c.seq_lens.tolist() == [20, 7, 9]


@pytest.mark.parametrize("rows", [[3], [-1], [0, 3], [2 ** 31]])
def test_prompts_are_refused_on_rows_outside_the_cache(rows):
    p = _paged()
    with pytest.raises(ValueError, match="rows of the cache"):
        p.prefill(_prompts(*[9] * len(rows)), rows)
    with pytest.raises(ValueError, match="at least one"):
        p.prefill([], [])
    assert p.cache.free_pages() == 24


def test_samples_that_run_out_of_pages_give_theirs_back():
    p = _paged(num_pages=5)
    with pytest.raises(RuntimeError, match="too few free pages"):
        p.sample(_prompts(30), 3, 12, temperature=0)  # 2 pages shared, 2 copies of the second, then 1 is left for 3
    assert p.cache.free_pages() == 5 and not p.cache.seq_lens.any()
    oc.check_status()
    (got,) = p.sample(_prompts(30), 3, 2, temperature=0)
    assert [len(t) for t in got] == [2, 2, 2]
    p.prefill(_prompts(4), [1])
    with pytest.raises(ValueError, match="idle"):
        p.sample(_prompts(5), 2, 2)
    assert p.cache.seq_lens.tolist() == [0, 4, 0]  # and the sequence that was there stays


def test_samples_leave_the_sequences_of_other_rows_alone():
    p, alone = _paged(max_seqs=4), _paged(max_seqs=4)
    step = torch.zeros(4, dtype=torch.long, device="cuda"), _ints(0, 0, 0, 1)
    for x in (p, alone):
        x.prefill(_prompts(20), [3])
    p.sample(_prompts(30), 3, 4, temperature=0)
    assert p.cache.seq_lens.tolist() == [0, 0, 0, 20] and p.cache.free_pages() == 22
    assert torch.equal(p.step(*step)[3], alone.step(*step)[3])


def test_no_steps_no_prompts_and_counts_that_mean_nothing():
    p = _paged()
    assert p.sample(_prompts(30), 2, 0) == [[[], []]] and p.sample([], 2, 3) == []
    assert [len(t) for t in p.sample(_prompts(30), 2, 1)[0]] == [1, 1]
    for samples, steps in ((0, 3), (-1, 3), (2, -1)):
        with pytest.raises(ValueError, match="must be positive"):
            p.sample(_prompts(30), samples, steps)
    assert p.cache.free_pages() == 24
