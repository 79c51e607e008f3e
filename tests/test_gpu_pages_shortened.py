"""Sequences that are shortened while others hold their pages (rejected draft tokens), and then grow again."""

import random

import pytest
import torch

import orthocache_gpu_b200 as oc

pytestmark = pytest.mark.gpu


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _cache(rows=3, pages=24, block=16, layers=1):
    return oc.PagedKVCache(layers, pages, 1, 8, max_seqs=rows, max_tokens=8 * block, block_size=block, dtype=torch.float16)


@pytest.mark.parametrize("cut, table, refs", [
    (20, [0, 3, 4], [2, 1, 1, 1, 1]),  # page 1 is copied (4 tokens of it stay), page 2 replaced
    (16, [0, 3, 4], [2, 1, 1, 1, 1]),  # both replaced
    (15, [3, 4, 5], [1, 1, 1, 1, 1, 1]),  # and the first one copied
    (0, [3, 4, 5], [1, 1, 1, 1, 1, 1]),
    (33, [0, 1, 3], [2, 2, 1, 1]),  # the last page alone
    (40, [0, 1, 2], [2, 2, 2])])  # not growing: nothing is written to
def test_pages_behind_the_tokens_that_others_hold_are_replaced(cut, table, refs):
    c = _cache()
    c.reserve(_ints([40, 0, 0]))
    c.seq_lens.copy_(_ints([40, 0, 0]))
    for x in c.caches:
        x[:3] = torch.arange(1, 4, device="cuda", dtype=torch.float16)[:, None, None, None]
    c.fork(_ints([0, 0, -1]))
    c.seq_lens[1] = cut
    c.reserve(_ints([0, 40 - cut, 0]))
    assert c.block_tables[0, :3].tolist() == [0, 1, 2] and c.block_tables[1, :3].tolist() == table
    assert c.refcounts.tolist() == refs + [0] * (24 - len(refs))
    for x in c.caches:
        assert x[:3, 0, 0, 0].tolist() == [1, 2, 3]
        if cut % 16 and cut < 40:  # the tokens that stay came along
            assert x[table[cut // 16], 0, 0, 0] == cut // 16 + 1


def test_the_last_holder_keeps_a_page_that_all_of_them_write_to_and_replaced_pages_become_free():
    c = _cache()
    c.reserve(_ints([40, 0, 0]))
    c.seq_lens.copy_(_ints([40, 0, 0]))
    c.fork(_ints([0, 0, -1]))
    c.seq_lens.copy_(_ints([20, 16, 0]))
    c.reserve(_ints([20, 24, 0]))
    # page 1: row 0 copies it, row 1 keeps it; page 2: both replace it
    assert c.block_tables[:2, :3].tolist() == [[0, 3, 4], [0, 1, 5]]
    assert c.refcounts.tolist() == [2, 1, 0, 1, 1, 1] + [0] * 18


def test_too_few_pages_change_nothing():
    c = _cache(pages=4)
    c.reserve(_ints([40, 0, 0]))
    c.seq_lens.copy_(_ints([40, 0, 0]))
    c.fork(_ints([0, 0, -1]))
    c.seq_lens[1] = 16
    before = c.block_tables.clone(), c.refcounts.clone()
    with pytest.raises(RuntimeError, match="too few free pages"):
        c.reserve(_ints([0, 24, 0]))
    assert torch.equal(c.block_tables, before[0]) and torch.equal(c.refcounts, before[1])


@pytest.mark.parametrize("block, rows, pages", [(4, 5, 200), (1, 9, 400), (16, 40, 900), (8, 1500, 30000)])
def test_what_sequences_see_through_forks_cuts_and_growth(block, rows, pages):
    """Every sequence sees the tokens that it was given, whoever else held their pages."""
    rng = random.Random(rows)
    c = _cache(rows, pages, block, layers=2)
    text, stamp = [[] for _ in range(rows)], 0
    for _ in range(12 if rows < 1000 else 4):
        wanted = [min(len(t) + rng.choice([0, 1, 1, 2, block, 3 * block]), 8 * block) for t in text]
        c.reserve(_ints([w - len(t) for w, t in zip(wanted, text)]))
        seq, pos, val = [], [], []
        for i, w in enumerate(wanted):
            for j in range(len(text[i]), w):
                stamp += 1
                seq.append(i), pos.append(j), val.append(stamp % 1000)
                text[i].append(stamp % 1000)
        s, p = torch.tensor(seq, device="cuda"), torch.tensor(pos, device="cuda")
        for plane, x in enumerate(c.caches):
            x[c.block_tables[s, p // block].long(), :, p % block] = (torch.tensor(val, device="cuda") + plane)[:, None, None].half()
        c.seq_lens.copy_(_ints([len(t) for t in text]))
        source = [rng.choice([i, i, -1, rng.randrange(rows), rng.randrange(rows)]) for i in range(rows)]
        c.fork(_ints(source))
        text = [list(text[k]) if k >= 0 else [] for k in source]
        text = [t[:rng.randint(0, len(t))] if rng.random() < 0.5 else t for t in text]
        c.seq_lens.copy_(_ints([len(t) for t in text]))
        table = c.block_tables.tolist()
        counts = [0] * pages
        for row in table:
            for q in row:
                if q >= 0:
                    counts[q] += 1
        assert c.refcounts.tolist() == counts
        for plane, x in enumerate(c.caches):
            flat = x[:, 0, :, 0].tolist()
            for i, t in enumerate(text):
                assert [flat[table[i][j // block]][j % block] for j in range(len(t))] == [v + plane for v in t]
    c.free(range(rows))
    assert c.free_pages() == pages
