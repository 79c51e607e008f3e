"""Page bookkeeping against plain Python, exactly, and the contents that sequences see."""

import random

import pytest
import torch

import orthocache_gpu_b200 as oc

pytestmark = pytest.mark.gpu


class Model:
    """The state in plain lists; every operation as its description says."""

    def __init__(self, pages, rows, cols, block):
        self.block, self.table = block, [[-1] * cols for _ in range(rows)]
        self.lens, self.refs = [0] * rows, [0] * pages

    def fork(self, source):
        old, lens = [list(r) for r in self.table], list(self.lens)
        for i, s in enumerate(source):
            self.lens[i] = lens[s] if s >= 0 else 0
            if s != i:
                self.table[i] = [p if s >= 0 and k * self.block < lens[s] else -1 for k, p in enumerate(old[s if s >= 0 else i])]
        self.refs = [0] * len(self.refs)
        for row in self.table:
            for p in row:
                if p >= 0:
                    self.refs[p] += 1

    def reserve(self, wanted):
        """False, and nothing changed, if pages or columns do not suffice."""
        cols, bs = len(self.table[0]), self.block
        if any(-(-w // bs) > cols for w in wanted):
            return False
        writers = {}
        for i, w in enumerate(wanted):
            n = self.lens[i]
            if w > n and n % bs:
                writers.setdefault(self.table[i][n // bs], []).append(i)
        free = iter([p for p, r in enumerate(self.refs) if r == 0])
        table, refs = [list(r) for r in self.table], list(self.refs)
        for i, w in enumerate(wanted):
            for k in range(cols):
                p, part = table[i][k], k == self.lens[i] // bs and self.lens[i] % bs
                copy = False
                if part and w > self.lens[i] and self.refs[p] > 1:
                    copy = not (len(writers[p]) == self.refs[p] and writers[p][-1] == i)
                if copy or (p < 0 and k * bs < w):
                    new = next(free, None)
                    if new is None:
                        return False
                    if copy:
                        refs[p] -= 1
                    table[i][k] = new
                    refs[new] = 1
        self.table, self.refs = table, refs
        return True

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        holes = iter([p for p in range(live) if self.refs[p] == 0])
        to = {p: p if p < live else next(holes) for p, r in enumerate(self.refs) if r > 0}
        refs = [0] * len(self.refs)
        for p, q in to.items():
            refs[q] = self.refs[p]
        self.refs, self.table = refs, [[to[p] if p >= 0 else -1 for p in row] for row in self.table]

    def same(self, c):
        assert c.block_tables.tolist() == self.table
        assert c.refcounts.tolist() == self.refs
        assert c.seq_lens.tolist() == self.lens


@pytest.mark.parametrize("block, rows, pages, tokens, heads, D, dtype", [
    (16, 6, 64, 200, 2, 64, torch.bfloat16), (8, 40, 300, 100, 1, 32, torch.float16), (1, 5, 80, 20, 1, 16, torch.float32),
    (4, 7, 40, 30, 3, 5, torch.float16), (64, 3, 5000, 100000, 1, 8, torch.float8_e4m3fn), (2, 1100, 4500, 8, 1, 8, torch.float16)])
def test_random_operations(block, rows, pages, tokens, heads, D, dtype):
    """Every table and count as the model has them, and every sequence sees the tokens that it was given."""
    rng = random.Random(block * 100 + rows)
    c = oc.PagedKVCache(2, pages, heads, D, max_seqs=rows, max_tokens=tokens, block_size=block, dtype=dtype)
    m = Model(pages, rows, c.block_tables.shape[1], block)
    text = [[] for _ in range(rows)]  # the tokens of each sequence
    stamp = 0

    def show():
        m.same(c)
        flat = [(x.view(torch.uint8) if dtype == torch.float8_e4m3fn else x)[:, 0, :, 0].tolist() for x in c.caches]
        for i, t in enumerate(text):
            for plane, x in enumerate(flat):
                got = [x[m.table[i][j // block]][j % block] for j in range(len(t))]
                assert got == [(s + plane) % 100 for s in t]

    for _ in range(14 if rows < 1000 else 4):
        grow = [rng.choice([0, 0, 1, 1, 3, block, 2 * block + 1]) for _ in range(rows)]
        wanted = [min(len(t) + g, len(m.table[0]) * block) for t, g in zip(text, grow)]
        if m.reserve(wanted):
            c.reserve(torch.tensor([w - len(t) for w, t in zip(wanted, text)], dtype=torch.int32, device="cuda"))
            seq, pos, val = [], [], []
            for i, w in enumerate(wanted):
                for j in range(len(text[i]), w):
                    stamp += 1
                    seq.append(i), pos.append(j), val.append(stamp % 100)
                    text[i].append(stamp % 100)
            m.lens = [len(t) for t in text]
            c.seq_lens.copy_(torch.tensor(m.lens, dtype=torch.int32))
            if seq:  # write by the tables, as an append does
                s, p = torch.tensor(seq, device="cuda"), torch.tensor(pos, device="cuda")
                page = c.block_tables[s, p // block].long()
                for plane, x in enumerate(c.caches):
                    v = torch.tensor([(a + plane) % 100 for a in val], device="cuda")
                    (x.view(torch.uint8) if dtype == torch.float8_e4m3fn else x)[page, :, p % block] = \
                        v[:, None, None].to(torch.uint8 if dtype == torch.float8_e4m3fn else dtype)
        else:
            with pytest.raises(RuntimeError, match="too few free pages"):
                c.reserve(torch.tensor([w - len(t) for w, t in zip(wanted, text)], dtype=torch.int32, device="cuda"))
        show()
        source = [rng.choice([i, i, i, -1, rng.randrange(rows)]) for i in range(rows)]
        m.fork(source)
        c.fork(torch.tensor(source, device="cuda"))
        text = [list(text[s]) if s >= 0 else [] for s in source]
        show()
        if rng.random() < 0.5:
            m.compact()
            c.compact()
            show()
    c.free(range(rows))
    assert c.free_pages() == pages and not c.seq_lens.any()


def test_copies_wait_until_a_write_and_the_last_writer_keeps_the_page():
    c = oc.PagedKVCache(1, 8, 1, 8, max_seqs=3, max_tokens=64, block_size=4)
    one = torch.tensor([6, 0, 0], dtype=torch.int32, device="cuda")
    c.reserve(one)
    c.seq_lens += one
    first = c.block_tables[0, :2].tolist()
    assert first == [0, 1]
    c.fork(torch.tensor([0, 0, 0], device="cuda"))
    assert c.block_tables[:, :2].tolist() == [first] * 3 and c.refcounts[:2].tolist() == [3, 3]
    c.reserve(torch.tensor([0, 1, 0], dtype=torch.int32, device="cuda"))  # one writer: it copies
    assert c.block_tables[:, 1].tolist() == [1, 2, 1] and c.refcounts[:3].tolist() == [3, 2, 1]
    c.reserve(torch.tensor([1, 0, 1], dtype=torch.int32, device="cuda"))  # both holders write: the first copies
    assert c.block_tables[:, 1].tolist() == [3, 2, 1] and c.refcounts[:4].tolist() == [3, 1, 1, 1]


@pytest.mark.parametrize("shape, dtype", [((9, 2, 16, 64), torch.bfloat16), ((9, 3, 5), torch.float16), ((9, 7), torch.uint8),
                                          ((9, 4, 100, 50), torch.float32), ((9, 1, 1, 8), torch.float8_e4m3fn)])
def test_copy_pages(shape, dtype):
    g = torch.Generator(device="cuda").manual_seed(1)
    caches = [torch.randint(0, 255, (shape[0], int(torch.tensor(shape[1:]).prod()) * torch.empty(0, dtype=dtype).element_size()),
                            generator=g, device="cuda", dtype=torch.uint8).view(dtype).view(shape) for _ in range(130)]
    want = [x.clone() for x in caches]
    src, dst = torch.tensor([0, -1, 8, 3], device="cuda"), torch.tensor([1, 5, 2, -1], device="cuda")
    oc.copy_pages(caches, src, dst)
    oc.check_status()
    for x, w in zip(caches, want):
        x, w = x.view(torch.uint8).flatten(1), w.view(torch.uint8).flatten(1)
        w[1], w[2] = w[0].clone(), w[8].clone()
        assert torch.equal(x, w)


def test_copy_pages_of_a_strided_cache_and_of_odd_addresses():
    both = torch.randn(6, 2, 4, 32, device="cuda")  # keys and values of a page side by side
    want = both.clone()
    want[4, 0] = want[1, 0]
    oc.copy_pages([both[:, 0]], torch.tensor([1], device="cuda"), torch.tensor([4], device="cuda"))
    assert torch.equal(both, want)
    odd = torch.arange(6 * 8 + 1, device="cuda", dtype=torch.uint8)[1:].view(6, 8)
    want = odd.clone()
    want[0] = want[5]
    oc.copy_pages([odd], torch.tensor([5], device="cuda"), torch.tensor([0], device="cuda"))
    assert torch.equal(odd, want)
    oc.copy_pages([odd], torch.tensor([6], device="cuda"), torch.tensor([0], device="cuda"))
    with pytest.raises(RuntimeError, match="block-table entry"):
        oc.check_status()
    assert torch.equal(odd, want)


def test_sources_and_pages_outside_are_reported():
    table = torch.tensor([[0, 1], [2, 9]], dtype=torch.int32, device="cuda")
    lens, refs = torch.tensor([30, 30], dtype=torch.int32, device="cuda"), torch.ones(4, dtype=torch.int32, device="cuda")
    new = oc.fork_sequences(table, lens, refs, torch.tensor([5, 1], device="cuda"), 16)
    with pytest.raises(RuntimeError, match="outside its tables"):
        oc.check_status()
    assert new[0].tolist() == table.tolist() and new[2].tolist() == [1, 1, 1, 1]
    oc.fork_sequences(table, lens, refs, torch.tensor([0, -1], device="cuda"), 16)
    with pytest.raises(RuntimeError, match="block-table entry"):
        oc.check_status()
    oc.compact_pages([], table, refs)
    with pytest.raises(RuntimeError, match="block-table entry"):
        oc.check_status()


def test_refusals():
    table, lens = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    refs, cache = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, 1, 16, 8, device="cuda")
    for err, call in [(TypeError, lambda: oc.fork_sequences(table.long(), lens, refs, lens, 16)),
                      (ValueError, lambda: oc.fork_sequences(table, lens[:1], refs, lens, 16)),
                      (ValueError, lambda: oc.fork_sequences(table, lens, refs, lens[:1], 16)),
                      (ValueError, lambda: oc.fork_sequences(table, lens, refs, lens, 0)),
                      (ValueError, lambda: oc.fork_sequences(table.t().contiguous().t(), lens, refs, lens, 16)),
                      (ValueError, lambda: oc.reserve_pages([cache[:2]], table, lens, refs, lens, 16)),
                      (ValueError, lambda: oc.reserve_pages([cache, cache[:, :, :8]], table, lens, refs, lens, 16)),
                      (TypeError, lambda: oc.reserve_pages([cache, 3], table, lens, refs, lens, 16)),
                      (TypeError, lambda: oc.reserve_pages(cache, table, lens, refs, lens, 16)),
                      (RuntimeError, lambda: oc.reserve_pages([cache.cpu()], table, lens, refs, lens, 16)),
                      (ValueError, lambda: oc.compact_pages([cache[:3]], table, refs)),
                      (ValueError, lambda: oc.copy_pages([cache.transpose(1, 2)[:, :, :, ::2]], lens, lens)),
                      (ValueError, lambda: oc.copy_pages([cache], lens, lens[:1]))]:
        with pytest.raises(err):
            call()
    big = torch.zeros(5000, 1, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="code 5"):
        oc.reserve_pages([], big, big[:, 0].contiguous(), refs, big[:, 0].contiguous(), 16)
