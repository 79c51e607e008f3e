"""Serving a Llama-shaped decoder from a paged cache: parallel samples of shared prompts.

:class:`PagedLlama` runs the weights of :class:`~orthocache_gpu_b200.model.GatedLlama` over a
:class:`~orthocache_gpu_b200.pages.PagedKVCache`: prompts of any lengths are packed into one pass
(rotary embedding with the append to the cache, then prompt attention), a prompt's pages are shared by all
of its samples (fork), and each step appends one token per live sequence, copying a shared page only when
it is about to be written (reserve), and attends over the pages.  Ended sequences give their pages back.

Run as a program it decodes a few samples of random prompts with a small random model:

    python -m orthocache_gpu_b200.paged_model
"""

from __future__ import annotations

from typing import Dict, List, Optional, Sequence

import torch
import torch.nn.functional as F

from .exact_attention import paged_decode_attention, prompt_attention
from .model import GatedLlama, LlamaShape, _rms
from .pages import PagedKVCache
from .rotary import rotary_append_paged, rotary_tables


class PagedLlama:
    """A decoder over a paged cache; rows of the cache's tables are the sequences.

    ``softcap``, ``alibi`` (a distance bias instead of rotary positions) and ``window`` apply to prompts
    and steps alike.
    """

    def __init__(self, model: GatedLlama, *, num_pages: int, max_seqs: int, max_tokens: int, block_size: int = 16,
                 softcap: float = 0.0, alibi: bool = False, window: int = 0, scaling: Optional[Dict] = None):
        s = model.s
        self.m, self.softcap, self.window = model, softcap, window
        self.cache = PagedKVCache(s.layers, num_pages, s.kv_heads, s.head_dim, max_seqs=max_seqs, max_tokens=max_tokens,
                                  block_size=block_size, dtype=model.dtype, device=model.dev)
        self.slopes = 2.0 ** (-8.0 * torch.arange(1, s.heads + 1, device=model.dev) / s.heads) if alibi else None
        self.cos, self.sin = (None, None) if alibi else rotary_tables(
            s.head_dim, max_tokens, s.rope_theta, scaling=scaling, device=model.dev)

    def _qkv(self, L, x):
        s = self.m.s
        qkv = F.linear(_rms(x, L["ln1"], s.eps), L["wqkv"]).view(x.shape[0], -1, s.head_dim)
        return qkv[:, :s.heads], qkv[:, s.heads:s.heads + s.kv_heads], qkv[:, s.heads + s.kv_heads:]

    def _rotate(self, i, q, k, v, positions, seq_ids, return_keys=False):
        c = self.cache
        if self.cos is None:  # positions come from the bias: append only
            rotary_append_paged(None, k, v, positions, None, None, c.k[i], c.v[i], c.block_tables, seq_ids=seq_ids)
            return (q, k) if return_keys else q
        return rotary_append_paged(q, k, v, positions, self.cos, self.sin, c.k[i], c.v[i], c.block_tables,
                                   seq_ids=seq_ids, return_keys=return_keys)

    def _finish(self, x):
        return F.linear(_rms(x, self.m.norm, self.m.s.eps), self.m.lm_head)

    @torch.no_grad()
    def prefill(self, prompts: Sequence[torch.Tensor], rows: Sequence[int]) -> torch.Tensor:
        """Prompt i becomes sequence rows[i] (an idle row); returns the logits after each prompt."""
        m, s, c = self.m, self.m.s, self.cache
        rows = [int(r) for r in rows]
        if not rows or len(prompts) != len(rows) or any(p.numel() == 0 for p in prompts):
            raise ValueError("give one row for each prompt, at least one, and no empty prompt")
        if len(set(rows)) != len(rows) or min(rows) < 0 or max(rows) >= c.seq_lens.numel():
            raise ValueError(f"rows ({rows}) must be distinct rows of the cache, of which there are {c.seq_lens.numel()}")
        lens = [p.numel() for p in prompts]
        row = torch.tensor(rows, device=m.dev)
        if bool(c.seq_lens[row].any()):  # its pages may be shared, and would be written to from their first slot on
            raise ValueError(f"rows ({rows}) must be idle; free the sequences that they hold first")
        n = torch.tensor(lens, device=m.dev, dtype=torch.int32)
        tokens = torch.zeros_like(c.seq_lens).index_copy_(0, row, n)
        c.reserve(tokens)
        cu = torch.zeros(len(lens) + 1, dtype=torch.int32, device=m.dev)
        cu[1:] = n.cumsum(0)
        seq_ids = torch.repeat_interleave(row.to(torch.int32), n)
        positions = torch.arange(sum(lens), device=m.dev) - torch.repeat_interleave(cu[:-1], n)
        x = m.embed[torch.cat([p.reshape(-1) for p in prompts]).to(m.dev)]
        for i, L in enumerate(m.layers):
            q, k, v = self._qkv(L, x)
            q, k = self._rotate(i, q, k, v, positions, seq_ids, return_keys=True)
            a = prompt_attention(q, k, v, cu, window=self.window, softcap=self.softcap, alibi_slopes=self.slopes)
            x = m._mlp(L, x + F.linear(a.flatten(1), L["wo"]))
        c.seq_lens += tokens
        return self._finish(x[(cu[1:] - 1).long()])

    @torch.no_grad()
    def step(self, tokens: torch.Tensor, live: torch.Tensor, check: bool = True) -> torch.Tensor:
        """One token for every row: tokens (rows,), live (rows,) int32, 0 for idle rows; returns their logits.

        Raises if there are too few pages.  Without ``check`` the host does not wait, and a step that finds too
        few pages leaves every sequence as it was: the device's status word tells (:func:`check_status`), and
        the logits are of no use.
        """
        m, c = self.m, self.cache
        done = c.reserve(live, check=check)
        if done is not None:
            live = live * done
        # idle rows sit anywhere that exists: one that is full has no next position
        positions = torch.where(live > 0, c.seq_lens, 0)
        c.seq_lens += live
        seq_ids = torch.where(live > 0, torch.arange(live.numel(), device=m.dev, dtype=torch.int32), -1)
        x = m.embed[tokens]
        for i, L in enumerate(m.layers):
            q = self._rotate(i, *self._qkv(L, x), positions, seq_ids)
            a = paged_decode_attention(q, c.k[i], c.v[i], c.block_tables, c.seq_lens, softcap=self.softcap,
                                       alibi_slopes=self.slopes, window=self.window)
            x = m._mlp(L, x + F.linear(a.flatten(1), L["wo"]))
        return self._finish(x)

    @torch.no_grad()
    def sample(self, prompts: Sequence[torch.Tensor], samples: int, steps: int, *, temperature: float = 1.0,
               generator: Optional[torch.Generator] = None) -> List[List[List[int]]]:
        """``samples`` continuations of ``steps`` tokens for each prompt (temperature 0: greedy).

        The prompts' pages are computed and held once.  The samples take the first rows of the cache, which must
        be idle and are so again, and the cache compacted, afterwards; other rows keep their sequences.
        """
        m, c = self.m, self.cache
        rows, n = c.seq_lens.numel(), len(prompts) * samples
        if samples < 1 or steps < 0:
            raise ValueError(f"samples ({samples}) must be positive and steps ({steps}) not negative")
        if n > rows:
            raise ValueError(f"{n} sequences, but the cache has {rows} rows")
        if bool(c.seq_lens[:n].any()):
            raise ValueError(f"the first {n} rows of the cache must be idle; free the sequences that they hold first")

        if n == 0 or steps == 0:
            return [[[] for _ in range(samples)] for _ in prompts]

        def pick(logits):
            if temperature == 0:
                return logits.argmax(-1)
            u = torch.rand(logits.shape, device=m.dev, generator=generator).clamp_(1e-10)
            return (logits.float() / temperature - torch.log(-torch.log(u))).argmax(-1)

        first = [i * samples for i in range(len(prompts))]
        try:
            logits = self.prefill(prompts, first)
            source = torch.arange(rows, dtype=torch.int32)
            source[:n] = torch.arange(n, dtype=torch.int32) // samples * samples
            c.fork(source.to(m.dev))
            live = torch.zeros(rows, dtype=torch.int32, device=m.dev)
            live[:n] = 1
            tokens = torch.zeros(rows, dtype=torch.long, device=m.dev)
            tokens[:n] = pick(logits.repeat_interleave(samples, 0))
            taken = [tokens[:n].clone()]
            for _ in range(steps - 1):
                tokens = pick(self.step(tokens, live))
                taken.append(tokens[:n].clone())
        finally:  # a step may find too few pages: what the samples hold goes back all the same
            c.free(range(n))
            c.compact()
        out = torch.stack(taken, 1).tolist()
        return [out[i * samples:(i + 1) * samples] for i in range(len(prompts))]


def main() -> None:
    model = GatedLlama(LlamaShape(layers=4, hidden=512, heads=8, kv_heads=2, mlp=1024, vocab=1000), max_len=64)
    paged = PagedLlama(model, num_pages=256, max_seqs=16, max_tokens=1024)
    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    prompts = [torch.randint(0, 1000, (n,), generator=g, device="cuda") for n in (37, 200, 5)]
    for i, samples in enumerate(paged.sample(prompts, samples=4, steps=12, generator=g)):
        for tokens in samples:
            print(f"prompt {i} ({prompts[i].numel()} tokens):", *tokens)
    print("free pages:", paged.cache.free_pages(), "of", paged.cache.refcounts.numel())


if __name__ == "__main__":
    main()
