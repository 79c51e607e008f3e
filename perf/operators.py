"""The operators of serving from a paged key-value cache: what is measured, and their plain forms.

Four kinds of case, each a step of one serving loop:

* ``rotary``: rotary embedding of a step's queries and keys, and the append of keys and values to the paged cache;
* ``decode``: attention of one new token per sequence over its pages;
* ``prompt``: attention of packed prompts over themselves;
* ``pages``: forking sequences and making the forks writable, or compacting the pages that are in use.

Where ``own`` is false, ``run`` computes a case with elementary torch operations in 32 bits, rounded once at
the end; where it is true, it calls the framework.  ``exact`` is the same from the definitions in 64 bits.
What decides the amount of work (lengths, page tables) comes from the case alone (``layout``), the values
and the order of the pages from the seed.
"""

import math
import random

import torch

own = False

_TYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "fp8": torch.float8_e4m3fn}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "fp8": 1}


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # one token of one sequence at the shape of the repository's own decoder: latency
        dict(name="rotary_step_1", kind="rotary", lens="step", tokens=1, seqs=1, q_heads=32, kv_heads=4, head_dim=64,
             rotary_dim=64, interleaved=False, type="bf16", cache="bf16", block=16, context=4096, layout=1),
        # one token for each of 64 sequences; half of each head is rotated, pairs side by side
        dict(name="rotary_step_64", kind="rotary", lens="step", tokens=64, seqs=64, q_heads=32, kv_heads=8, head_dim=128,
             rotary_dim=64, interleaved=True, type="fp16", cache="fp16", block=16, context=32768, layout=2),
        # five prompts of uneven lengths, 8191 tokens together, written to an 8-bit cache
        dict(name="rotary_prompt_8191", kind="rotary", lens="prompt", tokens=8191, seqs=5, q_heads=32, kv_heads=8,
             head_dim=128, rotary_dim=128, interleaved=False, type="bf16", cache="fp8", block=64, context=8192, layout=3),
        # a short chat turn at the shape of the repository's own decoder: latency
        dict(name="decode_1x300", kind="decode", lens="full", seqs=1, context=300, q_heads=32, kv_heads=4, head_dim=64,
             type="bf16", cache="bf16", block=16, softcap=0.0, alibi=False, window=0, lse=False, layout=4),
        # one long document: the work has to be split over the cache's length
        dict(name="decode_1x32768", kind="decode", lens="full", seqs=1, context=32768, q_heads=32, kv_heads=8,
             head_dim=128, type="bf16", cache="bf16", block=16, softcap=0.0, alibi=False, window=0, lse=True, layout=5),
        # a ragged batch with one key head per query head and capped scores; one slot of the batch is idle
        dict(name="decode_16xragged", kind="decode", lens="ragged", seqs=16, context=8191, q_heads=32, kv_heads=32,
             head_dim=64, type="fp16", cache="fp16", block=32, softcap=30.0, alibi=False, window=0, lse=False, layout=6),
        # a full batch over an 8-bit cache, groups of four, a bias that falls with distance
        dict(name="decode_64x8192_fp8", kind="decode", lens="ragged", seqs=64, context=8192, q_heads=32, kv_heads=8,
             head_dim=128, type="bf16", cache="fp8", block=64, softcap=0.0, alibi=True, window=0, lse=False, layout=7),
        # a short prompt at the shape of the repository's own decoder: latency
        dict(name="prompt_77", kind="prompt", tokens=77, docs=1, q_heads=32, kv_heads=4, head_dim=64, type="bf16",
             causal=True, prefix=False, softcap=0.0, alibi=False, window=0, layout=8),
        # packed prompts of uneven lengths, capped scores, a sliding window
        dict(name="prompt_4099_packed", kind="prompt", tokens=4099, docs=7, q_heads=16, kv_heads=4, head_dim=128,
             type="fp16", causal=True, prefix=False, softcap=50.0, alibi=False, window=1024, layout=9),
        # one long prompt
        dict(name="prompt_8192", kind="prompt", tokens=8192, docs=1, q_heads=32, kv_heads=8, head_dim=128, type="bf16",
             causal=True, prefix=False, softcap=0.0, alibi=False, window=0, layout=10),
        # a beam step: 32 of 64 sequences are replaced by forks of others and made writable, over 22 layers
        dict(name="pages_fork_64", kind="pages", op="fork", seqs=64, context=900, kv_heads=4, head_dim=64, tensors=44,
             type="bf16", block=16, pages=4096, layout=11),
        # compaction after half of the sequences have ended
        dict(name="pages_compact_4096", kind="pages", op="compact", seqs=64, context=900, kv_heads=4, head_dim=64,
             tensors=44, type="bf16", block=16, pages=4096, layout=12),
    ]


def _log_int(rng, low, high):
    """A whole number, spread over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


_HEADS = [(32, 4), (32, 8), (32, 32), (16, 16), (8, 1), (12, 4), (14, 2), (16, 4)]


def draw(rng):
    kind = rng.choice(["rotary", "decode", "prompt", "pages"])
    layout = rng.randrange(1 << 30)
    q_heads, kv_heads = rng.choice(_HEADS)
    block = rng.choice([8, 16, 32, 64, 128])
    if kind == "rotary":
        head_dim, rotary_dim = rng.choice([(64, 64), (64, 32), (128, 128), (128, 64), (80, 32), (96, 96), (256, 128)])
        dtype, cache = rng.choice([("bf16", "bf16"), ("fp16", "fp16"), ("bf16", "fp8"), ("fp16", "fp8"), ("fp32", "fp32")])
        case = dict(q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, rotary_dim=rotary_dim,
                    interleaved=rng.random() < 0.5, type=dtype, cache=cache, block=block)
        if rng.random() < 0.5:
            n = _log_int(rng, 1, 256)
            case.update(lens="step", tokens=n, seqs=n, context=_log_int(rng, 64, 32768))
        else:
            n = _log_int(rng, 64, 7168 * 48 * 128 // ((q_heads + 2 * kv_heads) * max(head_dim, 128)) // (2 if dtype == "fp32" else 1))
            case.update(lens="prompt", tokens=n, seqs=min(n, rng.randint(1, 8)), context=n)
    elif kind == "decode":
        head_dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
        dtype = rng.choice(["bf16", "fp16"])
        cache = rng.choice([dtype, dtype, "fp8"])
        # tokens of cache in all: at most what the largest listed cases hold, in keys and values
        most = 64 * 8192 * 8 * 64 // (kv_heads * head_dim) // _BYTES[cache]
        seqs = _log_int(rng, 1, 128)
        context = _log_int(rng, 1, min(32768, most // seqs))
        case = dict(lens=rng.choice(["full", "ragged"]), seqs=seqs, context=context, q_heads=q_heads, kv_heads=kv_heads,
                    head_dim=head_dim, type=dtype, cache=cache, block=block, softcap=rng.choice([0.0, 0.0, 30.0, 50.0]),
                    alibi=rng.random() < 0.3, window=rng.choice([0, 0, 0, _log_int(rng, 16, 4096)]),
                    lse=rng.random() < 0.5)
    elif kind == "prompt":
        tokens = _log_int(rng, 1, 8192 * 32 // max(32, q_heads))
        causal = rng.random() < 0.8
        case = dict(tokens=tokens, docs=min(tokens, rng.randint(1, 12)) if causal or tokens <= 4096 else rng.randint(3, 12),
                    q_heads=q_heads, kv_heads=kv_heads, head_dim=rng.choice([64, 64, 80, 96, 128, 128]),
                    type=rng.choice(["bf16", "fp16"]), causal=causal, prefix=causal and rng.random() < 0.3,
                    softcap=rng.choice([0.0, 0.0, 30.0, 50.0]), alibi=rng.random() < 0.3,
                    window=rng.choice([0, 0, 0, _log_int(rng, 16, 4096)]))
    else:
        seqs = _log_int(rng, 2, 64)
        context = _log_int(rng, 16, 1500)
        case = dict(op=rng.choice(["fork", "compact"]), seqs=seqs, context=context, kv_heads=rng.choice([1, 2, 4]),
                    head_dim=64, tensors=2 * rng.randint(1, 22), type=rng.choice(["bf16", "fp16", "fp8"]), block=block)
        case["pages"] = max(8 * seqs, min(4096, 2 * seqs * (context // block + 3)))
    return dict(case, kind=kind, layout=layout)


# --------------------------------------------------------------------------- what the case decides
def _lengths(case):
    """Tokens of each sequence (decode), or of each prompt (rotary and prompt cases)."""
    rng = random.Random(case["layout"])
    if case["kind"] == "decode":
        n, top = case["seqs"], case["context"]
        if case["lens"] == "full":
            return [top] * n
        lens = [rng.randint(max(1, top // 8), top) for _ in range(n)]
        lens[rng.randrange(n)] = top
        if n >= 4:
            lens[rng.randrange(n)] = 0  # a slot of the batch without a sequence
        return lens
    if case["kind"] == "rotary" and case["lens"] == "step":
        return [rng.randint(1, case["context"]) for _ in range(case["seqs"])]
    n, total = case.get("docs") or case["seqs"], case["tokens"]
    cuts = sorted(rng.sample(range(1, total), n - 1)) if n > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def _prefixes(case):
    rng = random.Random(case["layout"] + 1)
    return [rng.randint(0, n) if case["prefix"] else 0 for n in _lengths(case)]


def _holdings(case):
    """Pages cases: (lengths, table of page ids or -1, references to each page, source of each sequence, wanted lengths)."""
    rng = random.Random(case["layout"])
    n, top, bs, pages = case["seqs"], case["context"], case["block"], case["pages"]
    top = max(1, min(top, (pages // n - 3) * bs))
    lens = [rng.randint(max(1, top // 2), top) for _ in range(n)]
    cols = max(-(-x // bs) for x in lens) + 2
    order = list(range(pages))
    rng.shuffle(order)
    table, take = [], iter(order)
    ended = [case["op"] == "compact" and rng.random() < 0.5 for _ in range(n)]
    if case["op"] == "compact":
        ended[0], ended[-1] = False, True
    for i, x in enumerate(lens):
        held = [next(take) for _ in range(-(-x // bs))]
        if i % 4 == 3 and case["op"] == "compact":  # shares its first half with the sequence before it
            k = min(len(held), sum(p >= 0 for p in table[-1])) // 2
            held = table[-1][:k] + held[k:]
        table.append(held + [-1] * (cols - len(held)))
    for i in range(n):
        if ended[i]:
            table[i], lens[i] = [-1] * cols, 0
    refs = [0] * pages
    for row in table:
        for p in row:
            if p >= 0:
                refs[p] += 1
    source = [rng.randrange(n) if rng.random() < 0.5 else i for i in range(n)]
    wanted = [lens[s] + rng.randint(1, bs) for s in source]
    return lens, table, refs, source, wanted


def _visible_pairs(case):
    """Query-key pairs that the mask of a prompt case leaves."""
    total = 0
    for n, pre in zip(_lengths(case), _prefixes(case)):
        w = case["window"] or n
        for_row = n if not case["causal"] else None
        if for_row is None and pre == 0:
            m = min(w, n)
            total += m * (m + 1) // 2 + (n - m) * m
        else:
            for i in range(n):
                low, high = max(0, i - w + 1), (n if not case["causal"] else i + 1)
                total += high - low + (max(0, pre - high) + min(low, pre) if pre else 0)
    return total


def work(case):
    if case["kind"] == "rotary":
        t, size, kept = case["tokens"], _BYTES[case["type"]], _BYTES[case["cache"]]
        rows, kv = case["q_heads"], case["kv_heads"]
        nbytes = t * case["head_dim"] * (2 * rows * size + 2 * kv * (size + kept)) + t * (case["rotary_dim"] * 4 + 16)
        return {"bytes": nbytes, "flops": 3 * t * (rows + kv) * case["rotary_dim"]}
    if case["kind"] == "decode":
        lens = [min(n, case["window"] or n) for n in _lengths(case)]
        keys = sum(lens)
        per_key = 2 * case["kv_heads"] * case["head_dim"] * _BYTES[case["cache"]]
        rows = case["seqs"] * case["q_heads"] * case["head_dim"] * 2 * _BYTES[case["type"]]
        tables = 4 * sum(-(-n // case["block"]) for n in lens)
        return {"bytes": keys * per_key + rows + tables, "flops": 4 * keys * case["q_heads"] * case["head_dim"]}
    if case["kind"] == "prompt":
        size = _BYTES[case["type"]]
        nbytes = case["tokens"] * case["head_dim"] * size * 2 * (case["q_heads"] + case["kv_heads"])
        return {"bytes": nbytes, "flops": 4 * _visible_pairs(case) * case["q_heads"] * case["head_dim"]}
    lens, table, refs, source, wanted = _holdings(case)
    entries, page = len(table) * len(table[0]), case["kv_heads"] * case["block"] * case["head_dim"] * _BYTES[case["type"]]
    moved = len(_copies(case, lens, table, refs, source, wanted))
    return {"bytes": 2 * 4 * (entries + case["pages"]) + 2 * moved * page * case["tensors"], "flops": entries}


def _copies(case, lens, table, refs, source, wanted):
    """The pages that a pages case has to copy (one entry each)."""
    if case["op"] == "compact":
        live = sum(r > 0 for r in refs)
        return [p for p, r in enumerate(refs) if r > 0 and p >= live]
    last = {}
    for s in source:  # every sequence is wanted longer: those that share an unfilled page copy it, but for one
        if lens[s] % case["block"]:
            last.setdefault(table[s][lens[s] // case["block"]], []).append(s)
    return [p for p, rows in last.items() for _ in rows[1:]]


# --------------------------------------------------------------------------- inputs
def _tables(theta, factor, rotary_dim, positions, device):
    inverse = theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim) / factor
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * inverse
    return angle.cos().float(), angle.sin().float()


def _page_tables(counts, block, device, g):
    """A table (sequences, most pages) of shuffled page ids, -1 where a sequence has none, and the pages in all."""
    total = max(1, sum(counts))
    order = torch.randperm(total, generator=g, device=device).to(torch.int32)
    width = max(1, max(counts))
    n = torch.tensor(counts, device=device)
    held = torch.arange(width, device=device)[None] < n[:, None]
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device=device)
    table[held] = order[: int(sum(counts))]
    return table, total


def _cache(shape, cache, g, dev):
    """A cache as a running server has it: every slot holds something; 8-bit values with a scale."""
    x = torch.randn(shape, generator=g, device=dev, dtype=torch.float16 if cache == "fp8" else _TYPE[cache])
    return (x * 32).to(_TYPE["fp8"]) if cache == "fp8" else x


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float32).to(_TYPE[case["type"]])

    s = {"case": dict(case)}
    kind = case["kind"]
    if kind == "rotary":
        lens = _lengths(case)
        t, hq, hk, d = case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"]
        # queries, keys and values are parts of one projection's output
        qkv = randn(t, hq + 2 * hk, d)
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        if case["lens"] == "step":
            s["positions"] = torch.tensor([n - 1 for n in lens], device=dev)
            s["seq_ids"] = torch.arange(t, device=dev, dtype=torch.int32)
        else:
            n = torch.tensor(lens, device=dev)
            s["seq_ids"] = torch.repeat_interleave(torch.arange(len(lens), device=dev, dtype=torch.int32), n)
            s["positions"] = torch.arange(t, device=dev) - torch.repeat_interleave(n.cumsum(0) - n, n)
        s["cos"], s["sin"] = _tables(10000.0, 4.0 if case["context"] > 8192 else 1.0, case["rotary_dim"],
                                     max(lens), dev)
        bs = case["block"]
        if case["lens"] == "step":  # only the page that a step writes to is in hand: one page per sequence, at its column
            table = torch.full((len(lens), max(-(-n // bs) for n in lens)), 0, dtype=torch.int32, device=dev)
            order = torch.randperm(len(lens), generator=g, device=dev).to(torch.int32)
            table[torch.arange(len(lens), device=dev), s["positions"] // bs] = order
            s["table"], pages = table, len(lens)
        else:
            s["table"], pages = _page_tables([-(-n // bs) for n in lens], bs, dev, g)
        s["k_cache"] = _cache((pages, hk, bs, d), case["cache"], g, dev)
        s["v_cache"] = _cache((pages, hk, bs, d), case["cache"], g, dev)
        s["k_scale"], s["v_scale"] = (0.03125, 0.03125) if case["cache"] == "fp8" else (1.0, 1.0)
    elif kind == "decode":
        lens, bs = _lengths(case), case["block"]
        s["table"], pages = _page_tables([-(-n // bs) for n in lens], bs, dev, g)
        shape = (pages, case["kv_heads"], bs, case["head_dim"])
        s["k_cache"], s["v_cache"] = _cache(shape, case["cache"], g, dev), _cache(shape, case["cache"], g, dev)
        s["k_scale"], s["v_scale"] = (0.03125, 0.03125) if case["cache"] == "fp8" else (1.0, 1.0)
        s["q"] = randn(case["seqs"], case["q_heads"], case["head_dim"]) * 2
        s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        s["slopes"] = _slopes(case["q_heads"], dev) if case["alibi"] else None
        s["scale"] = case["head_dim"] ** -0.5
    elif kind == "prompt":
        t, hq, hk, d = case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"]
        s["q"], s["k"], s["v"] = randn(t, hq, d) * 2, randn(t, hk, d), randn(t, hk, d)
        cu = [0]
        for n in _lengths(case):
            cu.append(cu[-1] + n)
        s["cu_seqlens"] = torch.tensor(cu, dtype=torch.int32, device=dev)
        s["prefix_lens"] = torch.tensor(_prefixes(case), dtype=torch.int32, device=dev) if case["prefix"] else None
        s["slopes"] = _slopes(hq, dev) if case["alibi"] else None
        s["scale"] = d ** -0.5
    else:
        lens, table, refs, source, wanted = _holdings(case)
        pages = case["pages"]
        live = sum(r > 0 for r in refs)
        # the seed orders the pages, below and above the number in use on their own, so that as many move
        order = torch.cat([torch.randperm(live, generator=g, device=dev),
                           live + torch.randperm(pages - live, generator=g, device=dev)])
        table = torch.tensor(table, device=dev)
        s["table"] = torch.where(table >= 0, order[table.clamp(min=0)], -1).to(torch.int32)
        s["refs"] = torch.zeros(pages, dtype=torch.int32, device=dev)
        s["refs"][order] = torch.tensor(refs, dtype=torch.int32, device=dev)
        s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        s["source"] = torch.tensor(source, dtype=torch.int32, device=dev)
        s["wanted"] = torch.tensor(wanted, dtype=torch.int32, device=dev)
        s["all"] = _cache((case["tensors"], pages, case["kv_heads"], case["block"], case["head_dim"]), case["type"], g, dev)
        s["caches"] = list(s["all"].unbind(0))  # one tensor for the keys, one for the values, of each layer
    return s


def _slopes(heads, dev):
    return 2.0 ** (-8.0 * torch.arange(1, heads + 1, device=dev, dtype=torch.float32) / heads)


# --------------------------------------------------------------------------- one pass
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"rotary": _own_rotary, "decode": _own_decode, "prompt": _own_prompt, "pages": _own_pages}[kind](state)
    return {"rotary": _rotary, "decode": _decode, "prompt": _prompt, "pages": _pages}[kind](state)


def _own_rotary(s):
    from orthocache_gpu_b200 import rotary_append_paged
    q = rotary_append_paged(s["q"], s["k"], s["v"], s["positions"], s["cos"], s["sin"], s["k_cache"], s["v_cache"],
                            s["table"], seq_ids=s["seq_ids"], interleaved=s["case"]["interleaved"],
                            k_scale=s["k_scale"], v_scale=s["v_scale"])
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_decode(s):
    from orthocache_gpu_b200 import paged_decode_attention
    c = s["case"]
    return paged_decode_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["seq_lens"], scale=s["scale"],
                                  softcap=c["softcap"], alibi_slopes=s["slopes"], window=c["window"],
                                  k_scale=s["k_scale"], v_scale=s["v_scale"], return_lse=c["lse"])


def _own_prompt(s):
    from orthocache_gpu_b200 import prompt_attention
    c = s["case"]
    return prompt_attention(s["q"], s["k"], s["v"], s["cu_seqlens"], causal=c["causal"], prefix_lens=s["prefix_lens"],
                            window=c["window"], scale=s["scale"], softcap=c["softcap"], alibi_slopes=s["slopes"])


def _own_pages(s):
    from orthocache_gpu_b200 import compact_pages, fork_sequences, reserve_pages
    bs = s["case"]["block"]
    if s["case"]["op"] == "compact":
        table, refs = compact_pages(s["caches"], s["table"], s["refs"])
        return {"table": table, "refs": refs, "caches": s["all"]}
    table, lens, refs = fork_sequences(s["table"], s["seq_lens"], s["refs"], s["source"], bs)
    reserve_pages(s["caches"], table, lens, refs, s["wanted"], bs)
    return {"table": table, "seq_lens": lens, "refs": refs, "caches": s["all"]}


def _turn(x, cos, sin, rotary_dim, interleaved):
    """Rotary embedding of the first rotary_dim columns of x (tokens, heads, head_dim)."""
    x = x.float()
    part, rest = x[..., :rotary_dim], x[..., rotary_dim:]
    cos, sin = cos[:, None], sin[:, None]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = part.chunk(2, -1)
        part = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([part, rest], -1)


def _rotary(s):
    c = s["case"]
    cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
    q = _turn(s["q"], cos, sin, c["rotary_dim"], c["interleaved"])
    k = _turn(s["k"], cos, sin, c["rotary_dim"], c["interleaved"])
    page = s["table"][s["seq_ids"].long(), s["positions"] // c["block"]].long()
    at = s["positions"] % c["block"]
    _put(s["k_cache"], page, at, k / s["k_scale"], c["cache"])
    _put(s["v_cache"], page, at, s["v"].float() / s["v_scale"], c["cache"])
    return {"q": q.to(s["q"].dtype), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _put(cache, page, at, x, kind):
    if kind == "fp8":
        cache.view(torch.uint8)[page, :, at] = x.clamp(-448.0, 448.0).to(cache.dtype).view(torch.uint8)
    else:
        cache[page, :, at] = x.to(cache.dtype)


def _pages_of(cache, table, kind):
    """(sequences, kv heads, tokens, head_dim) in 32 bits."""
    x = cache.view(torch.uint8) if kind == "fp8" else cache
    x = x[table.clamp(min=0).long()]
    x = x.view(cache.dtype) if kind == "fp8" else x
    return x.transpose(1, 2).flatten(2, 3).float()


def _decode(s):
    c = s["case"]
    n, hk, d = c["seqs"], c["kv_heads"], c["head_dim"]
    k = _pages_of(s["k_cache"], s["table"], c["cache"])
    q = s["q"].float().view(n, hk, -1, d)
    scores = (q @ k.transpose(-1, -2)) * (s["scale"] * s["k_scale"])
    if c["softcap"]:
        scores = c["softcap"] * torch.tanh(scores / c["softcap"])
    at = torch.arange(k.shape[2], device=k.device)
    last = s["seq_lens"].view(n, 1, 1, 1).long() - 1
    if s["slopes"] is not None:
        scores = scores + s["slopes"].view(1, hk, -1, 1) * (at - last)
    seen = at <= last
    if c["window"]:
        seen = seen & (at > last - c["window"])
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    out = (p @ _pages_of(s["v_cache"], s["table"], c["cache"])) * s["v_scale"] / total.clamp(min=1e-30)
    out = out.view(n, -1, d).to(s["q"].dtype)
    return (out, (top + torch.log(total)).view(n, -1)) if c["lse"] else out


def _prompt_mask(s, t, dev):
    """(tokens, tokens) of which key a query sees, and the distance from key to query."""
    c, cu = s["case"], s["cu_seqlens"].long()
    at = torch.arange(t, device=dev)
    doc = torch.bucketize(at, cu[1:], right=True)
    away = at[None] - at[:, None]
    seen = away <= 0 if c["causal"] else torch.ones_like(away, dtype=torch.bool)
    if c["window"]:
        seen = seen & (away > -c["window"])
    if s["prefix_lens"] is not None:
        seen = seen | ((at - cu[doc]) < s["prefix_lens"][doc])[None]
    return seen & (doc[None] == doc[:, None]), away


def _prompt(s):
    c = s["case"]
    t, hk, d = c["tokens"], c["kv_heads"], c["head_dim"]
    q = s["q"].float().view(t, hk, -1, d).permute(1, 2, 0, 3)
    k, v = s["k"].float().transpose(0, 1)[:, None], s["v"].float().transpose(0, 1)[:, None]
    scores = (q @ k.transpose(-1, -2)) * s["scale"]
    if c["softcap"]:
        scores = c["softcap"] * torch.tanh(scores / c["softcap"])
    seen, away = _prompt_mask(s, t, q.device)
    if s["slopes"] is not None:
        scores = scores - s["slopes"].view(hk, -1, 1, 1) * away.abs()
    scores = scores.masked_fill(~seen, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = (p @ v) / p.sum(-1, keepdim=True)
    return out.permute(2, 0, 1, 3).reshape(t, -1, d).to(s["q"].dtype)


def _pages(s):
    c, table, refs = s["case"], s["table"], s["refs"]
    pages, bs = c["pages"], c["block"]
    every = s["all"].view(torch.uint8) if c["type"] == "fp8" else s["all"]
    ids = torch.arange(pages, device=refs.device)
    if c["op"] == "compact":
        live = refs > 0
        n = live.sum()
        holes, movers = ids[~live & (ids < n)], ids[live & (ids >= n)]
        to = ids.clone()
        to[movers] = holes
        every[:, holes] = every[:, movers]
        new_refs = torch.zeros_like(refs)
        new_refs[to[live]] = refs[live]
        return {"table": torch.where(table >= 0, to[table.clamp(min=0).long()], -1).to(torch.int32), "refs": new_refs,
                "caches": s["all"]}
    rows, cols = torch.arange(c["seqs"], device=refs.device), torch.arange(table.shape[1], device=refs.device)
    src = s["source"].long()
    lens = s["seq_lens"][src]
    stays = (src == rows)[:, None]
    forked = torch.where(cols < ((lens + bs - 1) // bs)[:, None], table[src], -1)
    new = torch.where(stays, table, forked)
    gone, come = table[~stays & (table >= 0)].long(), new[~stays & (new >= 0)].long()
    refs = refs + torch.bincount(come, minlength=pages) - torch.bincount(gone, minlength=pages)
    # the unfilled page that the next token goes to: one of its holders keeps it, the others copy it
    column = (lens // bs).long()
    last = new.gather(1, column.clamp(max=new.shape[1] - 1)[:, None])[:, 0]
    writes = (s["wanted"] > lens) & (lens % bs != 0)
    at = torch.where(writes, last, 0).long()
    writers = torch.zeros_like(refs).index_add_(0, at, writes.to(refs.dtype))
    final = torch.full_like(refs, -1).scatter_reduce(0, at, torch.where(writes, rows, -1).to(refs.dtype), "amax")
    copies = writes & (refs[at] > 1) & ~((writers[at] == refs[at]) & (final[at] == rows))
    held = (new >= 0).sum(1)
    need = (cols >= held[:, None]) & (cols < ((s["wanted"] + bs - 1) // bs)[:, None])
    need |= copies[:, None] & (cols == column[:, None])
    free = ids[refs == 0]
    got = free[(need.flatten().cumsum(0) - 1).clamp(min=0).view(need.shape)]
    every[:, got[copies, column[copies]]] = every[:, last[copies].long()]
    refs = refs - torch.bincount(last[copies].long(), minlength=pages)
    new = torch.where(need, got, new).to(torch.int32)
    refs[got[need]] = 1
    return {"table": new, "seq_lens": lens, "refs": refs.to(torch.int32), "caches": s["all"]}


# --------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "decode": _exact_decode, "prompt": _exact_prompt, "pages": _exact_pages}[case["kind"]](s, case)


def _exact_rotary(s, c):
    r = c["rotary_dim"]
    pairs = torch.arange(r // 2, device=s["q"].device)
    first, second = (2 * pairs, 2 * pairs + 1) if c["interleaved"] else (pairs, pairs + r // 2)
    z = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"]][:, None]  # e^(i angle) of each pair
    done = {}
    for name in ("q", "k"):
        x = s[name].double().clone()
        turned = torch.complex(x[..., first], x[..., second]) * z
        x[..., first], x[..., second] = turned.real, turned.imag
        done[name] = x
    answer = {"q": done["q"]}
    for name, x in (("k_cache", done["k"] / s["k_scale"]), ("v_cache", s["v"].double() / s["v_scale"])):
        cache = s[name].double()
        place = s["positions"] % c["block"]
        page = s["table"][s["seq_ids"].long(), s["positions"] // c["block"]].long()
        for h in range(c["kv_heads"]):
            cache[page, h, place] = x[:, h].clamp(-448, 448) if c["cache"] == "fp8" else x[:, h]
        answer[name] = cache
    return answer


def _exact_decode(s, c):
    d, group = c["head_dim"], c["q_heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    lse = torch.full(out.shape[:2], -math.inf, dtype=torch.float64, device=out.device)
    for i, n in enumerate(_lengths(c)):
        if n == 0:
            continue
        first = max(0, n - c["window"]) if c["window"] else 0
        ids = s["table"][i, : -(-n // c["block"])].long()
        byte = (lambda t: t.view(torch.uint8)[ids].view(t.dtype)) if c["cache"] == "fp8" else (lambda t: t[ids])
        k, v = (byte(s[w]).double().transpose(0, 1).reshape(c["kv_heads"], -1, d)[:, first:n] * s[z]
                for w, z in (("k_cache", "k_scale"), ("v_cache", "v_scale")))
        x = torch.einsum("hgd,hnd->hgn", s["q"][i].double().view(c["kv_heads"], group, d), k) * s["scale"]
        if c["softcap"]:
            x = torch.tanh(x / c["softcap"]) * c["softcap"]
        if c["alibi"]:
            x = x + s["slopes"].double().view(c["kv_heads"], group, 1) * torch.arange(first - n + 1, 1, device=x.device)
        out[i] = torch.einsum("hgn,hnd->hgd", torch.softmax(x, -1), v).reshape(-1, d)
        lse[i] = torch.logsumexp(x, -1).flatten()
    return (out, lse) if c["lse"] else out


def _exact_prompt(s, c):
    group = c["q_heads"] // c["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    start = 0
    for n, pre in zip(_lengths(c), _prefixes(c)):
        i, j = torch.arange(n, device=out.device)[:, None], torch.arange(n, device=out.device)[None]
        hidden = (j > i) if c["causal"] else torch.zeros_like(j > i)
        if c["window"]:
            hidden = hidden | (i - j >= c["window"])
        hidden = hidden & (j >= pre)
        rows = slice(start, start + n)
        for h in range(c["q_heads"]):
            x = s["q"][rows, h].double() @ s["k"][rows, h // group].double().T * s["scale"]
            if c["softcap"]:
                x = torch.tanh(x / c["softcap"]) * c["softcap"]
            if c["alibi"]:
                x = x - s["slopes"][h].double() * (i - j).abs()
            out[rows, h] = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ s["v"][rows, h // group].double()
        start += n
    return out


def _exact_pages(s, c):
    """Tables and references by plain bookkeeping; pages are moved, not computed."""
    table, refs, lens = s["table"].tolist(), s["refs"].tolist(), s["seq_lens"].tolist()
    bs, dev = c["block"], s["refs"].device

    def whole(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    if c["op"] == "compact":
        live = sum(r > 0 for r in refs)
        holes = iter(p for p in range(live) if refs[p] == 0)
        to = {p: (p if p < live else next(holes)) for p, r in enumerate(refs) if r > 0}
        after = [0] * len(refs)
        for p, where in to.items():
            after[where] = refs[p]
        return {"table": whole([[to.get(p, -1) for p in row] for row in table]), "refs": whole(after), "caches": None}
    old = [list(row) for row in table]
    new_lens = []
    for i, src in enumerate(s["source"].tolist()):
        new_lens.append(lens[src])
        if src != i:
            table[i] = [p if k < -(-lens[src] // bs) else -1 for k, p in enumerate(old[src])]
    refs = [0] * len(refs)
    for row in table:
        for p in row:
            if p >= 0:
                refs[p] += 1
    free = iter([p for p, r in enumerate(refs) if r == 0])
    for i, n in enumerate(s["wanted"].tolist()):
        for k in range(-(-n // bs)):
            p = table[i][k]
            shared = k == new_lens[i] // bs and new_lens[i] % bs and n > new_lens[i] and p >= 0 and refs[p] > 1
            if p < 0 or shared:
                if shared:
                    refs[p] -= 1
                table[i][k] = next(free)
                refs[table[i][k]] = 1
    return {"table": whole(table), "seq_lens": whole(new_lens), "refs": whole(refs), "caches": None}
