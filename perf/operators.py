"""The operators that many continuations of one prompt are made of, as cases that can be timed and compared.

A case is one call of one operator, as a step of such a batch makes it:

* ``attention``  the new tokens of a batch whose sequences share the pages of a long prefix, in groups (one prompt continued many
  times; several system prompts with their requests); a group may share nothing;
* ``tables``     page tables, positions and slots of a step, built on the device from the sequences' lengths;
* ``history``    which tokens occurred in a sequence and how often each was generated, from its prompt and its output;
* ``steer``      penalties, biases and masks of allowed tokens on a step's logits.

Where ``own`` is false an operator is computed in its plain form: elementary torch operations in 32 bits.  Head layouts and
vocabularies are those of the benchmark's models (``perf/cases.py``: 2k, 8b, 14b, 32b), besides generic ones.  Which lengths a case has
follows from the case alone; the seed makes the numbers.
"""
import math
import random
import types

import torch

own = False

DEVICE = "cuda:0"
PAGE = 64
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def _attention(batch, groups, prefix, low, high, tokens, heads, kv, dim, dtype, name=None):
    """prefix: positions of the longest shared prefix (one group: of the only one); low, high: a sequence's own cached positions lie
    between them; tokens: the most new tokens of a sequence."""
    c = dict(kind="attention", batch=batch, groups=groups, prefix=prefix, low=low, high=high, tokens=tokens, heads=heads, kv=kv, dim=dim,
             dtype=dtype)
    return dict(c, name=name) if name else c


def _tables(batch, context, tokens, forks, name=None):
    """context: the most cached positions of a sequence; tokens: the most new ones (1: one each); forks: sequences that start from the
    pages of the first one."""
    c = dict(kind="tables", batch=batch, context=context, tokens=tokens, forks=forks)
    return dict(c, name=name) if name else c


def _history(rows, vocab, prompt, output, name=None):
    """prompt, output: the most tokens of a row's prompt, and of those generated."""
    c = dict(kind="history", rows=rows, vocab=vocab, prompt=prompt, output=output)
    return dict(c, name=name) if name else c


def _steer(rows, vocab, history, bias, masks, allowed, name=None):
    """history: the most distinct tokens that occurred in a row; bias: biased tokens a row; masks: different masks of allowed tokens
    (0: no masks), every second row or so has one; allowed: the share of the vocabulary that a mask leaves."""
    c = dict(kind="steer", rows=rows, vocab=vocab, history=history, bias=bias, masks=masks, allowed=allowed)
    return dict(c, name=name) if name else c


def listed():
    return [
        # Four samples of a short prompt on a small model: all latency.
        _attention(4, 1, 512, 5, 60, 1, 16, 4, 128, "bfloat16", "shared_2k_b4"),
        # A full batch of answers to one long document.
        _attention(64, 1, 8192, 16, 700, 1, 32, 8, 128, "bfloat16", "shared_8b_b64"),
        # Seven system prompts with their requests, some of them alone with their own; no power of two anywhere.
        _attention(45, 7, 4100, 1, 900, 1, 40, 8, 128, "bfloat16", "shared_14b_groups"),
        # Very long shared context, eight query heads to a key head.
        _attention(24, 1, 31000, 30, 1500, 1, 64, 8, 128, "bfloat16", "shared_32b_long"),
        # Short questions of a few tokens each behind a system prompt, heads of 64.
        _attention(16, 2, 1500, 0, 90, 24, 24, 4, 64, "bfloat16", "shared_questions"),
        # The 32-bit path.
        _attention(6, 1, 1000, 3, 200, 1, 16, 4, 128, "float32", "shared_2k_f32"),
        # A decode step's description: one token each.
        _tables(48, 4000, 1, 0, "tables_decode"),
        # Prompts and single tokens together, forks of a long document among them.
        _tables(700, 30000, 400, 300, "tables_mixed"),
        # Three conversations on a small model, and the sequences of a full batch.
        _history(3, 32768, 7000, 400, "history_2k_b3"),
        _history(64, 151936, 2000, 300, "history_8b_b64"),
        # Penalties and biases, no masks.
        _steer(8, 151936, 700, 40, 0, 1.0, "steer_8b_b8"),
        # A full batch, half of it held to a grammar; a vocabulary that is no multiple of 4.
        _steer(61, 100003, 1500, 0, 12, 0.03, "steer_masks"),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm (from 1 on)."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(max(low, 1)), math.log(high)))))))


def _drawn(rng):
    kind = rng.choice(["attention"] * 6 + ["tables", "tables", "history", "steer", "steer"])
    if kind == "attention":
        heads, kv, dim = rng.choice([(16, 4, 128), (32, 8, 128), (40, 8, 128), (64, 8, 128), (24, 4, 64), (8, 8, 64), (32, 2, 128)])
        dtype = rng.choice(["bfloat16"] * 5 + ["float32"])
        tokens = rng.choice([1, 1, 1, _spread(rng, 2, 30)])
        batch = _spread(rng, 2, 24 if dtype == "float32" or tokens > 1 else 96)
        low = rng.choice([0, _spread(rng, 1, 100 if tokens > 1 else 300)])
        return _attention(batch, rng.choice([1, 1, rng.randint(1, min(9, batch))]), _spread(rng, 64, 4000 if dtype == "float32" else 24000), low,
                          low + _spread(rng, 1, 200 if tokens > 1 else 1500), tokens, heads, kv, dim, dtype)
    if kind == "tables":
        batch = _spread(rng, 1, 1000)
        return _tables(batch, _spread(rng, 64, 30000), rng.choice([1, _spread(rng, 2, 500)]), rng.choice([0, rng.randint(0, batch - 1)]))
    vocab = rng.choice([32768, 151936, 100003, _spread(rng, 1000, 200000)])
    if kind == "history":
        return _history(_spread(rng, 1, 64), vocab, _spread(rng, 1, 8000), _spread(rng, 1, 1000))
    masks = rng.choice([0, _spread(rng, 1, 32)])
    return _steer(_spread(rng, 1, 64), vocab, _spread(rng, 1, min(vocab // 4, 4000)), rng.choice([0, _spread(rng, 1, 300)]), masks,
                  round(rng.choice([0.001, 0.05, 0.9]), 3) if masks else 1.0)


def draw(rng):
    most = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    while True:
        c = _drawn(rng)
        w = work(c)
        # (a product in 32 bits off the tensor cores costs about ten of the others')
        if w["bytes"] <= most["bytes"] and w["flops"] * (10 if c.get("dtype") == "float32" else 1) <= most["flops"]:
            return c


# ---- sizes -----------------------------------------------------------------
def _rng(c):
    return random.Random(",".join("%s=%s" % (k, c[k]) for k in sorted(c) if k != "name"))


def _groups(c):
    """Sequences and shared pages of each group; cached and new tokens of each sequence."""
    rng, G = _rng(c), c["groups"]
    cuts = [0] + sorted(rng.sample(range(1, c["batch"]), G - 1)) + [c["batch"]]
    sizes = [b - a for a, b in zip(cuts, cuts[1:])]
    longest = max(1, c["prefix"] // PAGE)
    # (of several groups the first has the longest prefix, the last none)
    pages = [longest if g == 0 else 0 if g == G - 1 else _spread(rng, 1, longest) for g in range(G)]
    group_of = [g for g in range(G) for _ in range(sizes[g])]
    starts = [pages[g] * PAGE + rng.randint(c["low"], c["high"]) for g in group_of]
    return sizes, pages, group_of, starts, [rng.randint(1, c["tokens"]) for _ in group_of]


def _lengths(c):
    """Cached and new tokens of each sequence, and which start from the first one's pages."""
    rng, n = _rng(c), c["batch"]
    fork = [0 < b <= c["forks"] for b in range(n)]
    top = c["context"]
    starts = [top if b == 0 else (top // PAGE) * PAGE if fork[b] else rng.randint(0, top) for b in range(n)]
    return starts, [rng.randint(0 if c["tokens"] > 1 and b > 0 else 1, c["tokens"]) for b in range(n)], fork


def _cu(q):
    return [sum(q[:i]) for i in range(len(q) + 1)]


def _pages(n):
    return -(-n // PAGE)


def _row_lengths(c):
    rng = _rng(c)
    return [rng.randint((c["prompt"] + 1) // 2, c["prompt"]) for _ in range(c["rows"])], [rng.randint(0, c["output"]) for _ in range(c["rows"])]


def _mask_of(c):
    rng = _rng(c)
    return [rng.randrange(c["masks"]) if c["masks"] and rng.random() < 0.6 else -1 for _ in range(c["rows"])]


def work(case):
    if case["kind"] == "attention":
        sizes, pages, group_of, starts, q = _groups(case)
        width = 2 if case["dtype"] == "bfloat16" else 4
        shared = PAGE * sum(pages)
        mine = sum(s + n - PAGE * pages[g] for s, n, g in zip(starts, q, group_of))
        rows = sum(q) * case["heads"] * case["dim"]
        seen = sum(n * s + n * (n + 1) // 2 for s, n in zip(starts, q))
        return {"bytes": 2 * (shared + mine) * case["kv"] * case["dim"] * width + 2 * rows * width, "flops": 4 * case["dim"] * case["heads"] * seen}
    if case["kind"] == "tables":
        starts, q, fork = _lengths(case)
        held = sum(_pages(s) for s in starts)
        new = sum(_pages(s + n) - _pages(s) for s, n in zip(starts, q))
        table = case["batch"] * max(_pages(s + n) for s, n in zip(starts, q))
        forked = sum(_pages(s) for s, f in zip(starts, fork) if f)
        return {"bytes": 4 * (6 * case["batch"] + held + 2 * new + forked + table) + 16 * sum(q), "flops": 4 * (table + sum(q))}
    if case["kind"] == "history":
        prompt, output = _row_lengths(case)
        return {"bytes": 8 * (sum(prompt) + sum(output)) + 8 * sum(output) + case["rows"] * case["vocab"] // 4, "flops": 2 * (sum(prompt) + sum(output))}
    n, mask_of = case["rows"] * case["vocab"], _mask_of(case)
    out = sum(m >= 0 for m in mask_of) * case["vocab"] * (1.0 - case["allowed"])
    words = case["rows"] * case["vocab"] / 8 + case["masks"] * case["vocab"] / 8
    return {"bytes": int(8 * n - 4 * out + words + case["rows"] * (4 * case["history"] + 8 * case["bias"])), "flops": 4 * n}


# ---- inputs ----------------------------------------------------------------
def _ints(v):
    return torch.tensor(v, dtype=torch.int32).to(DEVICE)


def _words(bits):
    """[rows, n] truth values as 32-bit words, place i in bit i % 32 of word i // 32."""
    rows, n = bits.shape
    w = torch.zeros((rows, -(-n // 32) * 32), dtype=torch.int64, device=bits.device)
    w[:, :n] = bits
    w = (w.view(rows, -1, 32) << torch.arange(32, device=bits.device)).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def _bits(words, n):
    v = torch.arange(n, device=words.device)
    return (words[:, v >> 5] >> (v & 31)) & 1


def _prepare_attention(c, g):
    dt = DTYPES[c["dtype"]]
    sizes, pages, group_of, starts, q = _groups(c)
    n, kv_len = sum(q), [s + t for s, t in zip(starts, q)]
    own_pages = [_pages(k) - pages[g_] for k, g_ in zip(kv_len, group_of)]
    total = 1 + sum(pages) + sum(own_pages)
    ids = (torch.randperm(total - 1, generator=g, device=DEVICE) + 1).to(torch.int32)
    first, mine = _cu(pages), [sum(pages) + x for x in _cu(own_pages)]
    width = max(_pages(k) for k in kv_len)
    # (column j of sequence b: a page of its group's prefix, then its own, then the reserved page 0)
    at = torch.tensor([[first[a] + j if j < pages[a] else mine[b] + j - pages[a] if j < pages[a] + own_pages[b] else -1 for j in range(width)]
                       for b, a in enumerate(group_of)]).to(DEVICE)
    table = torch.where(at >= 0, ids[at.clamp(min=0)], 0).to(torch.int32)
    kv = torch.randn((total, 2, c["kv"], PAGE, c["dim"]), generator=g, device=DEVICE).to(dt)
    query = torch.randn((n, c["heads"], c["dim"]), generator=g, device=DEVICE)
    # (as in trained models some heads look sharply, some all around)
    query = (query * torch.linspace(0.5, 2.5, c["heads"], device=DEVICE)[:, None]).to(dt)
    seq = [b for b in range(len(q)) for _ in range(q[b])]
    batch = types.SimpleNamespace(
        n_seqs=len(q), n_tokens=n, table_width=width, q_lens=q, starts=starts, max_q_len=max(q), max_kv_len=max(kv_len), kv_bound=max(kv_len),
        cu_seqlens=_ints(_cu(q)), start=_ints(starts), kv_len=_ints(kv_len), page_table=table, seq_of_token=_ints(seq),
        positions=_ints([starts[b] + i for b in range(len(q)) for i in range(q[b])]))
    return dict(c=c, q=query, kv=kv, batch=batch, cu_groups=_ints(_cu(sizes)), pages=_ints(pages), group_of=_ints(group_of), max_pages=max(pages),
                own_bound=max(k - PAGE * pages[a] for k, a in zip(kv_len, group_of)), scale=1.0 / math.sqrt(c["dim"]),
                most=max(sum(q[b] for b in range(len(q)) if group_of[b] == a) for a in range(len(pages))))


def _prepare_tables(c, g):
    starts, q, fork = _lengths(c)
    n, width = c["batch"], max(_pages(s + t) for s, t in zip(starts, q))
    slots = torch.randperm(n, generator=g, device=DEVICE).to(torch.int32) + 1
    held = _ints([0 if f else _pages(s) for s, f in zip(starts, fork)])
    new = sum(_pages(s + t) - _pages(s) for s, t in zip(starts, q))
    total = int(sum(0 if f else _pages(s) for s, f in zip(starts, fork)))
    ids = torch.randperm(total + new + 7, generator=g, device=DEVICE).to(torch.int32) + 1
    j = torch.arange(width, device=DEVICE)
    at = (held.cumsum(0) - held)[:, None] + j
    tables = torch.zeros((n + 1, width), dtype=torch.int32, device=DEVICE)
    tables[slots.long()] = torch.where(j < held[:, None], ids[at.clamp(max=ids.numel() - 1)], 0).to(torch.int32)
    make = lambda *s, t=torch.int32: torch.zeros(s, dtype=t, device=DEVICE)      # noqa: E731
    free = torch.cat([make(5), ids[total:]])
    return dict(c=c, start=_ints(starts), q_len=_ints(q), slots=slots, tables=tables, free_pages=free, free_head=_ints([5]),
                parent=torch.where(_ints(fork) > 0, slots[0], -1).to(torch.int32), n=sum(q), width=width,
                out=dict(page_table=make(n, width), cu_seqlens=make(n + 1), kv_len=make(n), positions=make(sum(q)), seq_of_token=make(sum(q)),
                         slot_map=make(sum(q), t=torch.int64), head_out=make(1)))


def _tokens(g, n, vocab):
    """Ids as texts have them: few that come often, many that are rare."""
    u = torch.rand(n, generator=g, device=DEVICE)
    return (vocab ** u - 1).to(torch.int32).clamp(0, vocab - 1)


def _prepare_history(c, g):
    prompt, output = _row_lengths(c)
    rows = torch.arange(c["rows"], dtype=torch.int32, device=DEVICE)
    return dict(c=c, rows=rows, prompt=_tokens(g, sum(prompt), c["vocab"]), output=_tokens(g, sum(output), c["vocab"]),
                prompt_row=rows.repeat_interleave(_ints(prompt)), output_row=rows.repeat_interleave(_ints(output)),
                seen=torch.zeros((c["rows"], _pages32(c["vocab"])), dtype=torch.int32, device=DEVICE),
                counts=torch.zeros((c["rows"], c["vocab"]), dtype=torch.int32, device=DEVICE))


def _pages32(n):
    return -(-n // 32)


def _prepare_steer(c, g):
    R, V, rng = c["rows"], c["vocab"], _rng(c)
    tok = torch.stack([_tokens(g, c["history"], V) for _ in range(R)]).long()
    seen = torch.zeros((R, V), dtype=torch.int64, device=DEVICE).scatter_(1, tok, 1)
    # (half of what occurred was generated, some of it often)
    counts = torch.zeros((R, V), dtype=torch.int32, device=DEVICE)
    counts.scatter_add_(1, tok[:, ::2], torch.randint(1, 9, tok[:, ::2].shape, generator=g, device=DEVICE, dtype=torch.int32))
    n_bias = [rng.randint(c["bias"] // 2, c["bias"]) if c["bias"] else 0 for _ in range(R)]
    biased = [torch.randperm(V, generator=g, device=DEVICE)[:k].to(torch.int32) for k in n_bias]
    pick = lambda values: torch.tensor([rng.choice(values) for _ in range(R)], device=DEVICE)     # noqa: E731
    return dict(c=c, logits=torch.randn((R, V), generator=g, device=DEVICE) * 3, out=torch.empty((R, V), device=DEVICE),
                rows=torch.randperm(R, generator=g, device=DEVICE).to(torch.int32), seen=_words(seen), counts=counts,
                penalties=torch.stack([pick([1.0, 1.1, 1.3]), pick([0.0, 0.2, 0.7]), pick([0.0, 0.5, -0.1])], 1).float().contiguous(),
                bias_cu=_ints(_cu(n_bias)), bias_tokens=torch.cat(biased) if c["bias"] else None,
                bias_values=torch.randn(sum(n_bias), generator=g, device=DEVICE) * 5 if c["bias"] else None,
                masks=_words((torch.rand((c["masks"], V), generator=g, device=DEVICE) < c["allowed"]).long()) if c["masks"] else None,
                mask_of=_ints(_mask_of(c)) if c["masks"] else None)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    return {"attention": _prepare_attention, "tables": _prepare_tables, "history": _prepare_history, "steer": _prepare_steer}[case["kind"]](case, g)


# ---- the plain forms -------------------------------------------------------
def _plain_attention(s):
    """Scores against a group's shared keys for all of its tokens at once, against a token's own ones one by one; one softmax over both."""
    c, b = s["c"], s["batch"]
    H, KV, D = c["heads"], c["kv"], c["dim"]
    n, group = b.n_tokens, H // KV
    q = s["q"].float().view(n, KV, group, D)
    cu, first = s["cu_groups"].long(), b.cu_seqlens.long()
    seq, positions, pages = b.seq_of_token.long(), b.positions.long(), s["pages"].long()
    tok_first, G = first[cu[:-1]], pages.numel()
    g_of_tok = s["group_of"].long()[seq]
    place = torch.arange(n, device=q.device) - tok_first[g_of_tok]
    # a group's tokens, filled up to the largest group's number
    rows = torch.zeros((G, s["most"], KV, group, D), device=q.device)
    rows[g_of_tok, place] = q
    rows = rows.permute(0, 2, 1, 3, 4).reshape(G, KV, s["most"] * group, D)
    ids = b.page_table[cu[:-1], :s["max_pages"]].long()                       # [G, pages]
    L = s["max_pages"] * PAGE
    shared = s["kv"][ids].float()                                             # [G, pages, 2, KV, 64, D]
    k1, v1 = (shared[:, :, i].permute(0, 2, 1, 3, 4).reshape(G, KV, L, D) for i in (0, 1))
    s1 = torch.matmul(rows, k1.transpose(2, 3)) * s["scale"]                  # [G, KV, rows, L]
    s1 = s1.masked_fill(torch.arange(L, device=q.device) >= (pages * PAGE)[:, None, None, None], -math.inf)
    # a token's own keys
    width = -(-s["own_bound"] // PAGE)
    at = pages[g_of_tok][:, None] + torch.arange(width, device=q.device)
    mine = b.page_table[seq[:, None], at.clamp(max=b.table_width - 1)].long()
    key_at = (at[:, :, None] * PAGE + torch.arange(PAGE, device=q.device)).view(n, 1, 1, -1)
    hidden = key_at > positions[:, None, None, None]
    kv2 = s["kv"][mine]                                                       # [n, width, 2, KV, 64, D]
    k2, v2 = (kv2[:, :, i].permute(0, 2, 1, 3, 4).reshape(n, KV, width * PAGE, D).float() for i in (0, 1))
    s2 = (torch.matmul(q, k2.transpose(2, 3)) * s["scale"]).masked_fill(hidden, -math.inf)
    # one softmax
    m1 = s1.amax(-1, keepdim=True) if L else torch.full(s1.shape[:-1] + (1,), -math.inf, device=q.device)
    m1 = torch.where(m1 == -math.inf, torch.zeros_like(m1), m1)
    e1 = torch.exp(s1 - m1)
    back = lambda x: x.view(G, KV, s["most"], group, -1).permute(0, 2, 1, 3, 4)[g_of_tok, place]   # noqa: E731
    o1, l1, m1 = back(torch.matmul(e1, v1)), back(e1.sum(-1, keepdim=True)), back(m1)
    m2 = s2.amax(-1, keepdim=True)
    e2 = torch.exp(s2 - m2)
    o2, l2 = torch.matmul(e2, v2.masked_fill(hidden.transpose(2, 3), 0.0)), e2.sum(-1, keepdim=True)
    m = torch.where(l1 > 0, torch.maximum(m1, m2), m2)
    f1, f2 = torch.where(l1 > 0, torch.exp(m1 - m), torch.zeros_like(m)), torch.exp(m2 - m)
    return ((o1 * f1 + o2 * f2) / (l1 * f1 + l2 * f2)).reshape(n, H, D).to(s["q"].dtype)


def _plain_tables(s):
    start, q, slots, free, width = s["start"].long(), s["q_len"].long(), s["slots"].long(), s["free_pages"], s["width"]
    held, total = (start + PAGE - 1) // PAGE, (start + q + PAGE - 1) // PAGE
    need = total - held
    first = s["free_head"].long() + need.cumsum(0) - need
    j = torch.arange(width, device=start.device)
    parent = s["parent"].long()
    old = s["tables"][torch.where(parent >= 0, parent, slots)]
    at = first[:, None] + j - held[:, None]
    new = torch.where((at >= 0) & (at < free.numel()), free[at.clamp(0, free.numel() - 1)], 0)
    table = torch.where(j < held[:, None], old, torch.where(j < total[:, None], new, 0)).to(torch.int32)
    s["tables"][slots] = torch.where(j < total[:, None], table, s["tables"][slots])
    end = q.cumsum(0)
    cu = torch.cat([torch.zeros_like(end[:1]), end])
    t = torch.arange(s["n"], device=start.device)
    seq = torch.searchsorted(end, t, right=True)
    pos = start[seq] + t - cu[seq]
    slot = table[seq, pos // PAGE].long() * PAGE + pos % PAGE
    i32 = torch.int32
    return [table, cu.to(i32), (start + q).to(i32), pos.to(i32), seq.to(i32), slot, (s["free_head"] + need.sum()).to(i32), s["tables"]]


def _plain_history(s):
    R, V = s["counts"].shape
    at = lambda row, tok: row.long() * V + tok.long()                         # noqa: E731
    counts = torch.zeros(R * V, dtype=torch.int32, device=DEVICE)
    out = at(s["output_row"], s["output"])
    counts.index_add_(0, out, torch.ones_like(out, dtype=torch.int32))
    seen = torch.zeros(R * V, dtype=torch.int64, device=DEVICE)
    seen[at(s["prompt_row"], s["prompt"])] = 1
    seen[out] = 1
    return [_words(seen.view(R, V)), counts.view(R, V)]


def _plain_steer(s):
    V, r = s["c"]["vocab"], s["rows"].long()
    x, pen = s["logits"], s["penalties"][r]
    n = s["counts"][r].float()
    x = torch.where(_bits(s["seen"], V)[r] > 0, torch.where(x > 0, x / pen[:, :1], x * pen[:, :1]), x)
    x = x - (pen[:, 1:2] * n + pen[:, 2:3] * (n > 0))
    if s["bias_tokens"] is not None:
        k = torch.arange(s["bias_tokens"].numel(), device=x.device)
        row = torch.searchsorted(s["bias_cu"][1:].long(), k, right=True)
        bias = torch.zeros_like(x)
        bias[row, s["bias_tokens"].long()] = s["bias_values"]
        x = x + bias[r]
    if s["masks"] is not None:
        which = s["mask_of"].long()[r]
        x = x.masked_fill((which >= 0)[:, None] & (_bits(s["masks"], V)[which.clamp(min=0)] == 0), -math.inf)
    return x


# ---- the framework's operators ---------------------------------------------
def _own_attention(s):
    from wick_b200 import ops
    shared = ops.SharedPrefix(s["cu_groups"], s["pages"], s["group_of"], max_pages=s["max_pages"], own_bound=s["own_bound"])
    return ops.attention_shared(s["q"], s["kv"], s["batch"], shared, s["scale"])


def _own_tables(s):
    from wick_b200 import ops
    o = s["out"]
    ops.step_tables(s["start"], s["q_len"], s["slots"], s["tables"], s["free_pages"], s["free_head"], parent=s["parent"], **o)
    return [o["page_table"], o["cu_seqlens"], o["kv_len"], o["positions"], o["seq_of_token"], o["slot_map"], o["head_out"], s["tables"]]


def _own_history(s):
    from wick_b200 import ops
    ops.history_clear(s["seen"], s["counts"], s["rows"])
    ops.history_add(s["seen"], s["counts"], s["prompt"], s["prompt_row"], generated=False)
    ops.history_add(s["seen"], s["counts"], s["output"], s["output_row"], generated=True)
    return [s["seen"], s["counts"]]


def _own_steer(s):
    from wick_b200 import ops
    bias = None if s["bias_tokens"] is None else (s["bias_cu"], s["bias_tokens"], s["bias_values"])
    return ops.steer_logits(s["logits"], s["rows"], seen=s["seen"], counts=s["counts"], penalties=s["penalties"], bias=bias, masks=s["masks"],
                            mask_of=s["mask_of"], out=s["out"])


def run(state):
    kind = state["c"]["kind"]
    if own:
        return {"attention": _own_attention, "tables": _own_tables, "history": _own_history, "steer": _own_steer}[kind](state)
    return {"attention": _plain_attention, "tables": _plain_tables, "history": _plain_history, "steer": _plain_steer}[kind](state)


# ---- the definition in 64 bits ---------------------------------------------
def exact(case, seed):
    """One sequence, or one row, after the other."""
    s = prepare(case, seed)
    if case["kind"] == "attention":
        b, group = s["batch"], case["heads"] // case["kv"]
        out, t = [], 0
        for i, (start, new) in enumerate(zip(b.starts, b.q_lens)):
            end = start + new
            kv = s["kv"][b.page_table[i, :_pages(end)].long()].double()      # [pages, 2, KV, 64, D]
            k, v = kv.permute(1, 2, 0, 3, 4).reshape(2, case["kv"], -1, case["dim"])[:, :, :end]
            q = s["q"][t:t + new].double().view(new, case["kv"], group, case["dim"])
            score = torch.einsum("nkgd,kld->nkgl", q, k) * s["scale"]
            late = torch.arange(end, device=q.device) > (start + torch.arange(new, device=q.device))[:, None]
            p = torch.softmax(score.masked_fill(late[:, None, None], -math.inf), -1)
            out.append(torch.einsum("nkgl,kld->nkgd", p, v).reshape(new, case["heads"], case["dim"]))
            t += new
        return torch.cat(out)
    if case["kind"] == "steer":
        out = []
        v = torch.arange(case["vocab"], device=DEVICE)
        for i, r in enumerate(s["rows"].tolist()):
            x = s["logits"][i].double()
            rep, freq, pres = s["penalties"][r].double()
            seen = ((s["seen"][r][v // 32] >> (v % 32)) & 1).bool()
            x[seen] = torch.where(x[seen] > 0, x[seen] / rep, x[seen] * rep)
            n = s["counts"][r].double()
            x = x - freq * n - pres * (n > 0)
            if s["bias_tokens"] is not None:
                lo, hi = s["bias_cu"][r].item(), s["bias_cu"][r + 1].item()
                x[s["bias_tokens"][lo:hi].long()] += s["bias_values"][lo:hi].double()
            m = -1 if s["masks"] is None else s["mask_of"][r].item()
            if m >= 0:
                x[((s["masks"][m][v // 32] >> (v % 32)) & 1) == 0] = -math.inf
            out.append(x)
        return torch.stack(out)
    return None                                                              # (whole numbers)
