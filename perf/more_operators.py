"""The operators of a cache whose keys and values are held in 4 bits, as cases that can be timed and compared.

A case is one call of one operator, as a step of the engine makes it:

* ``append``     the projection's output of a step's new tokens: q and k normed per head and rotated, k and v stored in the paged cache in
  4 bits; what the cache then holds for these tokens is read back (the values that the codes stand for);
* ``attention``  causal attention of a step's new tokens (one a sequence, a few, or whole prompts) over such a cache.

The cache, ``[pages, kv_heads, 80 d]`` bytes with pages of 64 positions, holds per page and head, one behind the other: the keys' codes
(64 rows of d / 2 bytes), the values' codes, the keys' scales (64 rows of d / 32 pairs of bfloat16 numbers a, b) and the values' scales.
The value of code c (0 to 15) in a group of 32 neighbouring channels is bfloat16(b + a (1 + c / 16)).  A group's numbers x are stored
with a = bfloat16(16 (max - min) / 15), b = bfloat16(min - a) and c the whole number nearest to 16 (x - b) / a - 16 (halves to the even one),
kept within 0 to 15; 0 where a is 0.
Keys: eight channels a word, channel 8 w + i in bits 4 i to 4 i + 3, the word then turned left by 3 bits.  Values: two channels a byte, the
even one in the low bits, the byte then turned left by 3; a row's pieces of 32 bytes change places with the row's number (``_piece``).

Where ``own`` is false an operator is computed in its plain form: elementary torch operations in 32 bits, and in 64 where a number is
assigned its code.  Head layouts are those of the benchmark's models, besides generic ones.  Which lengths a case has follows from
the case alone; the seed makes the numbers.
"""
import math
import random
import types

import torch

own = False

DEVICE = "cuda:0"
PAGE = 64
EPS = 1e-6
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def _append(batch, low, high, tokens, splits, heads, kv, dim, dtype, name=None):
    """low, high: a sequence's cached positions before the step lie between them; tokens: the most new tokens of a sequence; splits: the
    float32 partial sums that the projection leaves (0: one array in the activations' type)."""
    c = dict(kind="append", batch=batch, low=low, high=high, tokens=tokens, splits=splits, heads=heads, kv=kv, dim=dim, dtype=dtype)
    return dict(c, name=name) if name else c


def _attention(batch, low, high, tokens, heads, kv, dim, dtype, name=None):
    c = dict(kind="attention", batch=batch, low=low, high=high, tokens=tokens, heads=heads, kv=kv, dim=dim, dtype=dtype)
    return dict(c, name=name) if name else c


def listed():
    return [
        # One sequence's next token: all latency.  The decode product leaves its sum in eight runs.
        _append(1, 777, 777, 1, 8, 32, 8, 128, "bfloat16", "append_8b_b1"),
        # A full batch's next tokens.
        _append(64, 10, 9000, 1, 4, 40, 8, 128, "bfloat16", "append_14b_b64"),
        # Prompts of unequal lengths that start together.
        _append(5, 0, 0, 1300, 1, 32, 8, 128, "bfloat16", "append_8b_prompts"),
        # A single short conversation on a small model: all latency.
        _attention(1, 700, 700, 1, 16, 2, 128, "bfloat16", "decode_2k_b1"),
        # A few conversations.
        _attention(8, 500, 4000, 1, 32, 8, 128, "bfloat16", "decode_8b_b8"),
        # A full batch of long ones: what the cache's size in memory decides.
        _attention(64, 4000, 8191, 1, 32, 8, 128, "bfloat16", "decode_8b_b64"),
        # Two very long documents, eight query heads to a key head.
        _attention(2, 100000, 130900, 1, 64, 8, 128, "bfloat16", "decode_32b_long"),
        # Many short ones; seven query heads to a key head, heads of 64, no power of two anywhere.
        _attention(37, 0, 900, 1, 14, 2, 64, "bfloat16", "decode_odd"),
        # The 32-bit path.
        _attention(6, 100, 1000, 1, 16, 2, 128, "float32", "decode_2k_f32"),
        # A few tokens a sequence: drafts that are checked, short replies.
        _attention(16, 2000, 6000, 5, 32, 8, 128, "bfloat16", "drafts_8b_b16"),
        # A prompt from its first token on.
        _attention(1, 0, 0, 2048, 32, 8, 128, "bfloat16", "prompt_8b_2048"),
        # New turns behind what several conversations hold.
        _attention(6, 300, 7000, 500, 40, 8, 128, "bfloat16", "turns_14b_b6"),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm (from 1 on)."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(max(low, 1)), math.log(high)))))))


def _drawn(rng):
    heads, kv, dim = rng.choice([(32, 8, 128), (40, 8, 128), (64, 8, 128), (16, 2, 128), (14, 2, 64), (8, 8, 64), (32, 2, 128), (16, 16, 128), (16, 4, 256)])
    dtype = rng.choice(["bfloat16"] * 5 + ["float32"])
    if rng.random() < 0.3:
        if rng.random() < 0.5:
            high = _spread(rng, 1, 20000)
            return _append(_spread(rng, 1, 128), rng.randint(0, high), high, 1, rng.choice([1, 2, 4, 8]), heads, kv, dim, dtype)
        high = rng.choice([0, _spread(rng, 1, 5000)])
        return _append(_spread(rng, 1, 8), 0, high, _spread(rng, 2, 1500), rng.choice([0, 1]), heads, kv, dim, dtype)
    if rng.random() < 0.6:
        high = _spread(rng, 1, 1500 if dtype == "float32" else 40000)
        return _attention(_spread(rng, 1, 96), rng.randint(0, high), high, 1, heads, kv, dim, dtype)
    high = rng.choice([0, _spread(rng, 1, 7000)])
    return _attention(_spread(rng, 1, 16), 0, high, _spread(rng, 2, 300 if dtype == "float32" else 1500), heads, kv, dim, dtype)


def draw(rng):
    most = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    held = max(_held(c) for c in listed())
    while True:
        c = _drawn(rng)
        w = work(c)
        # (a product in 32 bits off the tensor cores costs about twenty of the others')
        if w["bytes"] <= most["bytes"] and w["flops"] * (20 if c["dtype"] == "float32" else 1) <= most["flops"] and _held(c) <= held:
            return c


# ---- sizes -----------------------------------------------------------------
def _lengths(c):
    """Cached and new tokens of each sequence; the first one has the most of both."""
    rng = random.Random(",".join("%s=%s" % (k, c[k]) for k in sorted(c) if k != "name"))
    n = c["batch"]
    starts = [c["high"] if b == 0 else rng.randint(c["low"], c["high"]) for b in range(n)]
    return starts, [c["tokens"] if b == 0 else rng.randint(1, c["tokens"]) for b in range(n)]


def _pages(n):
    return -(-n // PAGE)


def _held(c):
    """Numbers that the plain form holds at most: keys and values of all sequences at the longest one's length, or all scores."""
    longest = c["batch"] * PAGE * _pages(c["high"] + c["tokens"])
    return max(2 * longest * c["kv"] * c["dim"], longest * c["tokens"] * c["heads"]) if c["kind"] == "attention" else 0


def work(case):
    starts, q = _lengths(case)
    width = 2 if case["dtype"] == "bfloat16" else 4
    n, kv, d = sum(q), case["kv"], case["dim"]
    rows = n * case["heads"] * d
    if case["kind"] == "append":
        taken = (rows + 2 * n * kv * d) * (4 * case["splits"] if case["splits"] else width)
        return {"bytes": taken + rows * width + 4 * n * d + 2 * n * kv * d * 5 // 8 + 4 * n * kv * d, "flops": 8 * rows + 20 * n * kv * d}
    cached = sum(s + t for s, t in zip(starts, q))
    seen = sum(t * s + t * (t + 1) // 2 for s, t in zip(starts, q))
    return {"bytes": 2 * cached * kv * d * 5 // 8 + 2 * rows * width, "flops": 4 * d * case["heads"] * seen}


# ---- the cache's form ------------------------------------------------------
def _turn_left(x, by, bits):
    return ((x << by) | (x >> (bits - by))) & ((1 << bits) - 1)


def _piece(rows, dim):
    """[rows, d / 64]: which piece of 32 bytes of a row of the values' codes stands at each place."""
    t = rows[:, None]
    turn = (t & 1) | (t >> 1 & 2) if dim == 256 else t >> 2 & 1 if dim == 128 else t * 0
    return torch.arange(dim // 64, device=rows.device) ^ turn


def _codes(x):
    """[..., d] -> codes (int64) [..., d], a and b (bfloat16) [..., d / 32]; in 64 bits."""
    g = x.double().unflatten(-1, (-1, 32))
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    a = ((high - low) * (16.0 / 15.0)).to(torch.bfloat16)
    b = (low - a.double()).to(torch.bfloat16)
    c = torch.where(a == 0, 0.0, ((g - b.double()) * 16.0 / a.double() - 16.0).round().clamp(0, 15)).long()
    return c.flatten(-2), a.squeeze(-1), b.squeeze(-1)


def _values(codes, a, b):
    """What codes stand for, as bfloat16 numbers."""
    c = codes.unflatten(-1, (-1, 32)).float()
    return (b.float()[..., None] + a.float()[..., None] * (1.0 + c / 16.0)).to(torch.bfloat16).flatten(-2)


def _key_bytes(codes):
    """[..., d] -> uint8 [..., d / 2]."""
    w = (codes.unflatten(-1, (-1, 8)) << torch.arange(0, 32, 4, device=codes.device)).sum(-1)
    w = _turn_left(w, 3, 32)
    return (w[..., None] >> torch.arange(0, 32, 8, device=codes.device) & 255).to(torch.uint8).flatten(-2)


def _value_bytes(codes, rows):
    """[n, ..., d] codes of positions ``rows`` [n] of their pages -> uint8 [n, ..., d / 2]."""
    p = codes.unflatten(-1, (-1, 2))
    v = _turn_left(p[..., 0] | p[..., 1] << 4, 3, 8).to(torch.uint8)
    dim = codes.shape[-1]
    at = _piece(rows, dim)
    at = (at[..., None] * 32 + torch.arange(32, device=rows.device)).flatten(1)
    at = at.view((at.shape[0],) + (1,) * (v.dim() - 2) + (-1,)).expand_as(v)
    return v.gather(-1, at)


def _scale_bytes(a, b):
    return torch.stack([a, b], -1).contiguous().view(torch.uint8).flatten(-2)


def _open(pages, dim):
    """uint8 [..., 80 d] -> codes of keys and of values (int32, [..., 64, d]), and their a and b (bfloat16, [..., 64, d / 32])."""
    half = 32 * dim
    kc, vc, sc = pages[..., :half], pages[..., half:2 * half], pages[..., 2 * half:]
    kc = kc.contiguous().view(torch.int32)
    # (turned back right by 3: the upper bits of an arithmetic shift are taken out)
    kc = (kc >> 3 & 0x1FFFFFFF) | kc << 29
    keys = (kc[..., None] >> torch.arange(0, 32, 4, device=pages.device, dtype=torch.int32) & 15).flatten(-2).unflatten(-1, (PAGE, dim))
    rows = torch.arange(PAGE, device=pages.device)
    at = (_piece(rows, dim)[..., None] * 32 + torch.arange(32, device=pages.device)).flatten(1)
    vc = vc.unflatten(-1, (PAGE, dim // 2))
    vc = vc.gather(-1, at.expand_as(vc)).int()
    vc = vc >> 3 | (vc & 7) << 5
    values = torch.stack([vc & 15, vc >> 4], -1).flatten(-2)
    sc = sc.contiguous().view(torch.bfloat16).unflatten(-1, (2, PAGE, dim // 32, 2))
    return keys, values, sc[..., 0, :, :, :], sc[..., 1, :, :, :]


def _put(kv, first, width, at, rows, data):
    """Rows [n, kv_heads, width] of bytes into pages ``at`` [n] at positions ``rows`` [n], in the block that begins at byte ``first`` of a head's part."""
    heads = torch.arange(kv.shape[1], device=kv.device)
    kv[:, :, first:first + PAGE * width].unflatten(-1, (PAGE, width))[at[:, None], heads, rows[:, None]] = data


def _store(kv, at, rows, k, v):
    """Keys and values [n, kv_heads, d] into pages ``at`` [n] at their positions ``rows`` [n]; what the cache then holds, [2, n, kv_heads, d]."""
    dim = k.shape[-1]
    (kc, ka, kb), (vc, va, vb) = _codes(k), _codes(v)
    _put(kv, 0, dim // 2, at, rows, _key_bytes(kc))
    _put(kv, 32 * dim, dim // 2, at, rows, _value_bytes(vc, rows))
    _put(kv, 64 * dim, dim // 8, at, rows, _scale_bytes(ka, kb))
    _put(kv, 72 * dim, dim // 8, at, rows, _scale_bytes(va, vb))
    return torch.stack([_values(kc, ka, kb), _values(vc, va, vb)])


# ---- inputs ----------------------------------------------------------------
def _ints(v):
    return torch.tensor(v, dtype=torch.int32).to(DEVICE)


def _batch(starts, q, g):
    """A step's description: sequences' lengths, and pages in no order."""
    n, kv_len = sum(q), [s + t for s, t in zip(starts, q)]
    need = [_pages(k) for k in kv_len]
    width = max(need)
    total = 1 + sum(need)
    ids = torch.randperm(total - 1, generator=g, device=DEVICE) + 1
    cu = [sum(q[:i]) for i in range(len(q) + 1)]
    need_t, j = _ints(need).long(), torch.arange(width, device=DEVICE)
    first = need_t.cumsum(0) - need_t
    table = torch.where(j < need_t[:, None], ids[(first[:, None] + j).clamp(max=total - 2)], 0).to(torch.int32)
    seq = torch.arange(len(q), device=DEVICE).repeat_interleave(_ints(q).long())
    positions = _ints(starts)[seq] + torch.arange(n, device=DEVICE) - _ints(cu)[seq]
    return total, types.SimpleNamespace(
        n_seqs=len(q), n_tokens=n, table_width=width, q_lens=q, starts=starts, max_q_len=max(q), max_kv_len=max(kv_len), kv_bound=max(kv_len),
        is_decode=max(q) == 1, cu_seqlens=_ints(cu), start=_ints(starts), kv_len=_ints(kv_len), page_table=table,
        seq_of_token=seq.to(torch.int32), positions=positions.to(torch.int32))


def prepare(case, seed):
    c, g = case, torch.Generator(device=DEVICE).manual_seed(int(seed))
    starts, q = _lengths(c)
    total, batch = _batch(starts, q, g)
    n, H, KV, D, dt = batch.n_tokens, c["heads"], c["kv"], c["dim"], DTYPES[c["dtype"]]
    # (as in trained models some channels of the keys are larger than others, and some stand beside zero)
    size = torch.linspace(0.5, 2.0, D, device=DEVICE)[torch.randperm(D, generator=g, device=DEVICE)]
    offset = torch.where(torch.rand(D, generator=g, device=DEVICE) < 0.1, 2.0, 0.0)
    if c["kind"] == "append":
        kv = torch.zeros((total, KV, 80 * D), dtype=torch.uint8, device=DEVICE)
        x = torch.randn((max(c["splits"], 1), n, (H + 2 * KV) * D), generator=g, device=DEVICE)
        half = D // 2
        angle = batch.positions.double()[:, None] * 1e6 ** (-torch.arange(half, device=DEVICE).double() / half)
        return dict(c=c, kv=kv, batch=batch, qkv=x if c["splits"] else x[0].to(dt), dtype=dt, cos=angle.cos().float(), sin=angle.sin().float(),
                    q_weight=1.0 + 0.1 * torch.randn(D, generator=g, device=DEVICE), k_weight=size + 0.1 * torch.randn(D, generator=g, device=DEVICE))
    kv = torch.empty((total, KV, 80 * D), dtype=torch.uint8, device=DEVICE)
    step = max(1, (1 << 27) // (KV * PAGE * D))                     # (some pages at a time: what lies in between stays small)
    for p in range(0, total, step):
        m = min(step, total - p)
        k = torch.randn((m, KV, PAGE, D), generator=g, device=DEVICE) * size + offset
        v = torch.randn((m, KV, PAGE, D), generator=g, device=DEVICE)
        parts, scales = [], []
        for i, x in ((0, k), (1, v)):
            codes, a, b = _codes(x)
            rows = torch.arange(PAGE, device=DEVICE)
            parts.append(_key_bytes(codes).flatten(2) if i == 0 else _value_bytes(codes.permute(2, 0, 1, 3), rows).permute(1, 2, 0, 3).flatten(2))
            scales.append(_scale_bytes(a, b).flatten(2))
        kv[p:p + m] = torch.cat(parts + scales, -1)
    query = torch.randn((n, H, D), generator=g, device=DEVICE)
    # (some heads look sharply, some all around)
    query = (query * torch.linspace(0.3, 1.5, H, device=DEVICE)[:, None]).to(dt)
    return dict(c=c, kv=kv, batch=batch, q=query, scale=1.0 / math.sqrt(D))


# ---- the plain forms -------------------------------------------------------
def _normed(x, weight):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight


def _rotated(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos[:, None] - b * sin[:, None], b * cos[:, None] + a * sin[:, None]], -1)


def _plain_append(s):
    c, b = s["c"], s["batch"]
    H, KV, D = c["heads"], c["kv"], c["dim"]
    x = s["qkv"].double().sum(0) if s["qkv"].dim() == 3 else s["qkv"].double()
    q, k, v = x.unflatten(1, (H + 2 * KV, D)).split([H, KV, KV], 1)
    cos, sin = s["cos"].double(), s["sin"].double()
    q, k = _rotated(_normed(q, s["q_weight"]), cos, sin), _rotated(_normed(k, s["k_weight"]), cos, sin)
    at = b.page_table[b.seq_of_token.long(), b.positions.long() // PAGE].long()
    held = _store(s["kv"], at, b.positions.long() % PAGE, k, v)
    return [q.to(s["dtype"]), held]


def _plain_attention(s):
    """Every sequence filled up to the longest one's length and number of new tokens."""
    c, b = s["c"], s["batch"]
    H, KV, D = c["heads"], c["kv"], c["dim"]
    B, T, L = b.n_seqs, b.max_q_len, b.table_width * PAGE
    keys, values, ks, vs = _open(s["kv"][b.page_table.long()], D)              # [B, pages, KV, 64, ...]
    k = _values(keys, ks[..., 0], ks[..., 1]).permute(0, 2, 1, 3, 4).reshape(B, KV, L, D).float()
    v = _values(values, vs[..., 0], vs[..., 1]).permute(0, 2, 1, 3, 4).reshape(B, KV, L, D).float()
    seq = b.seq_of_token.long()
    place = torch.arange(b.n_tokens, device=seq.device) - b.cu_seqlens.long()[seq]
    q = torch.zeros((B, T, KV, H // KV, D), device=seq.device)
    q[seq, place] = s["q"].float().view(-1, KV, H // KV, D)
    score = torch.matmul(q.permute(0, 2, 1, 3, 4).reshape(B, KV, T * (H // KV), D), k.transpose(2, 3)).view(B, KV, T, H // KV, L) * s["scale"]
    sees = b.start.long()[:, None] + torch.arange(T, device=seq.device)         # [B, T]: the last position that a token sees
    late = torch.arange(L, device=seq.device) > sees[..., None]
    score.masked_fill_(late[:, None, :, None], -math.inf)
    score -= score.amax(-1, keepdim=True)
    p = score.exp_()
    total = p.sum(-1, keepdim=True)
    # (what pages hold behind a sequence's end is nobody's)
    v = v.masked_fill((torch.arange(L, device=seq.device) >= b.kv_len.long()[:, None])[:, None, :, None], 0.0)
    out = torch.matmul(p.view(B, KV, T * (H // KV), L), v).view(B, KV, T, H // KV, D) / total
    return out.permute(0, 2, 1, 3, 4)[seq, place].reshape(-1, H, D).to(s["q"].dtype)


# ---- the framework's operators ---------------------------------------------
def _own_append(s):
    from wick_b200 import ops
    c, b = s["c"], s["batch"]
    q = ops.qk_norm_rope_append_kv4(s["qkv"], c["heads"], c["kv"], c["dim"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS, cos=s["cos"],
                                    sin=s["sin"], kv=s["kv"], page_table=b.page_table, seq_of_token=b.seq_of_token, positions=b.positions,
                                    dtype=s["dtype"])
    return [q, ops.kv4_read(s["kv"], c["dim"], b.page_table, b.seq_of_token, b.positions)]


def _own_attention(s):
    from wick_b200 import ops
    return ops.attention_kv4(s["q"], s["kv"], s["batch"], s["scale"])


def run(state):
    append = state["c"]["kind"] == "append"
    if own:
        return _own_append(state) if append else _own_attention(state)
    return _plain_append(state) if append else _plain_attention(state)


# ---- the definition in 64 bits ---------------------------------------------
def _exact_append(s):
    """One head of one kind after the other."""
    c, b = s["c"], s["batch"]
    H, KV, D = c["heads"], c["kv"], c["dim"]
    x = s["qkv"].to(torch.float64)
    x = (x if x.dim() == 2 else x.sum(0)).reshape(-1, H + 2 * KV, D)
    cos, sin = s["cos"].to(torch.float64), s["sin"].to(torch.float64)
    heads = []
    for h in range(H + 2 * KV):
        y = x[:, h]
        if h < H + KV:
            w = (s["q_weight"] if h < H else s["k_weight"]).to(torch.float64)
            y = y / torch.sqrt((y * y).sum(1, keepdim=True) / D + EPS) * w
            u, w = y[:, :D // 2], y[:, D // 2:]
            y = torch.cat((u * cos - w * sin, u * sin + w * cos), 1)
        if h >= H:
            groups = []
            for z in y.split(32, 1):
                low, high = z.min(1, keepdim=True).values, z.max(1, keepdim=True).values
                a = ((high - low) * 16 / 15).to(torch.bfloat16).to(torch.float64)
                e = (low - a).to(torch.bfloat16).to(torch.float64)
                code = torch.clamp(torch.round(16 * (z - e) / torch.where(a > 0, a, 1.0) - 16), 0, 15) * (a > 0)
                groups.append((e + a * (1 + code / 16)).to(torch.bfloat16).to(torch.float64))
            y = torch.cat(groups, 1)
        heads.append(y)
    return [torch.stack(heads[:H], 1), torch.stack([torch.stack(heads[H:H + KV], 1), torch.stack(heads[H + KV:], 1)])]


def _exact_pages(pages, D):
    """Keys and values, [n 64, D], from pages' bytes [n, 80 D]."""
    n, out = pages.shape[0], []
    byte = pages.to(torch.int64)
    t = torch.arange(PAGE, device=pages.device)
    for i in range(2):
        x = torch.empty((n, PAGE, D), dtype=torch.float64, device=pages.device)
        code = byte[:, i * 32 * D:(i + 1) * 32 * D].reshape(n, PAGE, D // 2)
        scale = pages[:, 64 * D + i * 8 * D:64 * D + (i + 1) * 8 * D].contiguous().view(torch.bfloat16).to(torch.float64).reshape(n, PAGE, D // 32, 2)
        for ch in range(D):
            if i == 0:
                w = sum(code[:, :, ch // 8 * 4 + k] << 8 * k for k in range(4))
                bit = 4 * (ch % 8) + 3
                nibble = (w >> bit if bit < 29 else w >> bit | w << 32 - bit) & 15
            else:
                turn = (t % 2) + 2 * (t // 4 % 2) if D == 256 else t // 4 % 2 if D == 128 else 0 * t
                at = ((ch // 64) ^ turn) * 32 + ch % 64 // 2
                v = code[:, t, at]
                nibble = v // 8 % 16 if ch % 2 == 0 else v // 128 + v % 8 * 2
            x[:, :, ch] = scale[:, :, ch // 32, 1] + scale[:, :, ch // 32, 0] * (1 + nibble / 16)
        out.append(x.to(torch.bfloat16).to(torch.float64).reshape(-1, D))
    return out


def exact(case, seed):
    """One sequence after the other."""
    s = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(s)
    b, KV, D = s["batch"], case["kv"], case["dim"]
    out, t = [], 0
    for i, (start, new) in enumerate(zip(b.starts, b.q_lens)):
        end = start + new
        pages = s["kv"][b.page_table[i, :_pages(end)].long()]
        k, v = (x.view(-1, KV, PAGE, D).transpose(0, 1).reshape(KV, -1, D)[:, :end] for x in _exact_pages(pages.view(-1, 80 * D), D))
        q = s["q"][t:t + new].to(torch.float64).view(new, KV, -1, D)
        late = torch.arange(end, device=DEVICE) > (start + torch.arange(new, device=DEVICE))[:, None, None, None]
        p = torch.softmax((torch.einsum("nhgd,hld->nhgl", q, k) * s["scale"]).masked_fill(late, -math.inf), -1)
        out.append(torch.einsum("nhgl,hld->nhgd", p, v).reshape(new, -1, D))
        t += new
    return torch.cat(out)
