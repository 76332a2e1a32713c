"""The cache in 4 bits on the device: what is stored, what is read back, the attention over it, against 64-bit arithmetic."""
import math
import types

import pytest
import torch

from plain import kv4_plain as P

pytestmark = pytest.mark.gpu
PAGE = 64
BF16, F32 = torch.bfloat16, torch.float32


def ops():
    from wick_b200 import ops as o
    return o


def ints(v):
    return torch.tensor(v, dtype=torch.int32).to("cuda")


def step(starts, q, g, spare=0, width=None):
    """A step's description; pages in no order, ``spare`` of them nobody's."""
    kv = [s + n for s, n in zip(starts, q)]
    need = [-(-k // PAGE) for k in kv]
    ids = (torch.randperm(sum(need) + spare, generator=g) + 1).tolist()
    w = width or max(need + [1])
    table, at = [], 0
    for n in need:
        table.append(ids[at:at + n] + [0] * (w - n))
        at += n
    cu = [sum(q[:i]) for i in range(len(q) + 1)]
    seq = [b for b in range(len(q)) for _ in range(q[b])]
    b = types.SimpleNamespace(
        n_seqs=len(q), n_tokens=sum(q), table_width=w, q_lens=q, starts=starts, max_q_len=max(q), max_kv_len=max(kv), kv_bound=max(kv),
        cu_seqlens=ints(cu), start=ints(starts), kv_len=ints(kv), page_table=ints(table), seq_of_token=ints(seq),
        positions=ints([starts[i] + t for i in range(len(q)) for t in range(q[i])]), table=table)
    return sum(need) + spare + 1, b


def random_cache(pages, n_kv, d, g):
    """A cache of random codes and scales (behind a sequence's end as well; any byte is two codes), and its keys and values as float64
    [pages, n_kv, 64, d]."""
    kv = torch.randint(0, 256, (pages, n_kv, 80 * d), generator=g, dtype=torch.uint8)
    a = torch.rand((pages, n_kv, 2, PAGE, d // 32), generator=g) * 2 + 0.5
    b = -1.47 * a + 0.4 * torch.randn(a.shape, generator=g)
    kv[:, :, 64 * d:] = torch.stack([a, b], -1).to(BF16).contiguous().view(torch.uint8).view(pages, n_kv, 16 * d)
    return kv, open_bytes(kv, d)


def open_bytes(kv, d):
    """uint8 [pages, n_kv, 80 d] -> keys and values, float64 [pages, n_kv, 64, d]."""
    pages, n_kv = kv.shape[:2]
    word = kv[:, :, :32 * d].contiguous().view(torch.int32).long() & 0xFFFFFFFF
    word = (word >> 3 | word << 29) & 0xFFFFFFFF
    keys = torch.stack([word >> 4 * i & 15 for i in range(8)], -1).view(pages, n_kv, PAGE, d)
    byte = kv[:, :, 32 * d:64 * d].long().view(pages, n_kv, PAGE, d // 64, 32)
    rows = []
    for t in range(PAGE):
        turn = {64: 0, 128: t // 4 % 2, 192: 0, 256: t % 2 + 2 * (t // 4 % 2)}[d]
        rows.append(byte[:, :, t, [p ^ turn for p in range(d // 64)]].reshape(pages, n_kv, d // 2))
    byte = torch.stack(rows, 2)
    byte = (byte >> 3 | byte << 5) & 255
    values = torch.stack([byte & 15, byte >> 4], -1).view(pages, n_kv, PAGE, d)
    s = kv[:, :, 64 * d:].contiguous().view(BF16).double().view(pages, n_kv, 2, PAGE, d // 32, 2)
    return P.decode(keys, s[:, :, 0, ..., 0], s[:, :, 0, ..., 1]), P.decode(values, s[:, :, 1, ..., 0], s[:, :, 1, ..., 1])


def of_sequence(x, table, length):
    """[pages, n_kv, 64, d] -> [n_kv, length, d]."""
    n = -(-length // PAGE)
    return x[table[:n]].permute(1, 0, 2, 3).reshape(x.shape[1], n * PAGE, -1)[:, :length]


def check_attention(q, out, cache, b, scale, d):
    """Per element: the result's own rounding, the weights' (2^-8 each in bfloat16, of what they weigh), and that of 32-bit sums: a score is a sum
    of d products (2^-23 of the sum of their sizes each, products and additions, in any order, truncated or rounded), turned into an exponent (two
    roundings more of its size) and weighs a value with twice the relative error that the score has absolutely (once itself, once in the sum of the
    weights); sums over the positions round once a position; a fold or a rescaling once a page."""
    t = 0
    keys, values = cache
    for i, n in enumerate(b.q_lens):
        length = b.starts[i] + n
        if n:
            want, size, reach = P.attention(q[t:t + n].double().cpu(), of_sequence(keys, b.table[i], length), of_sequence(values, b.table[i], length),
                                            b.starts[i], scale)
            exact = 2 * (d + 4) * 2.0 ** -23 * reach + (length + 4 * (length // PAGE) + 32) * 2.0 ** -23
            bound = size * exact + (2.0 ** -24 * want.abs() if q.dtype == F32 else 2.0 ** -8 * want.abs() + 2.0 ** -8 * size)
            err = (out[t:t + n].double().cpu() - want).abs()
            assert (err <= bound + 1e-30).all(), (i, n, b.starts[i], (err / (bound + 1e-30)).max().item())
        t += n


# ---- append and read ------------------------------------------------------------------
@pytest.mark.parametrize("heads,n_kv,d", [(4, 2, 64), (6, 2, 128), (5, 1, 192), (4, 4, 256), (7, 7, 64), (40, 8, 128)])
@pytest.mark.parametrize("splits,dtype,norm,turn", [(0, BF16, True, True), (3, BF16, True, True), (1, F32, True, False), (8, BF16, False, True),
                                                    (0, F32, False, False)])
def test_append(heads, n_kv, d, splits, dtype, norm, turn):
    o = ops()
    g = torch.Generator().manual_seed(heads * d + splits)
    pages, b = step([0, 61, 5, 200], [70, 3, 1, 1], g, spare=2)
    n = b.n_tokens
    x = torch.randn((max(splits, 1), n, (heads + 2 * n_kv) * d), generator=g) * 2
    x = x if splits else x[0].to(dtype)
    q_w, k_w = (torch.rand(d, generator=g) + 0.5, torch.rand(d, generator=g) + 0.5) if norm else (None, None)
    angle = b.positions.cpu().double()[:, None] * 1e4 ** (-torch.arange(d // 2).double() / (d // 2))
    cos, sin = (angle.cos().float(), angle.sin().float()) if turn else (None, None)
    up = lambda v: None if v is None else v.cuda()      # noqa: E731
    kv = torch.full((pages, n_kv, 80 * d), 0x5A, dtype=torch.uint8, device="cuda")
    q = o.qk_norm_rope_append_kv4(x.cuda(), heads, n_kv, d, q_weight=up(q_w), k_weight=up(k_w), eps=1e-6, cos=up(cos), sin=up(sin), kv=kv,
                                  page_table=b.page_table, seq_of_token=b.seq_of_token, positions=b.positions, dtype=dtype)
    eps = torch.tensor(1e-6, dtype=F32).double().item()             # (as the kernel gets it)
    want_q, k, v = P.project(x.double().sum(0) if splits else x.double(), heads, n_kv, d, q_w, k_w, eps, cos, sin)
    # 32 bits: the runs' sums, the norm's sum, its root and two products, two products and a sum of the rotation, each half a step of the row's largest
    top = want_q.abs().amax(-1, keepdim=True)
    assert ((q.double().cpu() - want_q).abs() <= (0 if dtype == F32 else 2.0 ** -8) * want_q.abs() + (d + splits + 16) * 2.0 ** -24 * top * 2).all()
    keys, values = P.encode(k), P.encode(v)
    held = o.kv4_read(kv, d, b.page_table, b.seq_of_token, b.positions).double().cpu()
    assert torch.equal(held[0], P.decode(*keys)) and torch.equal(held[1], P.decode(*values))
    # the bytes are where the form says, and no others were touched
    got = kv.cpu()
    blank = torch.full((80 * d,), 0x5A, dtype=torch.uint8)
    t = 0
    for i, new in enumerate(b.q_lens):
        for h in {0, n_kv - 1}:
            for p in {b.starts[i] // PAGE, (b.starts[i] + new - 1) // PAGE}:
                rows = [r for r in range(PAGE) if b.starts[i] <= p * PAGE + r < b.starts[i] + new]
                full = [tuple(torch.zeros((PAGE,) + y.shape[2:], dtype=y.dtype) for y in z) for z in (keys, values)]
                mine = torch.zeros(80 * d, dtype=torch.bool)
                for z, w in zip(full, (keys, values)):
                    for y, s in zip(z, w):
                        for r in rows:
                            y[r] = s[t + p * PAGE + r - b.starts[i], h]
                for r in rows:
                    for first, size in ((0, d // 2), (32 * d, d // 2), (64 * d, d // 8), (72 * d, d // 8)):
                        mine[first + r * size:first + (r + 1) * size] = True
                assert torch.equal(got[b.table[i][p], h], torch.where(mine, P.page_bytes(*full), blank)), (i, h, p)
        t += new
    used = {b.table[i][p] for i in range(b.n_seqs) for p in range(b.starts[i] // PAGE, (b.starts[i] + b.q_lens[i] - 1) // PAGE + 1)}
    assert all(torch.equal(got[p], blank.expand(n_kv, -1)) for p in range(pages) if p not in used)
    o.check_status()


def test_append_without_writing():
    o = ops()
    g = torch.Generator().manual_seed(1)
    _, b = step([3, 9], [2, 1], g)
    x = torch.randn((3, 6 * 64), generator=g).to(BF16).cuda()
    q = o.qk_norm_rope_append_kv4(x, 4, 1, 64, q_weight=None, k_weight=None, eps=0.0, cos=None, sin=None, kv=None, page_table=b.page_table,
                                  seq_of_token=b.seq_of_token, positions=b.positions, write_kv=False)
    assert torch.equal(q, x[:, :256].view(3, 4, 64))


def test_append_of_odd_numbers():
    """Equal numbers, zeros, steps of one size, tiny and huge ranges, halves between two codes, and numbers that are none."""
    o = ops()
    d = 64
    rows = torch.randn((14, 2, d), generator=torch.Generator().manual_seed(3)).double()
    rows[0] = 0.0
    rows[1] = 3.140625
    rows[2] = torch.arange(d).double()
    rows[3] = 1.0 + torch.arange(d).double() / 4096
    rows[4] *= 1e-38
    rows[5] *= 1e37
    rows[6, 0, 5] = math.inf
    rows[7, 1, 40] = math.nan
    rows[8, 0, 33] = -math.inf
    rows[9, 0, 2], rows[9, 0, 3] = 2.9e38, -2.9e38
    rows[10, 1, 2] = 1.9e38
    rows[11] = torch.where(torch.arange(d) % 2 == 0, 0.0, 15.0)
    rows[11, 0, 1::4] = torch.arange(16).double() % 15 + 0.5
    rows[12, 0] = -0.0
    rows[13, 1] *= 2.0 ** -130
    x = rows.float()
    n = x.shape[0]
    b = types.SimpleNamespace(page_table=ints([[1]]), seq_of_token=ints([0] * n), positions=ints(list(range(n))))
    kv = torch.zeros((2, 1, 80 * d), dtype=torch.uint8, device="cuda")
    data = torch.cat([torch.zeros(n, d), x.view(n, 2 * d)], 1).cuda()
    o.qk_norm_rope_append_kv4(data[None].contiguous(), 1, 1, d, q_weight=None, k_weight=None, eps=0.0, cos=None, sin=None, kv=kv, dtype=F32, **vars(b))
    held = o.kv4_read(kv, d, b.page_table, b.seq_of_token, b.positions).double().cpu()[:, :, 0]
    for i in range(2):
        want = P.decode(*P.encode(x.double()[:, i]))
        # (the sizes of numbers below the smallest normal one are not held to be kept: a is 0 or a multiple of 2^-133 there)
        assert torch.equal(torch.isnan(held[i]), torch.isnan(want))
        fine = torch.isfinite(want)
        assert torch.equal(held[i][fine], want[fine])
    for row, i, g in ((6, 0, 0), (7, 1, 1), (8, 0, 1), (9, 0, 0), (10, 1, 0)):
        assert torch.isnan(held[i, row, 32 * g:32 * g + 32]).all() and not torch.isnan(held[i, row, 32 - 32 * g:64 - 32 * g]).any()
    # a number is off by half a step of its group's range, and what rounding the scales adds
    usual = [r for r in range(n) if r not in (6, 7, 8, 9, 10)]
    for i in range(2):
        w = x.double()[usual][:, i].view(-1, 2, 32)
        err = (held[i][usual].view(-1, 2, 32) - w).abs().amax(-1)
        reach, top = w.amax(-1) - w.amin(-1), w.abs().amax(-1)
        assert (err <= reach / 30 + 2.0 ** -8 * (top + 3 * reach) + 1e-39).all()


# ---- attention ------------------------------------------------------------------------
CASES = [
    # starts, new tokens, heads, key heads, head size
    ([0], [1], 4, 2, 64),
    ([63], [1], 8, 1, 128),
    ([64], [1], 3, 3, 192),
    ([700], [1], 16, 2, 128),
    ([0, 1, 62, 127, 511, 512, 513, 1100], [1] * 8, 14, 2, 64),
    ([5, 900, 33], [1, 1, 1], 32, 2, 128),                         # sixteen rows
    ([5, 900, 33], [1, 1, 1], 12, 1, 128),
    ([300, 0, 64], [1, 1, 1], 4, 4, 256),
    ([1000, 63, 0, 64], [3, 2, 5, 1], 8, 2, 128),                  # several tokens
    ([120, 7], [4, 0], 6, 2, 64),                                  # one sequence brings none
    ([250, 0], [9, 20], 4, 2, 192),
    ([70, 0], [33, 7], 4, 1, 256),
    ([0], [130], 4, 2, 128),                                       # opened
    ([0, 100, 511, 64], [65, 33, 1, 64], 8, 2, 64),
    ([640, 3], [17, 200], 16, 4, 128),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(case, dtype):
    o = ops()
    starts, new, H, KV, d = CASES[case]
    g = torch.Generator().manual_seed(case)
    pages, b = step(starts, new, g, spare=1)
    kv, cache = random_cache(pages, KV, d, g)
    q = (torch.randn((b.n_tokens, H, d), generator=g) * 2).to(dtype).cuda()
    scale = 1.0 / math.sqrt(d)
    for plain in (True, False):
        out = o.attention_kv4(q, kv.cuda(), b, scale, plain=plain)
        check_attention(q, out, cache, b, scale, d)
    if dtype == BF16:
        # how the work is shared out changes no bit
        for kinds in (("records", "clusters") + (("stay",) if max(new) * H // KV <= 8 else ()), ("stay",)):
            want = None
            for kind in kinds:
                try:
                    o.attention_kv4_scratch(b, H, KV, d, dtype, kind=kind)
                except o.KernelError:
                    assert kind == "clusters" and max(starts) > 500
                    continue
                got = o.attention_kv4(q, kv.cuda(), b, scale, kind=kind)
                if want is None:
                    check_attention(q, got, cache, b, scale, d)
                    want = got
                assert torch.equal(got, want), kind
        if d in (64, 128):
            check_attention(q, o.attention_kv4(q, kv.cuda(), b, scale, kind="opened"), cache, b, scale, d)
    o.check_status()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_long_sequences(dtype):
    """Leaves of several pages, nodes up to the most there are, with one key head and with sixteen."""
    o = ops()
    for H, KV, length in ((4, 1, 70000), (32, 16, 21000), (16, 2, 40001)):
        g = torch.Generator().manual_seed(length)
        pages, b = step([length, 3], [1, 1], g)
        kv, cache = random_cache(pages, KV, 64, g)
        q = torch.randn((2, H, 64), generator=g).to(dtype).cuda()
        out = o.attention_kv4(q, kv.cuda(), b, 0.125)
        check_attention(q, out, cache, b, 0.125, 64)
        if dtype == BF16:
            assert torch.equal(o.attention_kv4(q, kv.cuda(), b, 0.125, kind="records"), out)
            if H // KV <= 8:
                assert torch.equal(o.attention_kv4(q, kv.cuda(), b, 0.125, kind="stay"), out)
    for H, KV, length, new in ((16, 1, 70000, 1), (8, 8, 9001, 1), (16, 2, 40001, 3)):
        g = torch.Generator().manual_seed(length)
        pages, b = step([length, 3], [new, 1], g)
        kv, cache = random_cache(pages, KV, 128, g)
        q = torch.randn((new + 1, H, 128), generator=g).to(dtype).cuda()
        check_attention(q, o.attention_kv4(q, kv.cuda(), b, 0.1), cache, b, 0.1, 128)
    o.check_status()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_shorter_sequence_of_more_pieces(dtype):
    """80 key heads: 32 pages are cut into 32 pieces, 33 into half as many."""
    o = ops()
    g = torch.Generator().manual_seed(33)
    pages, b = step([33 * PAGE - 1, 32 * PAGE - 3, 31 * PAGE], [1, 2, 1], g)
    kv, cache = random_cache(pages, 80, 64, g)
    q = torch.randn((4, 80, 64), generator=g).to(dtype).cuda()
    for kind in (None, "plain") + (("records", "clusters", "stay") if dtype == BF16 else ()):
        check_attention(q, o.attention_kv4(q, kv.cuda(), b, 0.125, kind=kind), cache, b, 0.125, 64)
    o.check_status()


@pytest.mark.parametrize("H,KV,d,starts,new,dtype", [(32, 16, 192, [70, 0, 5], [1250, 3, 0], BF16), (32, 16, 64, [0, 900], [150, 61], F32),
                                                     (32, 16, 128, [0, 900], [150, 61], BF16)])
def test_prompts_from_the_codes(H, KV, d, starts, new, dtype):
    """So many row tiles that no sequence is cut."""
    o = ops()
    g = torch.Generator().manual_seed(d)
    pages, b = step(starts, new, g, spare=2)
    kv, cache = random_cache(pages, KV, d, g)
    q = torch.randn((b.n_tokens, H, d), generator=g).to(dtype).cuda()
    for kind in ("plain",) + (("records", "stay") if dtype == BF16 else ()):
        check_attention(q, o.attention_kv4(q, kv.cuda(), b, 0.11, kind=kind), cache, b, 0.11, d)
        if kind == "plain" or d == 192:
            assert o.attention_kv4_scratch(b, H, KV, d, dtype, kind=kind) == 0
    o.check_status()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_alone_and_among_others(dtype):
    o = ops()
    g = torch.Generator().manual_seed(5)
    starts, new = [2000, 10, 700, 64, 5000, 0, 130], [1] * 7
    starts, new = starts + [900 + 7 * i for i in range(83)], new + [1] * 83      # (together: blocks that stay)
    pages, b = step(starts, new, g)
    kv = random_cache(pages, 2, 128, g)[0].cuda()
    q = torch.randn((90, 8, 128), generator=g).to(dtype).cuda()
    out = o.attention_kv4(q, kv, b, 0.09)
    for i in list(range(7)) + [40, 89]:
        one = types.SimpleNamespace(**vars(b))
        one.n_seqs = one.n_tokens = 1
        one.q_lens, one.starts, one.kv_bound = [1], [starts[i]], starts[i] + 1
        one.cu_seqlens, one.start, one.page_table, one.seq_of_token = ints([0, 1]), b.start[i:i + 1].clone(), b.page_table[i:i + 1].clone(), ints([0])
        assert torch.equal(o.attention_kv4(q[i:i + 1].clone(), kv, one, 0.09), out[i:i + 1]), i
        one.kv_bound = b.table_width * PAGE                        # (a bound that is far too large)
        assert torch.equal(o.attention_kv4(q[i:i + 1].clone(), kv, one, 0.09), out[i:i + 1]), i


@pytest.mark.parametrize("new,d", [([1, 1], 128), ([4, 3], 128), ([4, 3], 256), ([40, 41], 64)])
def test_what_is_not_seen_does_not_show(new, d):
    """Numbers that are none behind a sequence's end, in other pages, and in positions that only later tokens see."""
    o = ops()
    g = torch.Generator().manual_seed(d)
    starts = [100, 60]
    pages, b = step(starts, new, g, spare=2)
    kv, cache = random_cache(pages, 2, d, g)
    q = torch.randn((b.n_tokens, 4, d), generator=g).to(BF16).cuda()
    clean = o.attention_kv4(q, kv.cuda(), b, 0.1)
    used = {b.table[i][p]: (i, p) for i in range(2) for p in range(-(-(starts[i] + new[i]) // PAGE))}
    nan = torch.tensor([0.0, math.nan], dtype=BF16).view(torch.uint8)
    scales = kv[:, :, 64 * d:].view(pages, 2, 2, PAGE, d // 32, 4)
    for p in range(pages):
        first = used[p][1] * PAGE if p in used else 0
        end = starts[used[p][0]] + new[used[p][0]] - first if p in used else 0
        scales[p, :, :, max(0, min(PAGE, end)):] = nan
    for plain in (False, True):
        assert torch.equal(o.attention_kv4(q, kv.cuda(), b, 0.1, plain=plain).isnan(), torch.zeros_like(clean, dtype=torch.bool))
    assert torch.equal(o.attention_kv4(q, kv.cuda(), b, 0.1), clean)
    if new[0] > 1 and new[0] <= 8:
        # a value that only the first sequence's last token sees: its channels of that token's rows, nothing else
        last = starts[0] + new[0] - 1
        scales[b.table[0][last // PAGE], 1, 1, last % PAGE, 1] = nan
        want = torch.zeros_like(clean, dtype=torch.bool)
        want[new[0] - 1, 2:, 32:64] = True
        for plain in (False, True):
            assert torch.equal(o.attention_kv4(q, kv.cuda(), b, 0.1, plain=plain).isnan(), want)
        # and a key: all of that token's rows
        scales[b.table[0][last // PAGE], 0, 0, last % PAGE, 0] = nan
        want[new[0] - 1, :2] = True
        for plain in (False, True):
            assert torch.equal(o.attention_kv4(q, kv.cuda(), b, 0.1, plain=plain).isnan(), want)


@pytest.mark.parametrize("scale", [-0.07, 0.0])
def test_scales(scale):
    """A negative scale turns the order of the scores around, one of 0 weighs all alike."""
    o = ops()
    g = torch.Generator().manual_seed(8)
    pages, b = step([100, 700, 0], [1, 1, 1], g)
    kv, cache = random_cache(pages, 2, 128, g)
    q = torch.randn((3, 8, 128), generator=g).to(BF16).cuda()
    for kind in ("plain", "records", "stay"):
        check_attention(q, o.attention_kv4(q, kv.cuda(), b, scale, kind=kind), cache, b, scale, 128)


def test_rows_behind_the_last_sequence_stay():
    o = ops()
    g = torch.Generator().manual_seed(9)
    pages, b = step([100, 700], [1, 1], g)
    kv = random_cache(pages, 2, 64, g)[0].cuda()
    q = torch.randn((4, 4, 64), generator=g).to(BF16).cuda()
    want = o.attention_kv4(q[:2].clone(), kv, b, 0.1)
    b.n_tokens, b.seq_of_token = 4, ints([0, 1, 1, 1])
    for plain in (False, True):
        out = torch.full_like(q, 7.0)
        o.attention_kv4(q, kv, b, 0.1, out=out, plain=plain)
        assert (out[2:] == 7.0).all()
        if not plain:
            assert torch.equal(out[:2], want)


def test_places_beyond_32_bits():
    """A cache of more than 4 GiB, pages at its end."""
    o = ops()
    d, KV = 128, 8
    pages = (1 << 32) // (KV * 80 * d) + 50
    g = torch.Generator().manual_seed(2)
    _, b = step([130, 5], [1, 2], g)
    kv = torch.zeros((pages, KV, 80 * d), dtype=torch.uint8, device="cuda")
    small, cache = random_cache(5, KV, d, g)
    kv[pages - 5:] = small.cuda()
    b.page_table = ints([[p + pages - 5 if p else 0 for p in row] for row in b.table])
    q = torch.randn((3, 16, d), generator=g).to(BF16).cuda()
    x = torch.randn((3, 32 * d), generator=g).cuda()
    o.qk_norm_rope_append_kv4(x[None].contiguous(), 16, KV, d, q_weight=None, k_weight=None, eps=0.0, cos=None, sin=None, kv=kv,
                              page_table=b.page_table, seq_of_token=b.seq_of_token, positions=b.positions, dtype=BF16)
    v = x.double().cpu().view(3, 32, d)[:, 16:]
    held = o.kv4_read(kv, d, b.page_table, b.seq_of_token, b.positions).double().cpu()
    assert torch.equal(held[0], P.decode(*P.encode(v[:, :KV]))) and torch.equal(held[1], P.decode(*P.encode(v[:, KV:])))
    cache = open_bytes(kv[pages - 5:].cpu(), d)
    for plain in (False, True):
        check_attention(q, o.attention_kv4(q, kv, b, 0.08, plain=plain), cache, b, 0.08, d)
    del kv
    torch.cuda.empty_cache()


def test_another_stream_and_replays():
    """Captured once, replayed with other contents; on a stream of its own, two graphs over one scratch in turn."""
    o = ops()
    g = torch.Generator().manual_seed(4)
    d, KV, H = 128, 2, 8
    pages, b = step([900, 30, 64], [1, 1, 1], g)
    kv, cache = random_cache(pages, KV, d, g)
    kv = kv.cuda()
    q = torch.randn((3, H, d), generator=g).to(BF16).cuda()
    x = torch.randn((2, 3, (H + 2 * KV) * d), generator=g).cuda()
    words = o.attention_kv4_scratch(b, H, KV, d, BF16)
    scratch = torch.empty(words, dtype=F32, device="cuda")

    def run(scale):
        y = o.qk_norm_rope_append_kv4(x, H, KV, d, q_weight=None, k_weight=None, eps=0.0, cos=None, sin=None, kv=kv, page_table=b.page_table,
                                      seq_of_token=b.seq_of_token, positions=b.positions, dtype=BF16)
        return o.attention_kv4(y + q, kv, b, scale, scratch)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        first = run(0.1)
        graphs = []
        for scale in (0.1, 0.05):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                out = run(scale)
            graphs.append((graph, out, scale))
        graphs[0][0].replay()
        graphs[1][0].replay()
        assert torch.equal(graphs[0][1], first)
        assert torch.equal(graphs[1][1], run(0.05))
        x.copy_(torch.randn(x.shape, generator=g))
        q.mul_(2)
        b.start.copy_(ints([901, 31, 65 - 1]))
        for graph, out, scale in graphs:
            graph.replay()
            got = out.clone()
            assert torch.equal(got, run(scale))
    torch.cuda.synchronize()
    o.check_status()


def test_many_sequences():
    """More than the blocks that stay have places for."""
    o = ops()
    g = torch.Generator().manual_seed(1030)
    starts = [(7 * i) % 130 for i in range(1030)]
    pages, b = step(starts, [1] * 1030, g)
    kv, cache = random_cache(pages, 1, 64, g)
    q = torch.randn((1030, 4, 64), generator=g).to(BF16).cuda()
    for kind in (None, "records"):
        check_attention(q, o.attention_kv4(q, kv.cuda(), b, 0.125, kind=kind), cache, b, 0.125, 64)
    with pytest.raises(o.KernelError):
        o.attention_kv4(q, kv.cuda(), b, 0.125, kind="stay")
    o.check_status()


@pytest.mark.parametrize("H,KV,d,starts,new", [
    (32, 32, 64, [100 * (i + 4) for i in range(20)] + [5000, 0, 4607, 4608, 63, 2500, 6001], [1] * 27),      # up to nine nodes of a page a leaf, and four of several
    (16, 8, 128, [61 * (i + 20) for i in range(60)], [1 + i % 4 for i in range(60)]),
    (32, 8, 128, [61 * (i + 20) for i in range(45)] + [0], [1 + i % 5 for i in range(45)] + [0]),            # tiles of 24 rows
])
def test_more_nodes_than_warps(H, KV, d, starts, new):
    """Blocks that stay, several rounds of nodes of unequal sequences; 50 pages, which all of them share."""
    o = ops()
    g = torch.Generator().manual_seed(H + KV)
    _, b = step(starts, new, g)
    b.table = [[p % 50 for p in row] for row in b.table]
    b.page_table = ints(b.table)
    kv, cache = random_cache(50, KV, d, g)
    q = torch.randn((b.n_tokens, H, d), generator=g).to(BF16).cuda()
    scale = 1.0 / math.sqrt(d)
    got = o.attention_kv4(q, kv.cuda(), b, scale, kind="stay")
    check_attention(q, got, cache, b, scale, d)
    if max(new) * H // KV <= 8:
        assert torch.equal(o.attention_kv4(q, kv.cuda(), b, scale, kind="records"), got)
    o.check_status()


def test_captured_single_tokens_of_many_heads():
    """96 heads of one key head, captured at short lengths and replayed at longer ones."""
    o = ops()
    g = torch.Generator().manual_seed(96)
    pages, b = step([900, 130], [1, 1], g)
    kv, cache = random_cache(pages, 1, 128, g)
    kv, q = kv.cuda(), torch.randn((2, 96, 128), generator=g).to(BF16).cuda()
    early = types.SimpleNamespace(**{**vars(b), "starts": [3, 0], "start": ints([3, 0])})
    o.attention_kv4(q, kv, early, 0.1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = o.attention_kv4(q, kv, early, 0.1)
        early.start.copy_(b.start)
        graph.replay()
    torch.cuda.synchronize()
    check_attention(q, out, cache, b, 0.1, 128)
    o.check_status()


def test_misfits_are_reported():
    """Pages outside the cache, places outside the page table, sequences longer than said: nothing outside the arrays is touched."""
    o = ops()
    g = torch.Generator().manual_seed(6)
    pages, b = step([100, 700], [1, 1], g)
    kv = random_cache(pages, 2, 64, g)[0].cuda()
    q = torch.randn((2, 4, 64), generator=g).to(BF16).cuda()
    x = torch.randn((2, 8 * 64), generator=g).to(BF16).cuda()

    def said():
        with pytest.raises(o.KernelError, match="4-bit cache"):
            o.check_status()
        o.check_status()
    good = o.attention_kv4(q, kv, b, 0.1)
    for bad in (-1, pages, 1 << 30):
        broken = types.SimpleNamespace(**vars(b))
        broken.page_table = b.page_table.clone()
        broken.page_table[0, 1] = bad
        for plain in (False, True):
            out = o.attention_kv4(q, kv, broken, 0.1, plain=plain)
            said()
            if not plain:
                assert torch.equal(out[1], good[1])
        before = kv.clone()
        o.qk_norm_rope_append_kv4(x, 4, 2, 64, q_weight=None, k_weight=None, eps=0.0, cos=None, sin=None, kv=kv, page_table=broken.page_table,
                                  seq_of_token=ints([0, 0]), positions=ints([70, 100]))
        said()
        assert torch.equal(kv, before)
        held = o.kv4_read(kv, 64, broken.page_table, ints([0, 0]), ints([70, 10]))
        said()
        assert (held[:, 0] == 0).all() and (held[:, 1] != 0).any()
    width = b.table_width
    for seq, pos in ((0, -1), (0, width * PAGE), (2, 5), (-1, 5)):
        before = kv.clone()
        o.qk_norm_rope_append_kv4(x[:1].contiguous(), 4, 2, 64, q_weight=None, k_weight=None, eps=0.0, cos=None, sin=None, kv=kv,
                                  page_table=b.page_table, seq_of_token=ints([seq]), positions=ints([pos]))
        said()
        assert torch.equal(kv, before)
        assert (o.kv4_read(kv, 64, b.page_table, ints([seq]), ints([pos])) == 0).all()
        said()
    for start in (-5, 64 * width + 3):
        broken = types.SimpleNamespace(**vars(b))
        broken.start = ints([start, 700])
        for plain in (False, True):
            out = torch.full_like(q, 7.0)
            o.attention_kv4(q, kv, broken, 0.1, out=out, plain=plain)
            said()
            assert (out[0] == 7.0).all() and (out[1] != 7.0).any()
    # many rows: opened pages; one page more than the host counted
    pages, b = step([0, 60], [40, 70], g, width=4)
    kv = random_cache(pages, 2, 64, g)[0].cuda()
    q = torch.randn((110, 4, 64), generator=g).to(BF16).cuda()
    b.start = ints([0, 130])
    o.attention_kv4(q, kv, b, 0.1)
    said()


def test_refusals():
    o = ops()
    g = torch.Generator().manual_seed(7)
    pages, b = step([100, 7], [1, 1], g)
    kv = random_cache(pages, 2, 64, g)[0].cuda()
    q = torch.randn((2, 4, 64), generator=g).to(BF16).cuda()
    x = torch.randn((2, 8 * 64), generator=g).to(BF16).cuda()
    base = dict(q_weight=None, k_weight=None, eps=0.0, cos=None, sin=None, kv=kv, page_table=b.page_table, seq_of_token=b.seq_of_token,
                positions=b.positions)
    w, half = torch.ones(64, device="cuda"), torch.ones((2, 32), device="cuda")
    for change in (dict(kv=kv[:, :1].contiguous()), dict(kv=kv.view(pages, -1)), dict(kv=kv.float()), dict(kv=kv.cpu()), dict(kv=None), dict(q_weight=w),
                   dict(cos=half), dict(sin=half), dict(cos=half.double(), sin=half), dict(cos=half[:1].contiguous(), sin=half),
                   dict(page_table=b.page_table.long()), dict(page_table=b.page_table[0]), dict(positions=b.positions[:1]),
                   dict(seq_of_token=b.seq_of_token.cpu()), dict(q_out=q.float()), dict(q_weight=w.half(), k_weight=w)):
        with pytest.raises(o.KernelError):
            o.qk_norm_rope_append_kv4(x, 4, 2, 64, **{**base, **change})
    for bad in (x.half(), x[:, :-1], x[:, ::2], x.float()[None], x.cpu()):
        with pytest.raises(o.KernelError):
            o.qk_norm_rope_append_kv4(bad, 4, 2, 64, **base)
    with pytest.raises(o.KernelError):
        o.qk_norm_rope_append_kv4(x.view(2, 16 * 32), 12, 2, 32, **base)           # (a head size that is not built)
    for bad in (q.half(), q[:, :3].contiguous(), q[:1], q[:, :, :32].contiguous(), q.transpose(0, 1), q.cpu(), q[0]):
        with pytest.raises(o.KernelError):
            o.attention_kv4(bad, kv, b, 0.1)
    for name, bad in (("cu_seqlens", b.cu_seqlens[:-1]), ("start", b.start.long()), ("page_table", b.page_table[:, :1]), ("kv_bound", 10 ** 6),
                      ("seq_of_token", b.seq_of_token[:1])):
        broken = types.SimpleNamespace(**{**vars(b), name: bad})
        with pytest.raises(o.KernelError):
            o.attention_kv4(q, kv, broken, 0.1)
    for name in ("kv_bound", "max_q_len"):
        with pytest.raises(o.KernelError):
            o.attention_kv4(q, kv, types.SimpleNamespace(**{**vars(b), name: 0}), 0.1)
    with pytest.raises(o.KernelError):
        o.attention_kv4(q, kv, b, 0.1, out=q.float())
    for bad in (q, q.float()):
        with pytest.raises(o.KernelError):
            o.attention_kv4(bad, kv, b, 0.1, kind="other" if bad is q else "stay")
    long_pages, long = step([700, 7], [1, 1], g)
    kv2 = random_cache(long_pages, 2, 64, g)[0].cuda()
    with pytest.raises(o.KernelError):
        o.attention_kv4(q, kv2, long, 0.1, torch.empty(3, device="cuda"), kind="records")
    for bad in (kv[:, :, 1:], kv.view(pages, -1), kv.cpu()):
        with pytest.raises(o.KernelError):
            o.kv4_read(bad, 64, b.page_table, b.seq_of_token, b.positions)
    o.check_status()
