"""The cache in 4 bits on the device: descriptions that do not fit, numbers at the ends of their ranges, steps of many tokens."""
import math
import types

import pytest
import torch

from plain import kv4_plain as P
from test_gpu_kv4 import BF16, F32, PAGE, check_attention, ints, ops, random_cache, step

pytestmark = pytest.mark.gpu


def said():
    with pytest.raises(ops().KernelError, match="4-bit cache"):
        ops().check_status()
    ops().check_status()


@pytest.mark.parametrize("kind", ["plain", "records", "clusters", "stay"])
@pytest.mark.parametrize("start", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 64, 2 ** 31 - 200, 2 ** 30])
def test_a_start_near_the_end_of_32_bits(start, kind):
    """The sequence's length is beyond 32 bits: it is left out and reported, the others are what they were."""
    o = ops()
    g = torch.Generator().manual_seed(11)
    pages, b = step([100, 70, 400, 3], [2, 1, 2, 2], g)
    kv = random_cache(pages, 2, 64, g)[0].cuda()
    q = torch.randn((7, 4, 64), generator=g).to(BF16).cuda()
    good = o.attention_kv4(q, kv, b, 0.1, kind=kind)
    o.check_status()
    for i in (0, 2, 3):
        broken = types.SimpleNamespace(**vars(b))
        broken.start = b.start.clone()
        broken.start[i] = start
        out = torch.full_like(q, 7.0)
        o.attention_kv4(q, kv, broken, 0.1, out=out, kind=kind)
        said()
        mine = torch.tensor([x == i for x in b.seq_of_token.tolist()], device="cuda")
        assert (out[mine] == 7.0).all() and torch.equal(out[~mine], good[~mine])


@pytest.mark.parametrize("kind", ["plain", "records", "stay"])
def test_tokens_beyond_the_step(kind):
    """A sequence whose tokens lie outside the step's is left out and reported."""
    o = ops()
    g = torch.Generator().manual_seed(12)
    pages, b = step([100, 70], [2, 1], g)
    kv = random_cache(pages, 2, 64, g)[0].cuda()
    q = torch.randn((3, 4, 64), generator=g).to(BF16).cuda()
    good = o.attention_kv4(q, kv, b, 0.1, kind=kind)
    for cu in ([0, 2, 4], [-1, 0, 1], [2 ** 31 - 2, 2 ** 31 - 1, 3], [0, 2 ** 31 - 1, -2 ** 31]):
        broken = types.SimpleNamespace(**vars(b))
        broken.cu_seqlens = ints(cu)
        out = torch.full_like(q, 7.0)
        o.attention_kv4(q, kv, broken, 0.1, out=out, kind=kind)
        said()
        if cu[:2] == [0, 2]:
            assert torch.equal(out[:2], good[:2]) and (out[2] == 7.0).all()
        elif cu[0] != -1:
            assert (out == 7.0).all()


@pytest.mark.parametrize("width", [None, 9])
def test_opened_pages_have_a_name_in_every_place(width):
    """Whatever the scratch held: behind a sequence's last page, for sequences without a page, and with more room than pages."""
    from wick_b200.layout import pages_for
    o = ops()
    g = torch.Generator().manual_seed(13)
    for starts, new in (([0, 100, 300], [65, 64, 5]), ([64], [129]), ([0, 0, 7], [70, 0, 3])):
        pages, b = step(starts, new, g, width=width)
        kv, cache = random_cache(pages, 2, 64, g)
        q = torch.randn((b.n_tokens, 4, 64), generator=g).to(BF16).cuda()
        words = o.attention_kv4_scratch(b, 4, 2, 64, BF16, kind="opened")
        want = None
        for junk in (0, -1, 0x7FFFFFFF, 123456789):
            scratch = torch.full((words + 3,), junk, dtype=torch.int32, device="cuda").view(F32)
            out = o.attention_kv4(q, kv.cuda(), b, 0.1, scratch, kind="opened")
            used = [pages_for(s + n) for s, n in zip(starts, new)]
            at = sum(used) * 2 * PAGE * 64
            names = scratch.view(torch.int32)[at:at + b.n_seqs * b.table_width].view(b.n_seqs, -1).tolist()
            first = 0
            for row, n in zip(names, used):
                assert row == [first + i for i in range(n)] + [0] * (b.table_width - n)
                first += n
            assert (scratch.view(torch.int32)[words:] == junk).all()
            want = out if want is None else want
            assert torch.equal(out, want)
        check_attention(q, want, cache, b, 0.1, 64)
    o.check_status()


@pytest.mark.parametrize("start", [-5, -2 ** 31, 5 * PAGE - 64, 64 * PAGE, 2 ** 30, 2 ** 31 - 1, 2 ** 31 - 65, 2 ** 31 - 130])
def test_opened_pages_of_a_sequence_that_does_not_fit(start):
    """It is reported, the others are what they were."""
    o = ops()
    g = torch.Generator().manual_seed(14)
    pages, b = step([100, 0, 64], [65, 129, 70], g, width=5)
    kv = random_cache(pages, 2, 64, g)[0].cuda()
    q = torch.randn((b.n_tokens, 4, 64), generator=g).to(BF16).cuda()
    good = o.attention_kv4(q, kv, b, 0.1, kind="opened")
    o.check_status()
    for i in range(3):
        broken = types.SimpleNamespace(**vars(b))
        broken.start = b.start.clone()
        broken.start[i] = start
        out = o.attention_kv4(q, kv, broken, 0.1, kind="opened")
        said()
        others = torch.tensor([x != i for x in b.seq_of_token.tolist()], device="cuda")
        assert torch.equal(out[others], good[others]), i


def test_opened_pages_of_tokens_in_no_order():
    """Tokens outside the step, or sequences whose tokens go backwards: reported, and nothing outside the arrays is written."""
    o = ops()
    g = torch.Generator().manual_seed(15)
    pages, b = step([100, 0, 64], [65, 129, 70], g)
    kv = random_cache(pages, 2, 64, g)[0].cuda()
    q = torch.randn((b.n_tokens, 4, 64), generator=g).to(BF16).cuda()
    good = o.attention_kv4(q, kv, b, 0.1, kind="opened")
    n = b.n_tokens
    for cu in ([0, 65, 194, n + 1], [0, 65, 194, 2 ** 31 - 1], [0, 65, 194, -2 ** 31], [-1, 65, 194, n], [2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1, 3], [0, 200, 100, n]):
        broken = types.SimpleNamespace(**vars(b))
        broken.cu_seqlens = ints(cu)
        around = torch.full((n + 200, 4, 64), 7.0, dtype=BF16, device="cuda")
        o.attention_kv4(q, kv, broken, 0.1, out=around[100:100 + n], kind="opened")
        said()
        assert (around[:100] == 7.0).all() and (around[100 + n:] == 7.0).all()
        if cu[:3] == [0, 65, 194]:
            assert torch.equal(around[100:294], good[:194])


def test_opened_rows_behind_the_last_sequence_stay():
    o = ops()
    g = torch.Generator().manual_seed(16)
    pages, b = step([100, 7], [65, 100], g)
    kv = random_cache(pages, 2, 64, g)[0].cuda()
    q = torch.randn((170, 4, 64), generator=g).to(BF16).cuda()
    want = o.attention_kv4(q[:165].clone(), kv, b, 0.1, kind="opened")
    b.n_tokens, b.seq_of_token = 170, ints(b.seq_of_token.tolist() + [1] * 5)
    out = torch.full_like(q, 7.0)
    o.attention_kv4(q, kv, b, 0.1, out=out, kind="opened")
    assert (out[165:] == 7.0).all() and torch.equal(out[:165], want)
    o.check_status()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("scale", [-0.07, -0.4, 0.0, -0.0, 1e-60, -1e-60])
def test_opened_pages_and_scales(scale, d):
    """A negative scale turns the order of the scores around, one of 0 (as a float32, too) weighs all alike; the form that the rule takes, and by hand."""
    o = ops()
    g = torch.Generator().manual_seed(17)
    pages, b = step([0, 100, 70], [150, 33, 1], g)
    kv, cache = random_cache(pages, 2, d, g)
    q = torch.randn((b.n_tokens, 4, d), generator=g).to(BF16).cuda()
    for kind in ("opened", None):
        check_attention(q, o.attention_kv4(q, kv.cuda(), b, scale, kind=kind), cache, b, scale, d)
    # a key that is no number shows in the rows that see it, with any scale
    scales = kv[:, :, 64 * d:].view(pages, 2, 2, PAGE, d // 32, 4)
    scales[b.table[1][132 // PAGE], 1, 0, 132 % PAGE, 0] = torch.tensor([0.0, math.nan], dtype=BF16).view(torch.uint8)
    want = torch.zeros(q.shape, dtype=torch.bool, device="cuda")
    want[182, 2:] = True
    assert torch.equal(o.attention_kv4(q, kv.cuda(), b, scale, kind="opened").isnan(), want)
    o.check_status()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("starts,new", [([100, 60], [40, 90]), ([0, 64], [300, 65]), ([63], [2])])
def test_opened_values_that_are_no_numbers(starts, new, d):
    """A value that is no number shows in the rows of the tokens that see it, and in no others: in its channels where all of the step's tokens see
    it, else in all of its head's.  Behind a sequence's end and in other pages nothing shows."""
    o = ops()
    g = torch.Generator().manual_seed(d + new[0])
    pages, b = step(starts, new, g, spare=2)
    kv, cache = random_cache(pages, 2, d, g)
    q = torch.randn((b.n_tokens, 4, d), generator=g).to(BF16).cuda()
    nan = torch.tensor([0.0, math.nan], dtype=BF16).view(torch.uint8)
    used = {b.table[i][p]: (i, p) for i in range(len(new)) for p in range(-(-(starts[i] + new[i]) // PAGE))}
    clean = o.attention_kv4(q, kv.cuda(), b, 0.1, kind="opened")
    scales = kv[:, :, 64 * d:].view(pages, 2, 2, PAGE, d // 32, 4)
    for p in range(pages):
        end = starts[used[p][0]] + new[used[p][0]] - used[p][1] * PAGE if p in used else 0
        scales[p, :, :, max(0, min(PAGE, end)):] = nan
    assert torch.equal(o.attention_kv4(q, kv.cuda(), b, 0.1, kind="opened"), clean)
    for i in range(len(new)):
        for pos in {0, starts[i], starts[i] + 1, starts[i] + new[i] // 2, starts[i] + new[i] - 1}:
            one = kv.clone()
            at = one[:, :, 64 * d:].view(scales.shape)
            at[b.table[i][pos // PAGE], 1, 1, pos % PAGE, 1] = nan          # (the second key head, channels 32 to 63)
            first = max(0, pos - starts[i]) + sum(new[:i])
            want = torch.zeros(q.shape, dtype=torch.bool, device="cuda")
            if pos <= starts[i]:
                want[first:sum(new[:i + 1]), 2:, 32:64] = True
            else:
                want[first:sum(new[:i + 1]), 2:] = True
            for scale in (0.1, -0.1):
                out = o.attention_kv4(q, one.cuda(), b, scale, kind="opened")
                assert torch.equal(out.isnan(), want), (i, pos)
                if scale > 0:
                    assert torch.equal(out[~want], clean[~want])
    o.check_status()


# ---- append: numbers at the ends of their ranges, and steps of many tokens -------------
MANY = 300                                                           # tokens, of which a step's keys and values are looked at in 32 bits first


def append_rows(k, v, splits=1, w=None, eps=0.0):
    """Keys and values float32 [splits, n, d] of n tokens, one head each, into a cache of their own: its bytes, and what it holds (float64 [2, n, d])."""
    o = ops()
    n, d = k.shape[1:]
    pages = -(-n // PAGE)
    at = types.SimpleNamespace(page_table=ints([list(range(1, pages + 1))]), seq_of_token=ints([0] * n), positions=ints(list(range(n))))
    kv = torch.zeros((pages + 1, 1, 80 * d), dtype=torch.uint8, device="cuda")
    x = torch.cat([torch.zeros_like(k), k, v], 2).cuda().contiguous()
    o.qk_norm_rope_append_kv4(x, 1, 1, d, q_weight=w, k_weight=w, eps=eps, cos=None, sin=None, kv=kv, dtype=F32, **vars(at))
    held = o.kv4_read(kv, d, at.page_table, at.seq_of_token, at.positions).double().cpu()[:, :, 0]
    o.check_status()
    return kv.cpu(), held


@pytest.mark.parametrize("many", [False, True])
def test_append_of_ranges_that_bfloat16_cannot_hold(many):
    """32 finite numbers below 2^127 whose b is beyond bfloat16's range are stored as numbers that are none; somewhat smaller ones as ever."""
    d = 64
    n = MANY if many else 6
    x = torch.randn((2, n, d), generator=torch.Generator().manual_seed(21)).double()
    edges = ((0, -1.2e38, 1.2e38, True), (1, -1.0e38, 1.0e38, False), (2, -1.6e38, 0.2e38, True), (3, 0.0, 1.6e38, False), (4, -1.65e38, -1.6e38, False),
             (5, -1.1e38, 1.09e38, True))
    for i in range(2):
        for row, low, high, _ in edges:
            x[i, row, 32 * i:32 * i + 32] = torch.linspace(0, 1, 32).double() * (high - low) + low
    x = x.float()
    _, held = append_rows(x[:1], x[1:])
    for i in range(2):
        for row, low, high, beyond in edges:
            a = ((torch.tensor(high).float().double() - torch.tensor(low).float().double()) * (16 / 15)).to(BF16).double()
            b = (torch.tensor(low).float().double() - a).to(BF16)
            assert a.isfinite() and b.isfinite().item() != beyond, row   # (the table is right)
            part, rest = held[i, row, 32 * i:32 * i + 32], held[i, row, 32 - 32 * i:64 - 32 * i]
            assert part.isnan().all() if beyond else part.isfinite().all(), (i, row)
            assert rest.isfinite().all()
            if not beyond:
                assert torch.equal(part, P.decode(*P.encode(x[i, row:row + 1, 32 * i:32 * i + 32].double()))[0])


@pytest.mark.parametrize("heads,n_kv,d", [(4, 2, 64), (6, 2, 128), (5, 1, 192), (4, 2, 256)])
@pytest.mark.parametrize("splits,dtype,norm,turn", [(0, BF16, True, True), (3, BF16, True, True), (1, F32, True, False), (8, BF16, False, True), (2, F32, False, False),
                                                    (0, BF16, False, False), (0, F32, False, True), (0, F32, True, True)])
def test_append_of_many_tokens(heads, n_kv, d, splits, dtype, norm, turn):
    """Steps of more than 256 tokens look at keys and values in 32 bits first: the codes are those of 64 bits, and the same bytes as in smaller steps."""
    o = ops()
    g = torch.Generator().manual_seed(heads * d + splits)
    starts, new = [0, 61, 5], [300, 3, 1]
    pages, b = step(starts, new, g, spare=2)
    n = b.n_tokens
    x = torch.randn((max(splits, 1), n, (heads + 2 * n_kv) * d), generator=g) * 2
    x[:, 40:60] *= 100.0                                             # (tokens of other sizes)
    x[:, 60:80] *= 0.01
    x = x if splits else x[0].to(dtype)
    w = (torch.rand(d, generator=g) + 0.5) if norm else None
    angle = b.positions.cpu().double()[:, None] * 1e4 ** (-torch.arange(d // 2).double() / (d // 2))
    cos, sin = (angle.cos().float(), angle.sin().float()) if turn else (None, None)
    up = lambda v: None if v is None else v.cuda()      # noqa: E731

    def run(kv, first, last):
        part = x[:, first:last] if splits else x[first:last]
        return o.qk_norm_rope_append_kv4(part.contiguous().cuda(), heads, n_kv, d, q_weight=up(w), k_weight=up(w), eps=1e-6,
                                         cos=None if cos is None else cos[first:last].contiguous().cuda(),
                                         sin=None if sin is None else sin[first:last].contiguous().cuda(), kv=kv, page_table=b.page_table,
                                         seq_of_token=b.seq_of_token[first:last].contiguous(), positions=b.positions[first:last].contiguous(), dtype=dtype)
    kv = torch.full((pages, n_kv, 80 * d), 0x5A, dtype=torch.uint8, device="cuda")
    pieces = kv.clone()
    q = run(kv, 0, n)
    assert torch.equal(q, torch.cat([run(pieces, 0, 100), run(pieces, 100, 290), run(pieces, 290, n)]))
    assert torch.equal(kv, pieces)
    eps = torch.tensor(1e-6, dtype=F32).double().item()
    _, k, v = P.project(x.double().sum(0) if splits else x.double(), heads, n_kv, d, w, w, eps, cos, sin)
    held = o.kv4_read(kv, d, b.page_table, b.seq_of_token, b.positions).double().cpu()
    assert torch.equal(held[0], P.decode(*P.encode(k))) and torch.equal(held[1], P.decode(*P.encode(v)))
    o.check_status()


def test_append_of_many_odd_numbers():
    """Numbers on borders between codes, equal ones, runs that cancel, numbers that are none, in a step of many tokens."""
    d = 64
    g = torch.Generator().manual_seed(22)
    x = torch.randn((2, 3, MANY, d), generator=g)
    x[:, 1:] = 0
    whole = torch.arange(d).float()
    x[:, 0, 0], x[:, 0, 1], x[:, 0, 2] = 0.0, 3.140625, whole
    x[:, 0, 3] = 1.0 + whole / 4096
    x[:, 0, 4] = torch.where(whole % 2 == 0, 0.0, 15.0)
    x[:, 0, 4, 1::4] = torch.arange(16).float() % 15 + 0.5
    x[0, 0, 5, 5], x[1, 0, 6, 40], x[0, 0, 7, 33] = math.inf, math.nan, -math.inf
    x[:, 0, 8] *= 1e-38
    x[:, 0, 9] *= 1e37
    x[:, 0, 10:40] = torch.randint(-8, 8, (2, 30, d), generator=g).float()            # (few bits: halves between two codes)
    x[:, 0, 40:70] = (x[:, 0, 40:70] * 16).round() / 16
    x[:, 1, 100:150] = 1e4 * torch.randn((2, 50, d), generator=g)                     # (runs that cancel)
    x[:, 2, 100:150] = -x[:, 1, 100:150]
    x[:, 1, 150:200] = 3e6 * torch.randn((2, 50, d), generator=g)
    x[:, 2, 150:200] = -x[:, 1, 150:200]
    x[:, 0, 200:250] += 1e3                                                           # (a range far from zero)
    for splits in (1, 3):
        k, v = x[0, :splits], x[1, :splits]
        _, held = append_rows(k, v)
        for i, y in enumerate((k, v)):
            want = P.decode(*P.encode(y.double().sum(0)))
            assert torch.equal(held[i].isnan(), want.isnan()) and torch.equal(held[i].nan_to_num(7.0), want.nan_to_num(7.0)), (splits, i)


@pytest.mark.parametrize("size,weight,eps", [(1e-18, 1.0, 0.0), (1e-20, 1.0, 0.0), (3e-22, 1.0, 0.0), (1e-24, 1e3, 0.0), (1e-19, 1.0, 1e-38), (1e-38, 1e12, 1e-6),
                                             (1.0, 1e20, 1e-6), (1e15, 1.0, 1e-6), (1e19, 1e-3, 1e-6), (3e19, 1.0, 1e-6)])
def test_append_of_many_norms_at_the_ends_of_the_range(size, weight, eps):
    """Mean squares below the smallest normal 32-bit number (and above the largest) are as good as others."""
    d = 64
    g = torch.Generator().manual_seed(23)
    k = torch.randn((1, MANY, d), generator=g) * size
    k[:, :, 32:40] *= 1e-4                                           # (some numbers much smaller than their row's size)
    k[:, 100:, 32:] *= torch.exp2(-torch.arange(MANY - 100).float())[:, None]         # (... and whole groups)
    w = (torch.rand(d, generator=g) + 0.5) * weight
    _, held = append_rows(k, torch.zeros_like(k), w=w.cuda(), eps=eps)
    y = k[0].double()
    y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + torch.tensor(eps, dtype=F32).double()) * w.double()
    codes, a, b = P.encode(y)
    # (scales below the smallest normal number are not held to be kept, see the test of odd numbers)
    fine = (a >= 2.0 ** -126).repeat_interleave(32, -1)
    assert torch.equal(held[0][fine], P.decode(codes, a, b)[fine])
    assert fine[:100].all() or weight * size < 1e-20


# ---- attention: other devices, and no cache at all ----------------------------------------
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="one device")
def test_on_a_second_device():
    """Kernels with more shared memory than a device gives unasked, on the first device and then on another."""
    o = ops()
    g = torch.Generator().manual_seed(24)
    pages, b = step([900, 70, 3000], [2, 3, 1], g)
    kv, cache = random_cache(pages, 2, 128, g)
    q = torch.randn((6, 8, 128), generator=g).to(BF16)
    for device in ("cuda:0", "cuda:1"):
        with torch.cuda.device(device):
            there = types.SimpleNamespace(**{k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in vars(b).items()})
            for kind in ("records", "clusters", "stay", "opened"):
                check_attention(q, o.attention_kv4(q.to(device), kv.to(device), there, 0.1, kind=kind), cache, b, 0.1, 128)
            o.check_status()


def test_a_cache_without_pages():
    """There is nothing that a page outside it could be read as: refused, whatever the form; appending to it and reading from it is reported."""
    o = ops()
    for new in ([1, 1], [100, 3]):
        _, b = step([5, 0], new, torch.Generator().manual_seed(25))
        kv = torch.zeros((0, 2, 80 * 64), dtype=torch.uint8, device="cuda")
        for dtype, kinds in ((BF16, (None, "plain", "records", "stay", "opened")), (F32, (None, "plain"))):
            q = torch.zeros((b.n_tokens, 4, 64), dtype=dtype, device="cuda")
            for kind in kinds:
                with pytest.raises(o.KernelError, match="without pages"):
                    o.attention_kv4(q, kv, b, 0.1, kind=kind)
        o.check_status()
        o.qk_norm_rope_append_kv4(torch.zeros((b.n_tokens, 8 * 64), device="cuda"), 4, 2, 64, q_weight=None, k_weight=None, eps=0.0, cos=None, sin=None, kv=kv,
                                  page_table=b.page_table, seq_of_token=b.seq_of_token, positions=b.positions)
        said()
        assert (o.kv4_read(kv, 64, b.page_table, b.seq_of_token, b.positions) == 0).all()
        said()


@pytest.mark.parametrize("new,heads,d,dtype,kinds", [(130, 16, 256, BF16, (None, "records", "stay", "clusters")), (500, 16, 256, BF16, (None, "records", "stay", "clusters")),
                                                     (61, 17, 64, F32, (None,)), (2000, 17, 64, F32, (None,))])
def test_fewer_pieces_for_bounded_records(new, heads, d, dtype, kinds):
    """So many rows behind so long a cache that its length alone would cut it into records of more than 256 MB; beside a short sequence."""
    o = ops()
    g = torch.Generator().manual_seed(new)
    starts = [65600, 100]
    pages, b = step(starts, [new, 3], g)
    kv, cache = random_cache(pages, 1, d, g)
    n = b.n_tokens
    q = torch.randn((n, heads, d), generator=g).to(dtype).cuda()
    scale = 1.0 / math.sqrt(d)
    some = [0, 1, new // 2, new - 1]
    for kind in kinds:
        words = None
        try:
            words = o.attention_kv4_scratch(b, heads, 1, d, dtype, kind=kind)
        except o.KernelError:
            assert kind == "clusters"
            continue
        assert 4 * words <= 256 << 20
        scratch = torch.full((words + 100,), math.nan, device="cuda")
        out = o.attention_kv4(q, kv.cuda(), b, scale, scratch, kind=kind)
        assert scratch[words:].isnan().all()
        for t in some:
            one = types.SimpleNamespace(q_lens=[1], starts=[starts[0] + t], table=[b.table[0]])
            check_attention(q[t:t + 1], out[t:t + 1], cache, one, scale, d)
        check_attention(q[new:], out[new:], cache, types.SimpleNamespace(q_lens=[3], starts=[100], table=[b.table[1]]), scale, d)
    o.check_status()


def test_captured_decode_steps_do_not_keep_a_prompt_s_scratch():
    import gc
    import weakref

    from helpers import CONFIGS, random_tokens
    from test_gpu_kv4_engine import engine
    eng = engine("D", "bfloat16", max_tokens=16384)
    vocab = CONFIGS["D"]["vocab_size"]

    def run(n):
        s = eng.open_seq()
        toks = random_tokens(vocab, n + 3, n)
        eng.step([s], [toks[:n]], [[n - 1]])
        out = [eng.step([s], [[t]], [[0]]).clone() for t in toks[n:]]
        eng.close_seq(s)
        return out
    first = run(900)
    large = weakref.ref(eng.workspace.buffers["attention_kv4_prompt"])
    assert eng._graphs and all("attention_kv4_prompt" not in g.keepalive for g in eng._graphs.values())
    run(2000)                                                        # (a larger one takes its place)
    gc.collect()
    assert large() is None
    assert all(torch.equal(x, y) for x, y in zip(run(900), first))
    eng.check_kernels()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["D", "E"])
def test_logits_of_prompts_of_many_tokens(name, dtype):
    """Prompts whose steps decide codes in 32 bits first, alone, behind what is cached, and several together."""
    from helpers import CONFIGS, random_tokens
    from test_gpu_kv4_engine import check, engine
    eng = engine(name, dtype, max_tokens=4096)
    vocab = CONFIGS[name]["vocab_size"]
    toks = random_tokens(vocab, 640, 31)
    s = eng.open_seq()
    got = [eng.step([s], [toks[:300]], [[0, 150, 299]]).clone(), eng.step([s], [toks[300:]], [[0, 70, 339]]).clone()]
    check(eng, s, toks, torch.cat(got), [0, 150, 299, 300, 370, 639], name, dtype, (name, "alone"))
    eng.close_seq(s)
    lens = (280, 7, 129)
    toks = [random_tokens(vocab, n, 40 + n) for n in lens]
    slots = [eng.open_seq() for _ in lens]
    got = eng.step(slots, toks, [[0, n - 1] for n in lens]).clone()
    for b, n in enumerate(lens):
        check(eng, slots[b], toks[b], got[2 * b:2 * b + 2], [0, n - 1], name, dtype, (name, n, "together"))
    eng.check_kernels()


def test_opened_pages_of_one_step_behind_another():
    """Two steps of other lengths take turns over one scratch, with no other kernel in between: each finds its own description there."""
    o = ops()
    g = torch.Generator().manual_seed(26)
    d, KV, H = 128, 2, 8
    steps = []
    for starts, new in (([0, 500], [300, 100]), ([540, 10], [100, 300])):
        pages, b = step(starts, new, g, width=10)
        kv, cache = random_cache(pages, KV, d, g)
        q = torch.randn((b.n_tokens, H, d), generator=g).to(BF16).cuda()
        steps.append((q, kv.cuda(), b, cache))
    words = {o.attention_kv4_scratch(b, H, KV, d, BF16, kind="opened") for _, _, b, _ in steps}
    assert len(words) == 1                                           # (the descriptions lie in the same places)
    scratch = torch.empty(words.pop(), dtype=F32, device="cuda")
    want = []
    for q, kv, b, cache in steps:
        want.append(o.attention_kv4(q, kv, b, 0.1, scratch, kind="opened"))
        torch.cuda.synchronize()
        check_attention(q, want[-1], cache, b, 0.1, d)
    outs = [[torch.empty_like(q) for q, *_ in steps] for _ in range(50)]

    def run():
        for pair in outs:
            for (q, kv, b, _), out in zip(steps, pair):
                o.attention_kv4(q, kv, b, 0.1, scratch, out=out, kind="opened")
    run()
    assert all(torch.equal(out, w) for pair in outs for out, w in zip(pair, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for _ in range(20):
        for pair in outs:
            for out in pair:
                out.fill_(7.0)
        graph.replay()
        assert all(torch.equal(out, w) for pair in outs for out, w in zip(pair, want))
    o.check_status()
