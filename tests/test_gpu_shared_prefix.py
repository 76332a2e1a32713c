"""Attention over a shared prefix, tables built on the device, histories and steering of logits, each against a plain implementation in
64 bits at the sizes and masks where it can go wrong, and their refusals."""
import math
import types

import pytest
import torch

pytestmark = pytest.mark.gpu

PAGE = 64
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from wick_b200 import ops
    return ops


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def pages_for(n):
    return -(-n // PAGE)


class Case:
    """groups: a list of (shared pages, [(own cached positions, new tokens), ...]).  Page ids are dealt at random; places that no sequence
    has written hold NaN."""

    def __init__(self, groups, heads, kv_heads, dim, dtype, seed=0, more_width=0, sharp=2.0):
        g = torch.Generator().manual_seed(seed)
        self.heads, self.kv_heads, self.dim, self.dtype = heads, kv_heads, dim, dtype
        self.sizes, self.shared = [len(s) for _, s in groups], [p for p, _ in groups]
        group_of = [i for i, n in enumerate(self.sizes) for _ in range(n)]
        self.starts = [PAGE * p + own for p, s in groups for own, _ in s]
        self.q_lens = [q for _, s in groups for _, q in s]
        self.kv_lens = [s + q for s, q in zip(self.starts, self.q_lens)]
        need = sum(self.shared) + sum(max(pages_for(k) - self.shared[i], 0) for k, i in zip(self.kv_lens, group_of))
        ids = (torch.randperm(need, generator=g) + 1).tolist()
        prefix = [[ids.pop() for _ in range(p)] for p in self.shared]
        self.width = max(max(pages_for(k) for k in self.kv_lens), 1) + more_width
        self.tables = []
        kv = torch.randn((need + 1, 2, kv_heads, PAGE, dim), generator=g).to(dtype)
        used = torch.zeros((need + 1, PAGE), dtype=torch.bool)
        for k, i in zip(self.kv_lens, group_of):
            t = prefix[i] + [ids.pop() for _ in range(max(pages_for(k) - self.shared[i], 0))]
            for j, p in enumerate(t):
                used[p, :max(0, min(PAGE, k - j * PAGE)) if j >= self.shared[i] else PAGE] = True
            self.tables.append(t)
        kv[~used[:, None, None, :].expand(-1, 2, kv_heads, -1)] = math.nan
        n = sum(self.q_lens)
        self.q = (torch.randn((n, heads, dim), generator=g) * torch.linspace(0.3, sharp, heads)[:, None]).to(dtype)
        self.kv = kv
        self.scale = 1.0 / math.sqrt(dim)
        self.group_of = group_of

    def batch(self):
        cu = [sum(self.q_lens[:i]) for i in range(len(self.q_lens) + 1)]
        table = torch.zeros((len(self.tables), self.width), dtype=torch.int32)
        for b, t in enumerate(self.tables):
            table[b, :len(t)] = torch.tensor(t, dtype=torch.int32)
        seq = [b for b, q in enumerate(self.q_lens) for _ in range(q)]
        return types.SimpleNamespace(
            n_seqs=len(self.q_lens), n_tokens=cu[-1], table_width=self.width, max_q_len=max(self.q_lens), cu_seqlens=ints(cu), start=ints(self.starts),
            kv_len=ints(self.kv_lens), page_table=table.cuda(), seq_of_token=ints(seq), max_kv_len=max(self.kv_lens),
            positions=ints([self.starts[b] + i for b, q in enumerate(self.q_lens) for i in range(q)]))

    def want(self):
        """The result in 64 bits and how far a float32 computation (and, for bfloat16, weights rounded to it) may be off: see below."""
        out, most, t = [], [], 0
        for start, q_len, table in zip(self.starts, self.q_lens, self.tables):
            end = start + q_len
            if q_len == 0:
                continue
            kv = self.kv[torch.tensor(table)].double().permute(1, 2, 0, 3, 4).reshape(2, self.kv_heads, -1, self.dim)[:, :, :end]
            q = self.q[t:t + q_len].double().view(q_len, self.kv_heads, -1, self.dim)
            s = torch.einsum("nkgd,kld->nkgl", q, kv[0]) * self.scale
            # a product of d terms summed in 32 bits is off by at most (d + 2) 2^-24 of the sum of their sizes
            size = torch.einsum("nkgd,kld->nkgl", q.abs(), kv[0].abs()) * self.scale
            hidden = torch.arange(end) > (start + torch.arange(q_len))[:, None]
            s = s.masked_fill(hidden[:, None, None], -math.inf)
            p = torch.softmax(s, -1)
            y = torch.einsum("nkgl,kld->nkgd", p, kv[1])
            spread = torch.einsum("nkgl,kld->nkgd", p, kv[1].abs())
            off_s = (size * (self.dim + 2) * 2.0 ** -24 + size * 2.0 ** -22).masked_fill(hidden[:, None, None], 0).amax(-1, keepdim=True)
            # weights: twice the scores' error (theirs and the sum's), the exponential's 2^-21, the sums' (end + 8) 2^-24; then
            # bfloat16: weights and the result rounded, 2^-9 each, and their sum may be taken of either
            rel = 2 * off_s + 2.0 ** -21 + (end + 8) * 2.0 ** -23
            if self.dtype == BF16:
                rel = rel + 3 * 2.0 ** -9
            out.append(y.reshape(q_len, self.heads, self.dim))
            most.append((spread * rel + 1e-30).reshape(q_len, self.heads, self.dim))
            t += q_len
        return torch.cat(out), torch.cat(most)

    def run(self, ops, **kw):
        b = self.batch()
        shared = ops.SharedPrefix.of(self.sizes, self.shared, [max(k, PAGE * self.shared[g] + 1) for k, g in zip(self.kv_lens, self.group_of)], "cuda")
        return ops.attention_shared(self.q.cuda(), self.kv.cuda(), b, shared, self.scale, **kw)


def check(got, case):
    want, most = case.want()
    assert got.dtype == case.dtype and bool(torch.isfinite(got).all())
    over = ((got.double().cpu() - want).abs() / most).max().item()
    assert over <= 1.0, f"an element is off by {over:.3f} times what rounding allows"


ONE = [(1, 1)]
SHAPES = {
    # a prefix of one page; own keys from none (the new token opens a page) to whole pages
    "one_page": [(1, [(0, 1), (1, 1), (62, 1), (63, 1), (64, 1), (127, 1)])],
    # three pages (a unit that is half a pair of pages), one sequence alone
    "alone": [(3, [(17, 1)])],
    # nothing shared at all
    "nothing": [(0, [(0, 1), (5, 1), (200, 1)])],
    # groups of different sizes and prefixes, one empty, one without a prefix, a sequence that brings no token
    "groups": [(2, [(3, 1)] * 3), (0, [(70, 1), (0, 1)]), (5, [(1, 1), (9, 0), (130, 1), (64, 1), (7, 1)]), (1, []), (7, [(0, 1)] * 9)],
    # more rows than a tile, long own keys that are cut into parts, beside short ones
    "long_own": [(4, [(700, 1), (3, 1), (1300, 1), (511, 1), (512, 1)])],
    # several new tokens a sequence, some more than a tile holds
    "tokens": [(2, [(0, 3), (60, 7), (64, 1), (10, 41)]), (3, [(5, 2), (0, 64), (1, 17)])],
    # a prefix of many units
    "long_prefix": [(41, [(11, 1), (70, 1), (0, 1)])],
}


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 64), (8, 2, 128), (5, 1, 48), (20, 1, 16)])
@pytest.mark.parametrize("shape", sorted(SHAPES))
def test_attention_shared_is_the_attention_of_every_sequence_by_itself(ops, shape, heads, kv_heads, dim, dtype):
    case = Case(SHAPES[shape], heads, kv_heads, dim, dtype, seed=len(shape), more_width=3)
    check(case.run(ops), case)
    ops.check_status()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_attention_shared_with_many_rows(ops, dim, dtype):
    """More tokens than a tile of any form has rows, an odd number of them, heads that are no power of two."""
    case = Case([(9, [(i % 50, 1) for i in range(67)]), (2, [(3, 1)] * 30)], 12, 2, dim, dtype, seed=dim)
    check(case.run(ops), case)
    ops.check_status()


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_shared_of_256_heads_to_a_key_head(ops, dim):
    case = Case([(5, [(10, 1), (70, 1)])], 256, 1, dim, BF16, seed=3)
    check(case.run(ops), case)


def test_attention_shared_with_many_groups(ops):
    case = Case([(1 + i % 3, [(i % 7, 1)] * (1 + i % 2)) for i in range(90)], 4, 2, 64, BF16, seed=5)
    check(case.run(ops), case)
    ops.check_status()


def test_attention_shared_with_sharp_scores(ops):
    """Scores whose weights differ by more than 2^100: the prefix holds all the weight for some rows, none for others."""
    for dtype in (F32, BF16):
        case = Case([(6, [(30, 1), (100, 1), (600, 1)])], 8, 2, 128, dtype, seed=9, sharp=40.0)
        check(case.run(ops), case)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_shared_shows_infinities_and_nan(ops, dtype):
    """An infinite value is infinite for every row, a NaN among the queries shows in its own row only; places behind the last key (NaN
    everywhere in these tests) never do."""
    case = Case([(3, [(10, 1), (70, 1), (5, 1)])], 4, 2, 64, dtype, seed=2)
    page = case.tables[0][1]
    case.kv[page, 1, 0, 7, 5] = math.inf
    case.q[1, 3] = math.nan
    got = case.run(ops).float().cpu()
    assert bool((got[:, :2, 5] == math.inf).all()), "heads of key head 0 read it"
    assert bool(torch.isnan(got[1, 3]).all())
    got[:, :2, 5] = 0
    got[1, 3] = 0
    assert bool(torch.isfinite(got).all())


# Prefixes long enough for the kernel that computes them by themselves.
LONG = {
    # one tile of rows (both streams on it), an odd number of pages; one sequence brings nothing new
    "one_tile": ([(127, [(3, 1), (0, 1), (130, 1), (64, 0), (17, 1), (9, 1), (1, 1)])], 32, 8),
    # two tiles of rows, a stream each; heads that are no power of two, so that a tile has fewer than 128 rows
    "two_tiles": ([(70, [(i % 70, 1) for i in range(37)])], 12, 2),
    # three tiles: a pair and one by itself
    "three_tiles": ([(50, [(i * 13 % 200, 1) for i in range(41)])], 16, 2),
    # several tokens a sequence, groups of different lengths, one that shares nothing, an empty one
    "tokens": ([(33, [(5, 9), (70, 1), (0, 30)]), (0, [(40, 3)]), (19, []), (52, [(64, 17), (1, 1)])], 16, 4),
    # more items than thread blocks: some blocks have several runs, of one tile and of two
    "many_runs": ([(1 + i * 7 % 9, [(i % 5, 1)] * (1 + i * 11 % 4)) for i in range(60)] + [(7, [(2, 9)] * 5)], 64, 16),
    # one block of keys more than there are page numbers in a run of 32, two more
    "runs_of_32": ([(33, [(3, 1)] * 8), (34, [(3, 1)] * 8), (65, [(0, 1)] * 40)], 32, 4),
}


def kernels_of(ops, call):
    before = ops.launches[0]
    call()
    return ops.launches[0] - before


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("shape", sorted(LONG))
def test_attention_shared_behind_long_prefixes(ops, shape, dim):
    groups, heads, kv_heads = LONG[shape]
    if dim == 64:                                               # (the prefixes have to be twice as long there)
        groups = [(2 * p + (p > 0), s) for p, s in groups]
    case = Case(groups, heads, kv_heads, dim, BF16, seed=len(shape) + dim, more_width=1)
    assert kernels_of(ops, lambda: check(case.run(ops), case)) == 3
    ops.check_status()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", [5, 30])
@pytest.mark.parametrize("slope", [12.0, -12.0, 300.0])
def test_attention_shared_with_scores_that_rise(ops, slope, rows, dim):
    """Scores that rise, or fall, by a multiple of the slope from page to page, so that the maximum moves in every block, or never."""
    pages = 120 * 128 // dim
    case = Case([(pages, [(i % 40, 1) for i in range(rows)])], 32, 8, dim, BF16, seed=rows)
    u = torch.zeros(dim)
    u[::2] = 1.0
    case.q = (case.q.float() * 0.1 + 0.5 * u).to(BF16)
    for j, page in enumerate(case.tables[0][:pages]):
        case.kv[page, 0] = (case.kv[page, 0].float() + u * (slope * j / pages)).to(BF16)
    assert kernels_of(ops, lambda: check(case.run(ops), case)) == 3
    ops.check_status()


def test_attention_shared_behind_a_long_prefix_shows_infinities_and_nan(ops):
    case = Case([(110, [(10, 1), (70, 1), (5, 1), (9, 1)] * 4)], 16, 4, 128, BF16, seed=2)
    page = case.tables[0][37]
    case.kv[page, 1, 0, 7, 5] = math.inf
    case.q[1, 5] = math.nan
    got = case.run(ops).float().cpu()
    assert bool((got[:, :4, 5] == math.inf).all()), "heads of key head 0 read it"
    assert bool(torch.isnan(got[1, 5]).all())
    got[:, :4, 5] = 0
    got[1, 5] = 0
    assert bool(torch.isfinite(got).all())


def test_attention_shared_behind_a_long_prefix_same_bits_again(ops):
    groups, heads, kv_heads = LONG["tokens"]
    case = Case(groups, heads, kv_heads, 128, BF16, seed=4)
    a = case.run(ops)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = case.run(ops, out=torch.empty_like(a))
    s.synchronize()
    assert torch.equal(a, b)


@pytest.mark.parametrize("dim,dtype,kernels", [(64, BF16, 2), (128, BF16, 2), (48, BF16, 2), (128, F32, 2)])
def test_attention_shared_counts_its_kernels(ops, dim, dtype, kernels):
    case = Case([(2, [(10, 1), (70, 1)])], 4, 2, dim, dtype, seed=1)
    assert kernels_of(ops, lambda: case.run(ops)) == kernels


def test_attention_shared_same_bits_again_and_on_another_stream(ops):
    case = Case(SHAPES["groups"], 8, 2, 128, BF16, seed=4)
    a = case.run(ops)
    b = case.run(ops)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c = case.run(ops, out=torch.empty_like(a))
    s.synchronize()
    assert torch.equal(a, b) and torch.equal(a, c)


def test_attention_shared_in_a_graph_follows_the_description(ops):
    """A captured call reads lengths, groups and pages from the device: changed in place, the replay is that of the new description."""
    case = Case([(3, [(10, 1), (70, 1)]), (0, [(5, 1), (30, 1)])], 8, 2, 128, BF16, seed=6, more_width=2)
    b = case.batch()
    shared = ops.SharedPrefix.of(case.sizes, case.shared, case.kv_lens, "cuda")._replace(max_pages=4, own_bound=900)
    q, kv = case.q.cuda(), case.kv.cuda()
    scratch = torch.empty(ops.attention_shared_scratch(shared, b, 8, 2, 128, BF16), dtype=F32, device="cuda")
    out = torch.empty_like(q)
    ops.attention_shared(q, kv, b, shared, case.scale, scratch, out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.attention_shared(q, kv, b, shared, case.scale, scratch, out)
    g.replay()
    check(out, case)
    # one group shares less now, a sequence has become shorter
    shared.pages.copy_(ints([2, 0]))
    b.start.copy_(ints([case.starts[0], case.starts[1] - 60, 5, 30]))
    case.starts[1] -= 60
    g.replay()
    check(out, case)


def test_attention_shared_in_a_graph_behind_a_long_prefix(ops):
    """The same where the shared keys have a kernel of their own; twice in the graph, each beginning before the one before it has ended."""
    case = Case([(130, [(10, 1), (70, 1), (600, 1)] * 3), (3, [(5, 1)])], 32, 8, 128, BF16, seed=6, more_width=2)
    b = case.batch()
    shared = ops.SharedPrefix.of(case.sizes, case.shared, case.kv_lens, "cuda")._replace(max_pages=140, own_bound=900)
    q, kv = case.q.cuda(), case.kv.cuda()
    scratch = torch.empty(ops.attention_shared_scratch(shared, b, 32, 8, 128, BF16), dtype=F32, device="cuda")
    outs = [torch.empty_like(q), torch.empty_like(q)]
    ops.attention_shared(q, kv, b, shared, case.scale, scratch, outs[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for out in outs:
            assert kernels_of(ops, lambda: ops.attention_shared(q, kv, b, shared, case.scale, scratch, out)) == 3      # noqa: B023
    for out in outs:
        out.zero_()
    g.replay()
    for out in outs:
        check(out, case)
    # the group shares less now (its sequences hold the rest as their own), a sequence has become shorter
    shared.pages.copy_(ints([127, 3]))
    case.starts[1] -= 60
    b.start.copy_(ints(case.starts))
    g.replay()
    for out in outs:
        check(out, case)
    ops.check_status()


def test_attention_shared_reports_a_sequence_that_is_shorter_than_its_group(ops):
    case = Case([(2, [(10, 1), (70, 1)])], 4, 2, 64, BF16, seed=1)
    b = case.batch()
    b.start = ints([case.starts[0], 100])                       # (fewer positions than two pages)
    shared = ops.SharedPrefix.of(case.sizes, case.shared, case.kv_lens, "cuda")
    got = ops.attention_shared(case.q.cuda(), case.kv.cuda(), b, shared, case.scale)
    with pytest.raises(ops.KernelError, match="does not fit"):
        ops.check_status()
    assert bool((got[1] == 0).all())
    ops.check_status()


def test_attention_shared_reports_a_sequence_outside_its_group(ops):
    case = Case([(2, [(10, 1), (70, 1)]), (2, [(3, 1)])], 4, 2, 64, BF16, seed=1)
    shared = ops.SharedPrefix.of(case.sizes, case.shared, case.kv_lens, "cuda")
    shared = shared._replace(group_of=ints([0, 1, 1]))          # (group 1 begins with the sequence behind)
    got = ops.attention_shared(case.q.cuda(), case.kv.cuda(), case.batch(), shared, case.scale)
    with pytest.raises(ops.KernelError, match="does not fit"):
        ops.check_status()
    assert bool((got[1] == 0).all())
    want, most = case.want()
    assert bool((((got.double().cpu() - want).abs() / most)[[0, 2]] <= 1.0).all()), "the others' are their own"
    ops.check_status()


def test_attention_shared_refuses(ops):
    case = Case([(2, [(10, 1), (70, 1)])], 4, 2, 64, BF16, seed=1)
    b, q, kv = case.batch(), case.q.cuda(), case.kv.cuda()
    shared = ops.SharedPrefix.of(case.sizes, case.shared, case.kv_lens, "cuda")
    call = lambda **k: ops.attention_shared(*[k.get(n, v) for n, v in (("q", q), ("kv", kv), ("b", b), ("shared", shared))], case.scale,   # noqa: E731
                                            k.get("scratch"), k.get("out"))
    for bad, text in ((dict(q=q.cpu()), "CUDA tensor"), (dict(q=q.transpose(0, 1)), "contiguous"), (dict(kv=kv.float()), "must be torch.bfloat16"),
                      (dict(kv=kv[:, :1]), "kv must be|contiguous"), (dict(q=q[:1]), "rows"), (dict(q=q.half(), kv=kv.half()), "unsupported element type"),
                      (dict(shared=shared._replace(pages=shared.pages.long())), "must be torch.int32"),
                      (dict(shared=shared._replace(group_of=shared.group_of[:1])), "shape"),
                      (dict(scratch=torch.empty(4, device="cuda")), "scratch"), (dict(out=q.float()), "must be torch.bfloat16")):
        with pytest.raises(ops.KernelError, match=text):
            call(**bad)
    with pytest.raises(ops.KernelError, match="kv heads"):
        ops.attention_shared(case.q[:, :3].contiguous().cuda(), kv, b, shared, 1.0)
    with pytest.raises(ops.KernelError, match="longer than the pages"):
        ops.SharedPrefix.of([2], [3], [192, 300], "cuda")
    with pytest.raises(ops.KernelError, match="one group"):
        ops.SharedPrefix.of([1], [3], [200, 300], "cuda")


# ---- tables ------------------------------------------------------------------
def plain_tables(start, q, slots, tables, free, head, width, n_tokens, parent):
    tables = [list(t) for t in tables]
    old = [list(t) for t in tables]
    rows, cu, pos, seq, at = [], [0], [], [], []
    for b in range(len(start)):
        held, total = pages_for(start[b]), pages_for(start[b] + q[b])
        row = [0] * max(width, total)
        if slots[b] != 0:
            src = parent[b] if parent[b] >= 0 else slots[b]
            for j in range(total):
                if j < held:
                    row[j] = old[src][j]
                else:
                    row[j] = free[head] if head < len(free) else 0
                    head += 1
                tables[slots[b]][j] = row[j]
        rows.append(row[:width])
        cu.append(cu[-1] + q[b])
        for i in range(q[b]):
            p = start[b] + i
            pos.append(p), seq.append(b), at.append(row[p // PAGE] * PAGE + p % PAGE)
    pad = n_tokens - len(pos)
    return rows, cu, [s + n for s, n in zip(start, q)], pos + [0] * pad, seq + [0] * pad, at + [-1] * pad, [head], tables


def run_tables(ops, start, q, slots, tables, free, head, width, n_tokens, parent=None):
    n = len(start)
    make = lambda *s, t=torch.int32: torch.full(s, -7, dtype=t, device="cuda")   # noqa: E731
    out = dict(page_table=make(n, width), cu_seqlens=make(n + 1), kv_len=make(n), positions=make(n_tokens), seq_of_token=make(n_tokens),
               slot_map=make(n_tokens, t=torch.int64), head_out=make(1))
    tab = ints(tables)
    ops.step_tables(ints(start), ints(q), ints(slots), tab, ints(free), ints([head]), parent=None if parent is None else ints(parent), **out)
    return [out[k].tolist() for k in ("page_table", "cu_seqlens", "kv_len", "positions", "seq_of_token", "slot_map", "head_out")] + [tab.tolist()]


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("n", [1, 2, 31, 33, 257, 1030])
def test_step_tables(ops, n, seed):
    rng = __import__("random").Random(1000 * seed + n)
    width = rng.choice([1, 3, 40])
    top = width * PAGE
    edge = [0, 1, 63, 64, 65, 127, 128]
    start = [min(rng.choice(edge + [rng.randint(0, top)]), top) for _ in range(n)]
    q = [min(rng.choice([0, 1, 1, 64, rng.randint(0, 200)]), top - s) for s in start]
    slots = rng.sample(range(1, n + 5), n)
    for b in range(n):
        if rng.random() < 0.15:
            slots[b] = 0                                             # padding: one token at position 0 of page 0
            start[b], q[b] = 0, rng.randint(0, 1)
    pool = list(range(1, n * width + 400))
    rng.shuffle(pool)
    tables = [[0] * width for _ in range(n + 5)]
    for b in range(n):
        if slots[b]:
            for j in range(pages_for(start[b])):
                tables[slots[b]][j] = pool.pop()
    parent = [-1] * n
    if seed % 2 and n > 2:
        big = max(range(n), key=lambda b: start[b] if slots[b] else -1)
        for b in range(n):
            if b != big and slots[b] and slots[big] and rng.random() < 0.4:
                parent[b], start[b] = slots[big], rng.randint(0, start[big] // PAGE) * PAGE
                q[b] = min(q[b], top - start[b])
    head, n_tokens = rng.randint(0, 9), sum(q) + rng.choice([0, 5])
    want = plain_tables(start, q, slots, tables, pool, head, width, n_tokens, parent)
    got = run_tables(ops, start, q, slots, tables, pool, head, width, n_tokens, parent if seed % 2 else None)
    for name, a, b in zip(("page_table", "cu_seqlens", "kv_len", "positions", "seq_of_token", "slot_map", "head_out", "tables"), got, want):
        assert a == b, name
    ops.check_status()


def test_step_tables_slots_beyond_31_bits(ops):
    big = (1 << 31) // PAGE + 5
    got = run_tables(ops, [70], [1], [1], [[0, 0], [3, big]], [], 0, 2, 1)
    assert got[5] == [big * PAGE + 6]


def test_step_tables_runs_out_of_pages(ops):
    start, q, slots = [0, 64, 0], [64, 1, 65], [1, 2, 3]
    tables = [[0] * 3, [0] * 3, [9, 0, 0], [0] * 3]
    got = run_tables(ops, start, q, slots, tables, [4, 5, 6], 1, 3, sum(q))
    assert got[0] == [[5, 0, 0], [9, 6, 0], [0, 0, 0]] and got[6] == [5]
    with pytest.raises(ops.KernelError, match="free pages"):
        ops.check_status()
    # a sequence longer than its table
    got = run_tables(ops, [0], [130], [1], [[0, 0], [0, 0]], [4, 5, 6], 0, 2, 130)
    assert got[0] == [[4, 5]]
    with pytest.raises(ops.KernelError, match="outside its tables"):
        ops.check_status()
    # a record that does not exist
    got = run_tables(ops, [0], [1], [9], [[0, 0], [0, 0]], [4, 5, 6], 0, 2, 1)
    assert got[0] == [[0, 0]] and got[6] == [0]
    with pytest.raises(ops.KernelError, match="outside its tables"):
        ops.check_status()


def test_step_tables_refuses(ops):
    i = lambda *v: ints(list(v))   # noqa: E731
    make = lambda: dict(start=i(0), q_len=i(1), slots=i(1), tables=ints([[0], [0]]), free_pages=i(5), free_head=i(0), page_table=ints([[0]]),   # noqa: E731
                        cu_seqlens=i(0, 0), kv_len=i(0), positions=i(0), seq_of_token=i(0), slot_map=torch.zeros(1, dtype=torch.int64, device="cuda"),
                        head_out=i(0))
    ops.step_tables(**make())
    for k, v, text in (("start", i(0, 0), "shape"), ("slots", i(1).cpu(), "CUDA tensor"), ("tables", i(0, 0), "tables must be"),
                       ("slot_map", i(0), "must be torch.int64"), ("cu_seqlens", i(0), "shape"), ("page_table", ints([[0], [0]]), "tables must be")):
        with pytest.raises(ops.KernelError, match=text):
            ops.step_tables(**dict(make(), **{k: v}))
    a = make()
    a["head_out"] = a["free_head"]
    with pytest.raises(ops.KernelError, match="another tensor"):
        ops.step_tables(**a)
    with pytest.raises(ops.KernelError, match="sequences"):
        n = 9000
        z = torch.zeros(n, dtype=torch.int32, device="cuda")
        ops.step_tables(**dict(make(), start=z, q_len=z, slots=z, kv_len=z.clone(), page_table=z.view(n, 1).clone(),
                               cu_seqlens=torch.zeros(n + 1, dtype=torch.int32, device="cuda")))


# ---- histories and steering ----------------------------------------------------
def unpack(words, n):
    v = torch.arange(n)
    return ((words.cpu()[:, v // 32] >> (v % 32)) & 1).bool()


def pack(bits):
    rows, n = bits.shape
    w = torch.zeros((rows, (n + 31) // 32), dtype=torch.int64)
    for v in range(n):
        w[:, v // 32] += bits[:, v].long() << (v % 32)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


@pytest.mark.parametrize("vocab", [1, 31, 32, 33, 1000, 50001])
def test_history(ops, vocab):
    rng = __import__("random").Random(vocab)
    R = 5
    seen, counts = torch.zeros((R, ops.bit_words(vocab)), dtype=torch.int32, device="cuda"), torch.zeros((R, vocab), dtype=torch.int32, device="cuda")
    want_seen, want = torch.zeros((R, vocab), dtype=torch.bool), torch.zeros((R, vocab), dtype=torch.int64)
    for generated in (False, True, True):
        tok = [rng.choice([rng.randrange(vocab), 0, vocab - 1, vocab, -1]) for _ in range(700)]
        row = [rng.choice([0, 1, 2, 3, 4, -1, R]) for _ in tok]
        ops.history_add(seen, counts, ints(tok), ints(row), generated=generated)
        for t, r in zip(tok, row):
            if 0 <= t < vocab and 0 <= r < R:
                want_seen[r, t] = True
                want[r, t] += generated
    assert torch.equal(unpack(seen, vocab), want_seen) and torch.equal(counts.cpu().long(), want)
    ops.history_clear(seen, counts, ints([3, -1, 0, R, 3]))
    for r in (0, 3):
        want_seen[r], want[r] = False, 0
    assert torch.equal(unpack(seen, vocab), want_seen) and torch.equal(counts.cpu().long(), want)
    ops.history_add(seen, counts, ints([]), ints([]), generated=True)
    ops.history_clear(seen, counts, ints([]))


def plain_steer(x, rows, seen, counts, pen, bias, masks, mask_of):
    x = x.double().clone()
    for i, r in enumerate(rows):
        if not 0 <= r < len(pen):
            continue
        rep, freq, pres = pen[r].double().tolist()
        s = seen[r]
        x[i, s] = torch.where(x[i, s] > 0, x[i, s] / rep, x[i, s] * rep)
        n = counts[r].double()
        x[i] = torch.where(n > 0, x[i] - (freq * n + pres), x[i])
        for t, b in bias[r].items():
            x[i, t] += b
        if mask_of[r] >= 0:
            x[i, ~masks[mask_of[r]]] = -math.inf
    return x


@pytest.mark.parametrize("place", ["in place", "out", "strided", "out of step"])
@pytest.mark.parametrize("vocab", [1, 3, 32, 37, 1000, 4101, 33335])
def test_steer_logits(ops, vocab, place):
    g = torch.Generator().manual_seed(vocab)
    rng = __import__("random").Random(vocab)
    R, n = 6, 7
    rows = [4, 0, 2, 5, 3, -1, R + 2]
    x = torch.randn((n, vocab), generator=g) * 4
    x[0, vocab // 2] = math.inf
    x[1, 0] = -math.inf
    x[2, vocab - 1] = math.nan
    x[3, 0] = 0.0
    x[4] = torch.finfo(F32).min
    seen = torch.rand((R, vocab), generator=g) < 0.2
    seen[:, vocab - 1] = True
    counts = torch.where(seen & (torch.rand((R, vocab), generator=g) < 0.5), torch.randint(1, 50, (R, vocab), generator=g), 0).to(torch.int32)
    pen = torch.stack([torch.rand(R, generator=g) + 0.6, torch.randn(R, generator=g), torch.randn(R, generator=g)], 1).contiguous()
    masks = torch.rand((4, vocab), generator=g) < torch.tensor([0.5, 0.02, 0.98, 0.0])[:, None]     # (the last allows nothing)
    mask_of = [-1, 0, 2, 3, 1, 0]
    bias = [{rng.randrange(vocab): rng.uniform(-9, 9) for _ in range(k)} for k in (0, 3, 500, 1, 40, 1)]
    bias[4][vocab - 1] = math.inf
    cu = [0]
    for b in bias:
        cu.append(cu[-1] + len(b))
    values = torch.tensor([v for b in bias for v in b.values()], dtype=F32)
    bias = [dict(zip(b, values[a:].tolist())) for a, b in zip(cu, bias)]
    want = plain_steer(x, rows, seen, counts, pen, bias, masks, mask_of)
    dx = x.cuda()
    kw = dict(seen=pack(seen).cuda(), counts=counts.cuda(), penalties=pen.cuda(), bias=(ints(cu), ints([t for b in bias for t in b]), values.cuda()),
              masks=pack(masks).cuda(), mask_of=ints(mask_of))
    if place == "strided":                                           # rows further apart than the vocabulary, and not by a multiple of 4
        wide = torch.zeros((n, vocab + 5), device="cuda")
        dx = wide[:, :vocab]
        dx.copy_(x)
    out = None
    if place == "out":
        out = torch.full((n, vocab), 5.0, device="cuda")
    elif place == "out of step":                                     # begins 4 bytes further than the logits
        out = torch.full((n * vocab + 1,), 5.0, device="cuda")[1:].view(n, vocab)
    got = ops.steer_logits(dx, ints(rows), out=out, **kw)
    assert got is (dx if out is None else out)
    if out is not None:
        assert torch.equal(dx.cpu().nan_to_num(7.0), x.nan_to_num(7.0)), "the logits stay"
    elif place == "strided":
        assert bool((wide[:, vocab:] == 0).all())
    got = got.cpu().double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    # four roundings of numbers no larger than this in size
    size = x.double().abs()[fine] * 2 + 50 * 5 + 10
    assert bool(((got - want)[fine].abs() <= 4 * 2.0 ** -24 * size).all())


def test_steer_logits_with_some_of_its_rules(ops):
    x = torch.randn((3, 70), generator=torch.Generator().manual_seed(1)).cuda()
    assert torch.equal(ops.steer_logits(x.clone()), x)
    allowed = torch.zeros((1, 70), dtype=torch.bool)
    allowed[0, ::3] = True
    got = ops.steer_logits(x.clone(), masks=pack(allowed).cuda(), mask_of=ints([0, -1, 0]))
    assert torch.equal(got[1], x[1]) and bool((got[0].cpu()[~allowed[0]] == -math.inf).all()) and torch.equal(got[2][::3], x[2][::3])
    got = ops.steer_logits(x.clone(), bias=(ints([0, 0, 1, 1]), ints([69]), torch.tensor([2.5], device="cuda")))
    want = x.clone()
    want[1, 69] += 2.5
    assert torch.equal(got, want)
    assert ops.steer_logits(x[:0]).shape == (0, 70)


def test_steer_logits_is_what_the_repetition_penalty_kernel_does(ops):
    x = torch.randn((2, 999), generator=torch.Generator().manual_seed(1)).cuda()
    hist = [[5, 7, 5, 998], [0, 1, 2]]
    want = ops.repetition_penalty(x.clone(), hist, 1.3)
    seen, counts = torch.zeros((2, 32), dtype=torch.int32, device="cuda"), torch.zeros((2, 999), dtype=torch.int32, device="cuda")
    ops.history_add(seen, counts, ints([t for h in hist for t in h]), ints([i for i, h in enumerate(hist) for _ in h]), generated=False)
    got = ops.steer_logits(x.clone(), seen=seen, counts=counts, penalties=torch.tensor([[1.3, 0.5, 0.5]] * 2, device="cuda"))
    assert torch.equal(got, want)


def test_steer_and_history_refuse(ops):
    x = torch.zeros((2, 70), device="cuda")
    seen, counts, pen = torch.zeros((2, 3), dtype=torch.int32, device="cuda"), torch.zeros((2, 70), dtype=torch.int32, device="cuda"), torch.ones((2, 3), device="cuda")
    for kw, text in ((dict(seen=seen, counts=counts), "come together"), (dict(penalties=pen), "come together"), (dict(seen=seen[:, :2], counts=counts, penalties=pen), "contiguous|shape"),
                     (dict(seen=seen, counts=counts[:1], penalties=pen), "shape"), (dict(masks=seen), "come together"), (dict(mask_of=ints([0, 0])), "come together"),
                     (dict(masks=seen[:, :2].contiguous(), mask_of=ints([0, 0])), "shape"), (dict(rows=ints([0])), "shape"),
                     (dict(seen=seen, counts=counts, penalties=pen, mask_of=ints([0]), masks=seen), "places"),
                     (dict(bias=(ints([0, 0, 0]), ints([1]), torch.zeros(2, device="cuda"))), "shape"), (dict(out=x[:1]), "out must be")):
        with pytest.raises(ops.KernelError, match=text):
            ops.steer_logits(x, **kw)
    for bad in (x.cpu(), x.double(), x.t()):
        with pytest.raises(ops.KernelError, match="float32 rows"):
            ops.steer_logits(bad)
    with pytest.raises(ops.KernelError, match="shape"):
        ops.history_add(seen, counts, ints([1]), ints([1, 2]), generated=True)
    with pytest.raises(ops.KernelError, match="must be torch.int32"):
        ops.history_clear(seen, counts.long(), ints([1]))
